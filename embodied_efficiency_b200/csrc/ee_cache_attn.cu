// ee_cache_attn.cu -- C ABI: attention over a paged cache of quantised keys and
// values, behind a prefix in 16 bits that the sequences share.
#include <cfloat>

#include "ee_cache_attn.cuh"

namespace ee {

int* gemm_status_ptr();  // ee_ops.cu: the status word of the tensor-core kernels on the current device
int cache_view(const ee_cache* c, const int32_t* table, int64_t table_row, int32_t width, const int32_t* k_lens,
               int32_t n_seq, CacheView* v);                       // ee_cache.cu
// ee_prompt.cu
int prompt_sums_splits(long long tq, long long tk, int n_q, int n_kv);
int prompt_parts(long long tq, int n_seq, int n_q, int n_kv, long long keys, int tiles);
int launch_prompt_sums(const PromptArgs& a, int head_dim, int act_dtype, cudaStream_t s);
int launch_prompt_more(const PromptArgs& a, const PromptMore& more, int head_dim, int act_dtype, cudaStream_t s);
int launch_prompt_combine(const PromptArgs& a, int head_dim, int act_dtype, cudaStream_t s);
unsigned long long attention_wait_limit();

// How a call runs, by its mean of rows (queries x group) per sequence and key
// head: up to 8, one MMA column tile a warp; up to 16, two; above, the
// tensor-core kernel's 128-row tiles (64 x 50 rows behind 257..816, 16 heads of
// 128: the kernel for few rows in 64-row items took 239 us). One kernel serves the
// whole call: 63 single tokens behind 1..1632 beside one turn of 1024 tokens, 16 /
// 4 heads of 128, take 81 us, as two calls 22 + 36; beside a turn of 200 54, as two
// 22 + 20. Which tokens to put together is the caller's to say: the host does not
// know the lengths.
static CachePlan cache_plan(long long tq, int n_seq, int n_q, int n_kv, long long keys) {
  const int group = n_q / n_kv;
  const long long rows = tq * group;
  if (rows <= 8ll * n_seq) return CachePlan{1, 1};
  if (rows <= 16ll * n_seq || group > 128) return CachePlan{2, 1};
  return CachePlan{0, prompt_parts(tq, n_seq, n_q, n_kv, keys, 1)};
}
template <int HD, int BITS>
static int plan_workers_b(const CachePlan& p) {
  return p.nt > 1 ? CaShape<HD, BITS, 2>::WORKERS : CaShape<HD, BITS, 1>::WORKERS;
}
static int plan_workers(const CachePlan& p, int hd, int bits) {
  if (hd == 64) return bits == 8 ? plan_workers_b<64, 8>(p) : plan_workers_b<64, 4>(p);
  return bits == 8 ? plan_workers_b<128, 8>(p) : plan_workers_b<128, 4>(p);
}
// Partial rows: of the prefix, of the call's own keys in its layout. With one
// part of either (tensor-core kernel) the prefix comes second and finishes the
// rows: of the three passes over fp32 sums that joining them afterwards takes one
// is left (6400 tokens, 16 heads of 128: 158 us where the call took 184).
struct CacheParts {
  long long own, pre;
  int pre_splits;
  bool joined;
};
static CacheParts cache_parts(const CachePlan& p, long long tq, int n_q, int n_kv, int hd, int bits, long long prefix_len) {
  CacheParts c{0, 0, 0, false};
  if (prefix_len) c.pre_splits = prompt_sums_splits(tq, prefix_len, n_q, n_kv);
  c.joined = p.nt == 0 && p.splits == 1 && c.pre_splits == 1;
  c.pre = c.joined ? 0 : c.pre_splits * tq * n_q;
  if (p.nt == 0) c.own = p.splits > 1 || prefix_len ? p.splits * tq * n_q : 0;
  else c.own = (long long)device_sms() * plan_workers(p, hd, bits) * 2 * 8 * p.nt + (prefix_len ? tq * n_q : 0);
  return c;
}

}  // namespace ee

using namespace ee;

extern "C" {

size_t ee_cache_attention_workspace_bytes(int64_t tq, int32_t n_seq, int32_t n_q, int32_t n_kv, int32_t head_dim,
                                          int32_t bits, int64_t keys, int64_t prefix_len) {
  if (tq < 1 || n_seq < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv || keys < 0 || prefix_len < 0 || tq > 0x7fffff00 / n_q) return 0;
  if ((head_dim != 64 && head_dim != 128) || (bits != 8 && bits != 4)) return 0;
  if (prefix_len && n_q / n_kv > 128) return 0;  // the call refuses it
  const CacheParts c = cache_parts(cache_plan(tq, n_seq, n_q, n_kv, keys), tq, n_q, n_kv, head_dim, bits, prefix_len);
  return (size_t)(c.own + c.pre) * (head_dim + 2) * 4;
}

int ee_cache_attention(const ee_cache* cache, const void* q, int64_t q_tok, int64_t q_head, void* out, int64_t o_tok,
                       int64_t o_head, const int32_t* cu_q, const int32_t* table, int64_t table_row, int32_t width,
                       const int32_t* k_lens, const void* prefix_k, int64_t pk_tok, int64_t pk_head,
                       const void* prefix_v, int64_t pv_tok, int64_t pv_head, int64_t prefix_len, int64_t tq,
                       int32_t n_seq, int32_t n_q, int32_t causal, float scale, int32_t act_dtype, void* workspace,
                       size_t workspace_bytes, ee_stream_t stream) {
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  CacheAttnArgs a{};
  int rc = cache_view(cache, table, table_row, width, k_lens, n_seq, &a.c);
  if (rc) return rc;
  const int n_kv = cache->kv_heads, hd = cache->head_dim;
  if (tq < 0 || n_q < 1 || n_q > 65535 || n_q % n_kv != 0 || prefix_len < 0 || prefix_len > 0x7fffff00) return EE_ERR_SHAPE;
  if (tq > 0x7fffff00 / n_q) return EE_ERR_SHAPE;  // rows are 31-bit numbers
  if (prefix_len && n_q / n_kv > 128) return EE_ERR_UNSUPPORTED;
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.f) || !(scale_log2 <= FLT_MAX)) return EE_ERR_ARG;
  if (tq == 0 || n_seq == 0) return EE_OK;
  if (!q || !out || !cu_q || (prefix_len && (!prefix_k || !prefix_v))) return EE_ERR_ARG;
  if (!aligned16(q) || !aligned16(out) || ((uintptr_t)cu_q & 3)) return EE_ERR_ALIGN;
  if ((q_tok | q_head | o_tok | o_head) % 8 != 0) return EE_ERR_ALIGN;
  if (prefix_len && (!aligned16(prefix_k) || !aligned16(prefix_v) || (pk_tok | pk_head | pv_tok | pv_head) % 8 != 0))
    return EE_ERR_ALIGN;
  rc = check_device();
  if (rc) return rc;
  const long long keys = (long long)width * cache->page_size;
  const CachePlan plan = cache_plan(tq, n_seq, n_q, n_kv, keys);
  const CacheParts cp = cache_parts(plan, tq, n_q, n_kv, hd, cache->bits, prefix_len);
  const size_t need = ee_cache_attention_workspace_bytes(tq, n_seq, n_q, n_kv, hd, cache->bits, keys, prefix_len);
  if (need && (!workspace || workspace_bytes < need)) return EE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return EE_ERR_ALIGN;
  cudaStream_t s = (cudaStream_t)stream;
  int* status = gemm_status_ptr();
  if (!status) return EE_ERR_DEVICE;
  if (cache->pages == 0) a.c.width = 0;  // no keys but the prefix's: the maps are not used
  CacheMaps m{};
  if (a.c.width > 0) {
    const int rb = hd * cache->bits / 8;
    const uint64_t rows = (uint64_t)cache->pages * n_kv * cache->page_size;
    const auto sw = plan.nt == 0 ? CU_TENSOR_MAP_SWIZZLE_NONE
                    : rb == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                    : rb == 64   ? CU_TENSOR_MAP_SWIZZLE_64B
                                 : CU_TENSOR_MAP_SWIZZLE_32B;
    const int box = plan.nt ? kCaKeys : cache->page_size < 128 ? cache->page_size : 128;
    if (!make_tmap_2d(&m.k, cache->k_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rb, rows, rb, rb, box, sw) ||
        !make_tmap_2d(&m.v, cache->v_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rb, rows, rb, rb, box, sw))
      return EE_ERR_SHAPE;
  }
  float* part = reinterpret_cast<float*>(workspace);
  float* stat = part + (cp.own + cp.pre) * hd;
  // of the prefix: behind the parts of the call's own keys in the kernel for few rows, before them in the other
  const long long pre_at = plan.nt ? cp.own : 0;
  PromptArgs p{};
  p.q = q;
  p.q_tok = q_tok; p.q_head = q_head;
  p.tq = (int)tq;
  p.n_q = n_q; p.n_kv = n_kv; p.group = n_q / n_kv;
  p.scale_log2 = scale_log2;
  PromptArgs x = p;  // the prefix: one sequence of all rows
  if (prefix_len) {
    x.k = prefix_k; x.v = prefix_v;
    x.k_tok = pk_tok; x.k_head = pk_head; x.v_tok = pv_tok; x.v_head = pv_head;
    x.tk = (int)prefix_len;
    x.n_seq = 1;
    x.splits = cp.pre_splits;
    x.sums = !cp.joined;
    x.part = part + pre_at * hd;
    x.stat = stat + pre_at * 2;
    x.out = out;
    x.o_tok = o_tok; x.o_head = o_head;
    rc = cp.joined ? EE_OK : launch_prompt_sums(x, hd, act_dtype, s);
    if (rc) return rc;
  }
  if (plan.nt) {
    a.q = q; a.out = out;
    a.cu_q = cu_q;
    a.q_tok = q_tok; a.q_head = q_head; a.o_tok = o_tok; a.o_head = o_head;
    a.tq = (int)tq; a.n_q = n_q; a.group = n_q / n_kv;
    a.causal = causal != 0;
    a.rows = 8 * plan.nt;
    a.rows_log2 = plan.nt > 1 ? 4 : 3;
    a.scale_log2 = scale_log2;
    a.k_steps = cache->k_steps; a.v_steps = cache->v_steps;
    a.part = part; a.stat = stat;
    a.whole = cp.own - (prefix_len ? tq * n_q : 0);
    a.pre_splits = cp.pre_splits;
    if (prefix_len) {
      const int tpt = 128 / a.group;
      const long long items = (tq + 2 * tpt - 1) / (2 * tpt) * n_kv * cp.pre_splits;
      a.pre_ctas = items < 0x7fffffff ? (int)items : 0x7fffffff;
    }
    a.status = status;
    a.timeout_ns = attention_wait_limit();
    if (act_dtype == EE_BF16)
      return hd == 64 ? launch_cache_few<__nv_bfloat16, 64>(m, a, plan, cache->bits, s)
                      : launch_cache_few<__nv_bfloat16, 128>(m, a, plan, cache->bits, s);
    return hd == 64 ? launch_cache_few<__half, 64>(m, a, plan, cache->bits, s)
                    : launch_cache_few<__half, 128>(m, a, plan, cache->bits, s);
  }
  PromptTcArgs t{};
  p.out = out;
  p.o_tok = o_tok; p.o_head = o_head;
  p.cu_q = cu_q;
  p.k_lens = k_lens;
  p.tk = a.c.width << a.c.shift;
  p.n_seq = n_seq;
  p.causal = causal != 0;
  p.splits = plan.splits;
  const bool whole = plan.splits == 1 && !prefix_len;  // rows are finished where they are summed
  p.sums = !whole;
  p.part = part + cp.pre * hd;
  p.stat = stat + cp.pre * 2;
  t.p = p;
  t.tpt = 128 / p.group;
  t.status = status;
  t.timeout_ns = attention_wait_limit();
  t.c = a.c;
  t.k_steps = cache->k_steps; t.v_steps = cache->v_steps;
  if (act_dtype == EE_BF16)
    rc = hd == 64 ? launch_cache_many<__nv_bfloat16, 64>(m, t, cache->bits, s)
                  : launch_cache_many<__nv_bfloat16, 128>(m, t, cache->bits, s);
  else
    rc = hd == 64 ? launch_cache_many<__half, 64>(m, t, cache->bits, s) : launch_cache_many<__half, 128>(m, t, cache->bits, s);
  if (rc || whole) return rc;
  if (cp.joined) return launch_prompt_more(x, PromptMore{p.part, p.stat, cu_q, n_seq}, hd, act_dtype, s);
  p.splits = cp.pre_splits + plan.splits;
  p.part = part;
  p.stat = stat;
  return launch_prompt_combine(p, hd, act_dtype, s);
}

}  // extern "C"
