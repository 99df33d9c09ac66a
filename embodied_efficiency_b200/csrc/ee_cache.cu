// ee_cache.cu -- C ABI: keys and values of new tokens quantised into a paged
// cache, and read back in 16 bits.
//
// Per token and head a step s = max(amax |x| / most, 1e-8), most = 127 or 7,
// and codes rint(x / s) (true division, ties to even; the framework's weight
// format). A head that holds an infinity or NaN gets codes of 0 and a NaN step,
// so it stays visible in every result that reads it.
//
// HBM-bound: 2 bytes a value on one side, 1 or 1/2 and 4 / hd on the other. One
// warp per token: hd / 8 lanes a head, 16 bytes a lane, several heads of keys
// and values in flight; the loads of a token's values are under way before its
// place is looked up (a search over the offsets and one entry of the table).
//
// Measured: 128 prompts of 257 to 816 tokens, 16 heads of 64, written in 8 bits in
// 82 us (5.4 TB/s of the 6.46 that a copy reaches); 64 such prompts, heads of 128,
// read in 73 (6.0); 64 x 1 token written in 3.3, a launch. In 4 bits the write takes
// what it takes in 8 (instructions a value), the read 0.92 of it. Several tokens a
// warp were slower in either direction.
#include "ee_cache.cuh"
#include "ee_host.h"

namespace ee {

struct CacheCopyArgs {
  CacheView c;
  void *k_codes, *v_codes;
  float *k_steps, *v_steps;
  void *k, *v;  // packed tokens
  long long k_tok, k_head, v_tok, v_head;  // strides, elements
  const int* cu;
  int tokens;
};

constexpr int kCacheWarps = 4;

// Divisions by Markstein's correction of a quotient with its remainder (IBM J.
// Res. Dev. 34, 1990): q' = q + (v - q s) / s in two fused operations, rounded as
// the division rounds -- for every 16-bit value under every 16-bit largest value,
// all of which the tests go through.
template <int BITS>
EE_DEV float cache_step(float amax) {
  constexpr float MOST = BITS == 8 ? 127.f : 7.f, INV = 1.f / MOST;
  const float q = amax * INV;
  return fmaxf(fmaf(fmaf(-q, MOST, amax), INV, q), 1e-8f);
}
// Nearest integers (ties to even) of the quotients of eight values and s: 8
// bytes, or 4 with two codes each.
template <int BITS>
EE_DEV uint2 cache_codes(const uint64_t (&v)[4], float s) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  inv = fmaf(fmaf(-s, inv, 1.f), inv, inv);
  const uint64_t inv2 = both(inv), neg2 = both(-s), magic = both(12582912.f);  // 1.5 * 2^23: the sum's rounding is rint
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t q = mul2f(v[i], inv2);
    unpack64(add2f(fma2f(fma2f(q, neg2, v[i]), inv2, q), magic), b[2 * i], b[2 * i + 1]);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = prmt(prmt(b[4 * h], b[4 * h + 1], 0x0040u), prmt(b[4 * h + 2], b[4 * h + 3], 0x0040u), 0x5410u);
  if (BITS == 8) return make_uint2(w[0], w[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] &= 0x0F0F0F0Fu;
    w[h] |= w[h] >> 4;  // bytes 0 and 2: a pair of codes each
  }
  return make_uint2(prmt(w[0], w[1], 0x6420u), 0u);
}
// Larger magnitude of the halves of two words by themselves, NaN if either is
template <typename T> EE_DEV uint32_t max_abs2(uint32_t a, uint32_t b);
template <> EE_DEV uint32_t max_abs2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{\n\t.reg .b32 x, y;\n\tabs.bf16x2 x, %1;\n\tabs.bf16x2 y, %2;\n\tmax.NaN.bf16x2 %0, x, y;\n\t}" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <> EE_DEV uint32_t max_abs2<__half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{\n\t.reg .b32 x, y;\n\tabs.f16x2 x, %1;\n\tabs.f16x2 y, %2;\n\tmax.NaN.f16x2 %0, x, y;\n\t}" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_write_kernel(const __grid_constant__ CacheCopyArgs a) {
  constexpr int CH = HD / 8, HL = 32 / CH, UN = 2;  // lanes a head, heads at once, of them (K and V) in flight
  constexpr int RB = HD * BITS / 8;
  pdl_entry();
  const int lane = threadIdx.x & 31, c = lane % CH;
  const long long tt = (long long)blockIdx.x * kCacheWarps + (threadIdx.x >> 5);
  if (tt >= a.tokens) return;
  const int t = (int)tt;
  const T* ks = reinterpret_cast<const T*>(a.k) + t * a.k_tok + (lane / CH) * a.k_head + 8 * c;
  const T* vs = reinterpret_cast<const T*>(a.v) + t * a.v_tok + (lane / CH) * a.v_head + 8 * c;
  long long at = -1;  // this lane's row of codes
#pragma unroll 1
  for (int h0 = 0; h0 < a.c.n_kv; h0 += UN * HL) {
    uint4 x[UN][2];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      x[u][0] = x[u][1] = make_uint4(0, 0, 0, 0);
      if (h0 + u * HL + lane / CH < a.c.n_kv) {
        x[u][0] = *reinterpret_cast<const uint4*>(ks);
        x[u][1] = *reinterpret_cast<const uint4*>(vs);
      }
      ks += HL * a.k_head;
      vs += HL * a.v_head;
    }
    if (h0 == 0) {  // under the first loads
      const long long row = cache_place(a.c, a.cu, cache_seq(a.cu, a.c.n_seq, t), t);
      if (row < 0) return;
      at = row + ((long long)(lane / CH) << a.c.shift);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (h0 + u * HL >= a.c.n_kv) break;
      uint32_t mx[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mx[i] = max_abs2<T>(max_abs2<T>(x[u][i].x, x[u][i].y), max_abs2<T>(x[u][i].z, x[u][i].w));
      uint32_t m = max_abs2<T>(prmt(mx[0], mx[1], 0x5410u), prmt(mx[0], mx[1], 0x7632u));  // K's and V's
#pragma unroll
      for (int o = 1; o < CH; o <<= 1) m = max_abs2<T>(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float2 amax = Act<T>::unpack2(m);
      const bool have = h0 + u * HL + lane / CH < a.c.n_kv;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {x[u][i].x, x[u][i].y, x[u][i].z, x[u][i].w};
        const bool finite = (i ? amax.y : amax.x) <= 3.4028234e38f;  // false for infinities and NaN
        const float s = cache_step<BITS>(i ? amax.y : amax.x);
        uint64_t v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 p = Act<T>::unpack2(w[e]);
          v[e] = pack64(__float_as_uint(p.x), __float_as_uint(p.y));
        }
        uint2 codes = cache_codes<BITS>(v, s);
        if (!finite) codes = make_uint2(0, 0);
        if (!have) continue;
        uint8_t* dst = reinterpret_cast<uint8_t*>(i ? a.v_codes : a.k_codes) + at * RB + c * BITS;
        if (BITS == 8) *reinterpret_cast<uint2*>(dst) = codes;
        else *reinterpret_cast<uint32_t*>(dst) = codes.x;
        if (c == 0) (i ? a.v_steps : a.k_steps)[at] = finite ? s : __int_as_float(0x7fffffff);
      }
      at += (long long)HL << a.c.shift;
    }
  }
}

template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_read_kernel(const __grid_constant__ CacheCopyArgs a) {
  constexpr int CH = HD / 8, HL = 32 / CH, UN = 2, RB = HD * BITS / 8;
  pdl_entry();
  const int lane = threadIdx.x & 31, c = lane % CH;
  const long long tt = (long long)blockIdx.x * kCacheWarps + (threadIdx.x >> 5);
  if (tt >= a.tokens) return;
  const int t = (int)tt;
  const long long row = cache_place(a.c, a.cu, cache_seq(a.cu, a.c.n_seq, t), t);
  if (row < 0) return;
  long long at = row + ((long long)(lane / CH) << a.c.shift);
  T* kd = reinterpret_cast<T*>(a.k) + t * a.k_tok + (lane / CH) * a.k_head + 8 * c;
  T* vd = reinterpret_cast<T*>(a.v) + t * a.v_tok + (lane / CH) * a.v_head + 8 * c;
#pragma unroll 1
  for (int h = lane / CH; h < a.c.n_kv; h += UN * HL) {
    uint2 w[UN][2];
    float s[UN][2];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (h + u * HL >= a.c.n_kv) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(i ? a.v_codes : a.k_codes) + at * RB + c * BITS;
        if (BITS == 8) w[u][i] = *reinterpret_cast<const uint2*>(src);
        else w[u][i] = make_uint2(*reinterpret_cast<const uint32_t*>(src), 0u);
        s[u][i] = (i ? a.v_steps : a.k_steps)[at];
      }
      at += (long long)HL << a.c.shift;
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (h + u * HL >= a.c.n_kv) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // codes as fp16, exact
          const uint32_t x = BITS == 8 && e > 1 ? w[u][i].y : w[u][i].x;
          const float2 f =
              Act<__half>::unpack2(BITS == 8 ? code_pair8<__half>(x ^ 0x80808080u, e & 1) : code_pair4<__half>(x, x >> 4, e));
          uint32_t y0, y1;
          unpack64(mul2f(pack64(__float_as_uint(f.x), __float_as_uint(f.y)), both(s[u][i])), y0, y1);
          o[e] = Act<T>::pack2(__uint_as_float(y0), __uint_as_float(y1));
        }
        *reinterpret_cast<uint4*>(i ? vd : kd) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      kd += HL * a.k_head;
      vd += HL * a.v_head;
    }
  }
}

template <typename T, int HD, int BITS>
static int launch_copy_b(const CacheCopyArgs& a, bool write, cudaStream_t s) {
  const dim3 grid((unsigned)((a.tokens + (long long)kCacheWarps - 1) / kCacheWarps)), blk(kCacheWarps * 32);
  const cudaError_t e = write ? launch_pdl(cache_write_kernel<T, HD, BITS>, grid, blk, 0, s, a)
                              : launch_pdl(cache_read_kernel<T, HD, BITS>, grid, blk, 0, s, a);
  return e == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}
template <typename T>
static int launch_copy(const CacheCopyArgs& a, int hd, int bits, bool write, cudaStream_t s) {
  if (hd == 64) return bits == 8 ? launch_copy_b<T, 64, 8>(a, write, s) : launch_copy_b<T, 64, 4>(a, write, s);
  return bits == 8 ? launch_copy_b<T, 128, 8>(a, write, s) : launch_copy_b<T, 128, 4>(a, write, s);
}

// What every call on a cache checks; fills the view.
int cache_view(const ee_cache* c, const int32_t* table, int64_t table_row, int32_t width, const int32_t* k_lens,
               int32_t n_seq, CacheView* v) {
  if (!c) return EE_ERR_ARG;
  if (c->bits != 8 && c->bits != 4) return EE_ERR_UNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return EE_ERR_UNSUPPORTED;
  if (c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256) return EE_ERR_UNSUPPORTED;
  if (c->pages < 0 || c->kv_heads < 1 || c->kv_heads > 65535 || n_seq < 0 || width < 0) return EE_ERR_SHAPE;
  if ((int64_t)c->pages * c->kv_heads > 0x7fffffff / c->page_size) return EE_ERR_SHAPE;  // rows are 31-bit numbers
  if ((int64_t)width > 0x7fff0000 / c->page_size) return EE_ERR_SHAPE;  // so are keys, and a tile past the last
  if (c->pages && (!c->k_codes || !c->v_codes || !c->k_steps || !c->v_steps)) return EE_ERR_ARG;
  if (n_seq && (!k_lens || (width && !table))) return EE_ERR_ARG;
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->k_steps | (uintptr_t)c->v_steps) & 15)
    return EE_ERR_ALIGN;
  if (((uintptr_t)table | (uintptr_t)k_lens) & 3) return EE_ERR_ALIGN;
  v->table = table;
  v->k_lens = k_lens;
  v->table_row = table_row;
  v->n_seq = n_seq;
  v->width = width;
  v->pages = c->pages;
  v->n_kv = c->kv_heads;
  v->shift = c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : c->page_size == 128 ? 7 : 8;
  return EE_OK;
}

static int cache_copy(const ee_cache* c, void* k, int64_t k_tok, int64_t k_head, void* v, int64_t v_tok, int64_t v_head,
                      const int32_t* cu, const int32_t* table, int64_t table_row, int32_t width, const int32_t* k_lens,
                      int64_t tokens, int32_t n_seq, int32_t act_dtype, bool write, cudaStream_t s) {
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  CacheCopyArgs a{};
  int rc = cache_view(c, table, table_row, width, k_lens, n_seq, &a.c);
  if (rc) return rc;
  if (tokens < 0 || tokens > 0x7fffff00) return EE_ERR_SHAPE;
  if (tokens == 0 || n_seq == 0 || width == 0 || c->pages == 0) return EE_OK;
  if (!k || !v || !cu) return EE_ERR_ARG;
  if (!aligned16(k) || !aligned16(v) || ((uintptr_t)cu & 3)) return EE_ERR_ALIGN;
  if ((k_tok | k_head | v_tok | v_head) % 8 != 0) return EE_ERR_ALIGN;
  rc = check_device();
  if (rc) return rc;
  a.k_codes = c->k_codes; a.v_codes = c->v_codes;
  a.k_steps = c->k_steps; a.v_steps = c->v_steps;
  a.k = k; a.v = v;
  a.k_tok = k_tok; a.k_head = k_head; a.v_tok = v_tok; a.v_head = v_head;
  a.cu = cu;
  a.tokens = (int)tokens;
  return act_dtype == EE_BF16 ? launch_copy<__nv_bfloat16>(a, c->head_dim, c->bits, write, s)
                              : launch_copy<__half>(a, c->head_dim, c->bits, write, s);
}

}  // namespace ee

using namespace ee;

extern "C" {

int ee_cache_write(const ee_cache* cache, const void* k, int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
                   int64_t v_head, const int32_t* cu, const int32_t* table, int64_t table_row, int32_t width,
                   const int32_t* k_lens, int64_t tokens, int32_t n_seq, int32_t act_dtype, ee_stream_t stream) {
  return cache_copy(cache, const_cast<void*>(k), k_tok, k_head, const_cast<void*>(v), v_tok, v_head, cu, table, table_row,
                    width, k_lens, tokens, n_seq, act_dtype, true, (cudaStream_t)stream);
}

int ee_cache_read(const ee_cache* cache, void* k, int64_t k_tok, int64_t k_head, void* v, int64_t v_tok, int64_t v_head,
                  const int32_t* cu, const int32_t* table, int64_t table_row, int32_t width, const int32_t* k_lens,
                  int64_t tokens, int32_t n_seq, int32_t act_dtype, ee_stream_t stream) {
  return cache_copy(cache, k, k_tok, k_head, v, v_tok, v_head, cu, table, table_row, width, k_lens, tokens, n_seq,
                    act_dtype, false, (cudaStream_t)stream);
}

}  // extern "C"
