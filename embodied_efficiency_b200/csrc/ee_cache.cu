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
#include "ee_cache.cuh"
#include "ee_host.h"
#include "ee_quant.cuh"

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

// Codes of eight values: 8 bytes, or 4 with two codes each.
template <int BITS>
EE_DEV uint2 cache_codes(const float (&f)[8], float s, uint64_t inv2) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = quant_word(pack64(__float_as_uint(f[4 * h]), __float_as_uint(f[4 * h + 1])),
                      pack64(__float_as_uint(f[4 * h + 2]), __float_as_uint(f[4 * h + 3])), s, inv2);
  if (BITS == 8) return make_uint2(w[0], w[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] &= 0x0F0F0F0Fu;
    w[h] |= w[h] >> 4;  // bytes 0 and 2: a pair of codes each
  }
  return make_uint2(prmt(w[0], w[1], 0x6420u), 0u);
}

template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_write_kernel(const __grid_constant__ CacheCopyArgs a) {
  constexpr int CH = HD / 8, HL = 32 / CH, UN = 4;  // lanes a head, heads at once, of them in flight
  pdl_entry();
  const int lane = threadIdx.x & 31, c = lane % CH;
  const long long tt = (long long)blockIdx.x * kCacheWarps + (threadIdx.x >> 5);
  if (tt >= a.tokens) return;
  const int t = (int)tt, heads = 2 * a.c.n_kv;
  long long row = -1;
  for (int h0 = 0; h0 < heads; h0 += UN * HL) {
    uint4 x[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u * HL + lane / CH;
      x[u] = make_uint4(0, 0, 0, 0);
      if (h < heads) {
        const T* src = h < a.c.n_kv ? reinterpret_cast<const T*>(a.k) + t * a.k_tok + h * a.k_head
                                    : reinterpret_cast<const T*>(a.v) + t * a.v_tok + (h - a.c.n_kv) * a.v_head;
        x[u] = *reinterpret_cast<const uint4*>(src + 8 * c);
      }
    }
    if (h0 == 0) {
      row = cache_place(a.c, a.cu, cache_seq(a.cu, a.c.n_seq, t), t);
      if (row < 0) return;
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u * HL + lane / CH;
      const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
      uint32_t mx = 0;  // 15-bit magnitudes as integers: an infinity or NaN wins
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = __vmaxu2(mx, xw[e] & 0x7FFF7FFFu);
      mx = max(mx & 0xFFFFu, mx >> 16);
#pragma unroll
      for (int o = 1; o < CH; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (h >= heads) continue;
      const float amax = Act<T>::unpack2(mx).x;
      const bool finite = amax <= 3.4028234e38f;
      const float s = fmaxf(__fdiv_rn(amax, BITS == 8 ? 127.f : 7.f), 1e-8f);
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 p = Act<T>::unpack2(xw[e]);
        f[2 * e] = finite ? p.x : 0.f;
        f[2 * e + 1] = finite ? p.y : 0.f;
      }
      const uint2 codes = cache_codes<BITS>(f, s, both(finite ? __frcp_rn(s) : 0.f));
      const bool isk = h < a.c.n_kv;
      const long long r = row + ((long long)(isk ? h : h - a.c.n_kv) << a.c.shift);
      uint8_t* dst = reinterpret_cast<uint8_t*>(isk ? a.k_codes : a.v_codes) + r * (HD * BITS / 8) + c * BITS;
      if (BITS == 8) *reinterpret_cast<uint2*>(dst) = codes;
      else *reinterpret_cast<uint32_t*>(dst) = codes.x;
      if (c == 0) (isk ? a.k_steps : a.v_steps)[r] = finite ? s : __int_as_float(0x7fffffff);
    }
  }
}

template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(kCacheWarps * 32) cache_read_kernel(const __grid_constant__ CacheCopyArgs a) {
  constexpr int CH = HD / 8, HL = 32 / CH, UN = 4;
  pdl_entry();
  const int lane = threadIdx.x & 31, c = lane % CH;
  const long long tt = (long long)blockIdx.x * kCacheWarps + (threadIdx.x >> 5);
  if (tt >= a.tokens) return;
  const int t = (int)tt, heads = 2 * a.c.n_kv;
  const long long row = cache_place(a.c, a.cu, cache_seq(a.cu, a.c.n_seq, t), t);
  if (row < 0) return;
  for (int h0 = lane / CH; h0 < heads; h0 += UN * HL) {
    uint2 w[UN];
    float s[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u * HL;
      if (h >= heads) continue;
      const bool isk = h < a.c.n_kv;
      const long long r = row + ((long long)(isk ? h : h - a.c.n_kv) << a.c.shift);
      const uint8_t* src = reinterpret_cast<const uint8_t*>(isk ? a.k_codes : a.v_codes) + r * (HD * BITS / 8) + c * BITS;
      if (BITS == 8) w[u] = *reinterpret_cast<const uint2*>(src);
      else w[u] = make_uint2(*reinterpret_cast<const uint32_t*>(src), 0u);
      s[u] = (isk ? a.k_steps : a.v_steps)[r];
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u * HL;
      if (h >= heads) continue;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        int q;  // the code, sign-extended
        if (BITS == 8) q = (int)((e < 4 ? w[u].x : w[u].y) << (24 - 8 * (e % 4))) >> 24;
        else q = (int)(w[u].x << (28 - 4 * e)) >> 28;
        f[e] = (float)q * s[u];
      }
      T* dst = h < a.c.n_kv ? reinterpret_cast<T*>(a.k) + t * a.k_tok + h * a.k_head
                            : reinterpret_cast<T*>(a.v) + t * a.v_tok + (h - a.c.n_kv) * a.v_head;
      *reinterpret_cast<uint4*>(dst + 8 * c) = make_uint4(Act<T>::pack2(f[0], f[1]), Act<T>::pack2(f[2], f[3]),
                                                          Act<T>::pack2(f[4], f[5]), Act<T>::pack2(f[6], f[7]));
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
