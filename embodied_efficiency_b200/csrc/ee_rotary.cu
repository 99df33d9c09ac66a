// ee_rotary.cu -- C ABI: rotary positions with up to four axes (time, height,
// width, ...) applied to the query and key heads of packed tokens.
//
// Pair i of a head (elements i and i + hd/2, or 2i and 2i + 1 interleaved)
// turns by pos[axis(i)][token] * base^(-2i / hd). The table holds each
// frequency as a 64-bit fraction of a turn, F = round(freq / 2 pi * 2^64), so
// pos * F modulo 2^64 is the angle's fraction of a turn, at most |pos| * 2^-65
// turns off if F is the rounded value (more digits than a double has): whole
// turns drop out in the integer multiply instead of costing the float angle its
// low bits at far positions. Its top 32 bits, as an fp32 value of [-1, 1) half
// turns, add 2^-25 of those.
//
// HBM-bound: every value is read and written once (4 bytes), the angles are
// hd/2 sine / cosine pairs per token shared by all its heads. One warp per
// token: each lane evaluates hd/64 pairs, the warp exchanges them by
// shuffles, and a lane then turns the same 8 pairs of every head it visits
// (two 16-byte loads and stores per head, three heads in flight: with four the
// registers leave 5 CTAs an SM and 71 us instead of 65 for the case below).
// Measured: 65537 tokens, 16 + 8 heads of 64: 65 us, 6.2 TB/s, 0.94 of the
// copy rate; 6528 tokens, 16 + 16 heads of 128: 17 us.
#include <type_traits>

#include "ee_common.cuh"
#include "ee_host.h"

namespace ee {

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  const void* pos;                     // [axes][tokens]
  const unsigned long long* freqs;     // [hd / 2] fractions of a turn per position
  long long q_tok, q_head, k_tok, k_head, qo_tok, qo_head, ko_tok, ko_head;  // strides, elements
  long long pos_axis, tokens;
  int n_q, n_kv;
  int end0, end1, end2;                // pairs below end0: axis 0, below end1: axis 1, ...
  int pos64, interleaved;
};

constexpr int kRotWarps = 4;

template <typename T, int HD>
__global__ void __launch_bounds__(kRotWarps * 32) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int HALF = HD / 2, CH = HALF / 8;  // 8-pair chunks per head
  constexpr int HL = 32 / CH;                  // heads a warp turns at once
  constexpr int PP = HALF >= 32 ? HALF / 32 : 1;
  pdl_entry();
  const int lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  // this lane's pairs lane * PP ..
  float sn[PP], cs[PP];
#pragma unroll
  for (int p = 0; p < PP; ++p) {
    const int i = lane * PP + p;
    sn[p] = 0.f;
    cs[p] = 1.f;
    if (i < HALF) {
      const int axis = i < a.end0 ? 0 : (i < a.end1 ? 1 : (i < a.end2 ? 2 : 3));
      const long long at = axis * a.pos_axis + t;
      const long long pos = a.pos64 ? __ldg(reinterpret_cast<const long long*>(a.pos) + at)
                                    : (long long)__ldg(reinterpret_cast<const int*>(a.pos) + at);
      const unsigned long long turn = (unsigned long long)pos * __ldg(a.freqs + i);
      // the top 32 bits, signed: the angle in [-1, 1) half turns
      sincospif((float)(int)(turn >> 32) * 4.656612873077393e-10f, &sn[p], &cs[p]);
    }
  }
  const int c = lane % CH;
  float sv[8], cv[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int src = (8 * c + e) / PP;
    if (PP == 1) {
      sv[e] = __shfl_sync(0xffffffffu, sn[0], src);
      cv[e] = __shfl_sync(0xffffffffu, cs[0], src);
    } else {
      sv[e] = __shfl_sync(0xffffffffu, sn[e % PP], src);
      cv[e] = __shfl_sync(0xffffffffu, cs[e % PP], src);
    }
  }
  const int lo = a.interleaved ? 16 * c : 8 * c, hi = a.interleaved ? lo + 8 : lo + HALF;
  const int heads = a.n_q + a.n_kv;
  auto turn_heads = [&](int h0, auto un) {
    constexpr int UN = decltype(un)::value;
    uint4 x[UN], y[UN];
    T* dst[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int h = h0 + u * HL;
      if (h < heads) {
        const bool isq = h < a.n_q;
        const T* src = isq ? reinterpret_cast<const T*>(a.q) + t * a.q_tok + h * a.q_head
                           : reinterpret_cast<const T*>(a.k) + t * a.k_tok + (h - a.n_q) * a.k_head;
        dst[u] = isq ? reinterpret_cast<T*>(a.qo) + t * a.qo_tok + h * a.qo_head
                     : reinterpret_cast<T*>(a.ko) + t * a.ko_tok + (h - a.n_q) * a.ko_head;
        x[u] = *reinterpret_cast<const uint4*>(src + lo);
        y[u] = *reinterpret_cast<const uint4*>(src + hi);
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (h0 + u * HL >= heads) continue;
      const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, yw[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
      uint32_t xo[4], yo[4];
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Act<T>::unpack2(xw[e]), g = Act<T>::unpack2(yw[e]);
          xo[e] = Act<T>::pack2(f.x * cv[e] - f.y * sv[e], f.x * sv[e] + f.y * cv[e]);
          yo[e] = Act<T>::pack2(g.x * cv[4 + e] - g.y * sv[4 + e], g.x * sv[4 + e] + g.y * cv[4 + e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Act<T>::unpack2(xw[e]), g = Act<T>::unpack2(yw[e]);
          xo[e] = Act<T>::pack2(f.x * cv[2 * e] - g.x * sv[2 * e], f.y * cv[2 * e + 1] - g.y * sv[2 * e + 1]);
          yo[e] = Act<T>::pack2(f.x * sv[2 * e] + g.x * cv[2 * e], f.y * sv[2 * e + 1] + g.y * cv[2 * e + 1]);
        }
      }
      *reinterpret_cast<uint4*>(dst[u] + lo) = make_uint4(xo[0], xo[1], xo[2], xo[3]);
      *reinterpret_cast<uint4*>(dst[u] + hi) = make_uint4(yo[0], yo[1], yo[2], yo[3]);
    }
  };
  for (int h0 = lane / CH; h0 < heads; h0 += 3 * HL) turn_heads(h0, std::integral_constant<int, 3>{});
}

template <typename T>
static int launch_rotary(const RotaryArgs& a, int hd, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.tokens + kRotWarps - 1) / kRotWarps);
  cudaError_t e = cudaErrorInvalidValue;
  switch (hd) {
    case 32: e = launch_pdl(rotary_kernel<T, 32>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
    case 64: e = launch_pdl(rotary_kernel<T, 64>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
    case 128: e = launch_pdl(rotary_kernel<T, 128>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
    case 256: e = launch_pdl(rotary_kernel<T, 256>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
  }
  return e == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}

}  // namespace ee

using namespace ee;

extern "C" int ee_rotary(const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok, int64_t qo_head,
                         const void* k, int64_t k_tok, int64_t k_head, void* k_out, int64_t ko_tok, int64_t ko_head,
                         const void* positions, int64_t pos_axis, int32_t pos_bits, const uint64_t* freqs,
                         int64_t tokens, int32_t n_q, int32_t n_kv, int32_t head_dim, const int32_t* sections,
                         int32_t n_axes, int32_t interleaved, int32_t act_dtype, ee_stream_t stream) {
  if (!sections || n_axes < 1 || n_axes > 4 || tokens < 0 || n_q < 0 || n_kv < 0) return EE_ERR_ARG;
  if (pos_bits != 32 && pos_bits != 64) return EE_ERR_ARG;
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return EE_ERR_UNSUPPORTED;
  long long sum = 0;
  for (int i = 0; i < n_axes; ++i) {
    if (sections[i] < 0) return EE_ERR_SHAPE;
    sum += sections[i];
  }
  if (sum != head_dim / 2 || tokens > (long long)kRotWarps * 0x7fffffff) return EE_ERR_SHAPE;
  if (tokens == 0 || n_q + (long long)n_kv == 0) return EE_OK;
  if (n_q + (long long)n_kv > 65536) return EE_ERR_SHAPE;
  if (!positions || !freqs || (n_q && (!q || !q_out)) || (n_kv && (!k || !k_out))) return EE_ERR_ARG;
  if ((n_q && (!aligned16(q) || !aligned16(q_out))) || (n_kv && (!aligned16(k) || !aligned16(k_out))))
    return EE_ERR_ALIGN;
  if (((uintptr_t)positions & (pos_bits / 8 - 1)) || ((uintptr_t)freqs & 7)) return EE_ERR_ALIGN;
  const int64_t strides[8] = {q_tok, q_head, qo_tok, qo_head, k_tok, k_head, ko_tok, ko_head};
  for (int i = 0; i < 8; ++i)
    if ((i < 4 ? n_q : n_kv) && (strides[i] % 8) != 0) return EE_ERR_ALIGN;
  const int rc = check_device();
  if (rc) return rc;
  RotaryArgs a{};
  a.q = q; a.k = k; a.qo = q_out; a.ko = k_out;
  a.pos = positions;
  a.freqs = reinterpret_cast<const unsigned long long*>(freqs);
  a.q_tok = q_tok; a.q_head = q_head; a.qo_tok = qo_tok; a.qo_head = qo_head;
  a.k_tok = k_tok; a.k_head = k_head; a.ko_tok = ko_tok; a.ko_head = ko_head;
  a.pos_axis = pos_axis;
  a.tokens = tokens;
  a.n_q = n_q; a.n_kv = n_kv;
  a.end0 = sections[0];
  a.end1 = n_axes > 1 ? a.end0 + sections[1] : 0x7fffffff;
  a.end2 = n_axes > 2 ? a.end1 + sections[2] : 0x7fffffff;
  if (n_axes == 1) a.end0 = 0x7fffffff;
  a.pos64 = pos_bits == 64;
  a.interleaved = interleaved != 0;
  cudaStream_t s = (cudaStream_t)stream;
  return act_dtype == EE_BF16 ? launch_rotary<__nv_bfloat16>(a, head_dim, s) : launch_rotary<__half>(a, head_dim, s);
}
