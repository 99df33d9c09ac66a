// ee_rotary.cu -- C ABI: rotary positions with up to four axes (time, height,
// width, ...) applied to the query and key heads of packed tokens, by
// themselves (ee_rotary) or after an RMS norm of each head (ee_norm_rotary).
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
//
// The norm, y = w x / sqrt(mean(x^2) + eps), is taken in fp32 on the 8 values that
// a lane of norm_rotary_kernel holds of a head, their squares summed over the
// head's hd / 8 lanes by shuffles: one rounding, at the end, and no pass of its
// own.
#include <cfloat>
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
  const void *qw, *kw;                 // norm: weights [hd] of the query and key heads
  int w32;                             // they are fp32, not of the act dtype
  float eps;
};

constexpr int kRotWarps = 4;

// four weights as fp32
template <typename T>
EE_DEV void norm_weights(const void* w, int w32, int at, float (&r)[4]) {
  if (w32) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + at));
    r[0] = x.x; r[1] = x.y; r[2] = x.z; r[3] = x.w;
  } else {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(w) + at));
    const float2 f = Act<T>::unpack2(x.x), g = Act<T>::unpack2(x.y);
    r[0] = f.x; r[1] = f.y; r[2] = g.x; r[3] = g.y;
  }
}

// Sines and cosines of token t's pairs N c .. N c + N - 1, c = lane % (hd / 2 N):
// each lane evaluates hd / 64 pairs, the warp exchanges them.
template <int HD, int N>
EE_DEV void rotary_angles(const RotaryArgs& a, long long t, float (&sv)[N], float (&cv)[N]) {
  constexpr int HALF = HD / 2, CH = HALF / N, PP = HALF >= 32 ? HALF / 32 : 1;
  const int lane = threadIdx.x & 31;
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
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int src = (N * c + e) / PP;
    if (PP == 1) {
      sv[e] = __shfl_sync(0xffffffffu, sn[0], src);
      cv[e] = __shfl_sync(0xffffffffu, cs[0], src);
    } else {
      sv[e] = __shfl_sync(0xffffffffu, sn[e % PP], src);
      cv[e] = __shfl_sync(0xffffffffu, cs[e % PP], src);
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kRotWarps * 32) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int HALF = HD / 2, CH = HALF / 8;  // 8-pair chunks per head
  constexpr int HL = 32 / CH;                  // heads a warp turns at once
  pdl_entry();
  const int lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const int c = lane % CH;
  float sv[8], cv[8];
  rotary_angles<HD, 8>(a, t, sv, cv);
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

// The same behind a norm of each head. Queries and keys by turns, as their
// weights differ, the weights multiplied into the turn's coefficients once for a
// token. A lane has four pairs of a head (8-byte loads): with eight, as above,
// the coefficients leave 20 warps an SM and 80 us where these took 69 (65537
// tokens, 16 + 8 heads of 64, the same ones again and again; 75 us on tensors
// that change from call to call, 5.4 TB/s); UN passes of HL heads are in flight.
template <typename T, int HD>
__global__ void __launch_bounds__(kRotWarps * 32, 8) norm_rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int HALF = HD / 2, CH = HALF / 4, HL = 32 / CH, UN = 4;
  pdl_entry();
  const int lane = threadIdx.x & 31, c = lane % CH;
  const long long t = (long long)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const int lo = a.interleaved ? 8 * c : 4 * c, hi = a.interleaved ? lo + 4 : lo + HALF;
  float sv[4], cv[4];
  bool angles = false;
  auto pair = [](float u, float v) { return pack64(__float_as_uint(u), __float_as_uint(v)); };
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {  // queries, keys
    const int heads = part ? a.n_kv : a.n_q;
    const long long head = part ? a.k_head : a.q_head, out_head = part ? a.ko_head : a.qo_head;
    const T* src = reinterpret_cast<const T*>(part ? a.k : a.q) + t * (part ? a.k_tok : a.q_tok) + (lane / CH) * head;
    T* dst = reinterpret_cast<T*>(part ? a.ko : a.qo) + t * (part ? a.ko_tok : a.qo_tok) + (lane / CH) * out_head;
    // the turn with the weights in it, for two values of x or y at once: x' = x A + x~ B, y' = y D + y~ C, where x~ is y
    // and the other way round, or (interleaved) the neighbour
    uint64_t A[2], B[2], C[2], D[2];
#pragma unroll 1
    for (int h0 = 0; h0 < heads; h0 += UN * HL) {
      uint2 x[UN], y[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        x[u] = y[u] = make_uint2(0, 0);
        if (h0 + u * HL + lane / CH < heads) {
          x[u] = *reinterpret_cast<const uint2*>(src + lo);
          y[u] = *reinterpret_cast<const uint2*>(src + hi);
        }
        src += HL * head;
      }
      if (h0 == 0) {  // under the first loads
        float wl[4], wh[4];
        norm_weights<T>(part ? a.kw : a.qw, a.w32, lo, wl);
        norm_weights<T>(part ? a.kw : a.qw, a.w32, hi, wh);
        if (!angles) rotary_angles<HD, 4>(a, t, sv, cv);
        angles = true;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (a.interleaved) {
            A[e] = pair(wl[2 * e] * cv[e], wl[2 * e + 1] * cv[e]);
            B[e] = pair(-wl[2 * e + 1] * sv[e], wl[2 * e] * sv[e]);
            D[e] = pair(wh[2 * e] * cv[2 + e], wh[2 * e + 1] * cv[2 + e]);
            C[e] = pair(-wh[2 * e + 1] * sv[2 + e], wh[2 * e] * sv[2 + e]);
          } else {
            A[e] = pair(wl[2 * e] * cv[2 * e], wl[2 * e + 1] * cv[2 * e + 1]);
            B[e] = pair(-wh[2 * e] * sv[2 * e], -wh[2 * e + 1] * sv[2 * e + 1]);
            D[e] = pair(wh[2 * e] * cv[2 * e], wh[2 * e + 1] * cv[2 * e + 1]);
            C[e] = pair(wl[2 * e] * sv[2 * e], wl[2 * e + 1] * sv[2 * e + 1]);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        if (h0 + u * HL >= heads) break;
        const uint32_t xw[2] = {x[u].x, x[u].y}, yw[2] = {y[u].x, y[u].y};
        uint64_t f[2], g[2], sum2 = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 p = Act<T>::unpack2(xw[e]), q = Act<T>::unpack2(yw[e]);
          f[e] = pair(p.x, p.y);
          g[e] = pair(q.x, q.y);
          sum2 = fma2f(f[e], f[e], fma2f(g[e], g[e], sum2));
        }
        uint32_t s0, s1;
        unpack64(sum2, s0, s1);
        float sum = __uint_as_float(s0) + __uint_as_float(s1);
#pragma unroll
        for (int o = 1; o < CH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        float r;  // the mean is at least eps, no subnormal number
        asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(sum, 1.f / HD, a.eps)));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f[e] = mul2f(f[e], both(r));
          g[e] = mul2f(g[e], both(r));
        }
        uint32_t xo[2], yo[2];
        auto turned = [&](uint64_t own, uint64_t other, uint64_t c1, uint64_t c2) {
          uint32_t u0, u1;
          unpack64(fma2f(own, c1, mul2f(other, c2)), u0, u1);
          return Act<T>::pack2(__uint_as_float(u0), __uint_as_float(u1));
        };
        if (a.interleaved) {
          auto swapped = [](uint64_t v) {
            uint32_t u0, u1;
            unpack64(v, u0, u1);
            return pack64(u1, u0);
          };
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            xo[e] = turned(f[e], swapped(f[e]), A[e], B[e]);
            yo[e] = turned(g[e], swapped(g[e]), D[e], C[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            xo[e] = turned(f[e], g[e], A[e], B[e]);
            yo[e] = turned(g[e], f[e], D[e], C[e]);
          }
        }
        if (h0 + u * HL + lane / CH < heads) {
          *reinterpret_cast<uint2*>(dst + lo) = make_uint2(xo[0], xo[1]);
          *reinterpret_cast<uint2*>(dst + hi) = make_uint2(yo[0], yo[1]);
        }
        dst += HL * out_head;
      }
    }
  }
}

template <typename T, bool NORM>
static int launch_rotary(const RotaryArgs& a, int hd, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.tokens + kRotWarps - 1) / kRotWarps);
  cudaError_t e = cudaErrorInvalidValue;
  switch (hd) {
    case 32: e = launch_pdl(NORM ? norm_rotary_kernel<T, 32> : rotary_kernel<T, 32>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
    case 64: e = launch_pdl(NORM ? norm_rotary_kernel<T, 64> : rotary_kernel<T, 64>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
    case 128: e = launch_pdl(NORM ? norm_rotary_kernel<T, 128> : rotary_kernel<T, 128>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
    case 256: e = launch_pdl(NORM ? norm_rotary_kernel<T, 256> : rotary_kernel<T, 256>, dim3(grid), dim3(kRotWarps * 32), 0, s, a); break;
  }
  return e == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}

}  // namespace ee

using namespace ee;

static int rotary(const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok, int64_t qo_head,
                  const void* k, int64_t k_tok, int64_t k_head, void* k_out, int64_t ko_tok, int64_t ko_head,
                  const void* positions, int64_t pos_axis, int32_t pos_bits, const uint64_t* freqs, int64_t tokens,
                  int32_t n_q, int32_t n_kv, int32_t head_dim, const int32_t* sections, int32_t n_axes,
                  int32_t interleaved, int32_t act_dtype, bool norm, const void* q_weight, const void* k_weight,
                  int32_t weight_dtype, float eps, cudaStream_t s) {
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
  if (norm) {
    if (weight_dtype != EE_F32 && weight_dtype != act_dtype) return EE_ERR_DTYPE;
    if (!(eps >= FLT_MIN) || !(eps <= FLT_MAX)) return EE_ERR_ARG;
    if ((n_q && !q_weight) || (n_kv && !k_weight)) return EE_ERR_ARG;
    if ((n_q && !aligned16(q_weight)) || (n_kv && !aligned16(k_weight))) return EE_ERR_ALIGN;
  }
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
  if (norm) {
    a.qw = q_weight; a.kw = k_weight;
    a.w32 = weight_dtype == EE_F32;
    a.eps = eps;
    return act_dtype == EE_BF16 ? launch_rotary<__nv_bfloat16, true>(a, head_dim, s)
                                : launch_rotary<__half, true>(a, head_dim, s);
  }
  return act_dtype == EE_BF16 ? launch_rotary<__nv_bfloat16, false>(a, head_dim, s)
                              : launch_rotary<__half, false>(a, head_dim, s);
}

extern "C" {

int ee_rotary(const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok, int64_t qo_head, const void* k,
              int64_t k_tok, int64_t k_head, void* k_out, int64_t ko_tok, int64_t ko_head, const void* positions,
              int64_t pos_axis, int32_t pos_bits, const uint64_t* freqs, int64_t tokens, int32_t n_q, int32_t n_kv,
              int32_t head_dim, const int32_t* sections, int32_t n_axes, int32_t interleaved, int32_t act_dtype,
              ee_stream_t stream) {
  return rotary(q, q_tok, q_head, q_out, qo_tok, qo_head, k, k_tok, k_head, k_out, ko_tok, ko_head, positions, pos_axis,
                pos_bits, freqs, tokens, n_q, n_kv, head_dim, sections, n_axes, interleaved, act_dtype, false, nullptr,
                nullptr, 0, 0.f, (cudaStream_t)stream);
}

int ee_norm_rotary(const void* q, int64_t q_tok, int64_t q_head, void* q_out, int64_t qo_tok, int64_t qo_head,
                   const void* k, int64_t k_tok, int64_t k_head, void* k_out, int64_t ko_tok, int64_t ko_head,
                   const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps, const void* positions,
                   int64_t pos_axis, int32_t pos_bits, const uint64_t* freqs, int64_t tokens, int32_t n_q, int32_t n_kv,
                   int32_t head_dim, const int32_t* sections, int32_t n_axes, int32_t interleaved, int32_t act_dtype,
                   ee_stream_t stream) {
  return rotary(q, q_tok, q_head, q_out, qo_tok, qo_head, k, k_tok, k_head, k_out, ko_tok, ko_head, positions, pos_axis,
                pos_bits, freqs, tokens, n_q, n_kv, head_dim, sections, n_axes, interleaved, act_dtype, true, q_weight,
                k_weight, weight_dtype, eps, (cudaStream_t)stream);
}

}  // extern "C"
