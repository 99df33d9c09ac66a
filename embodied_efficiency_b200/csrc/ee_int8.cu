// ee_int8.cu -- C ABI: 8-bit integer linears with a scale for each token and
// each output channel,
//   y[m][n] = epi( (sum_k xq[m][k] * w[n][k]) * sx[m] * sw[n] + bias[n] ),
// and the token quantiser xq = rint(x / sx), sx = max(amax |x| / 127, 1e-8).
#include <atomic>
#include <cmath>

#include "ee_host.h"
#include "ee_int8_tc.cuh"

namespace ee {

// ---------------------------------------------------------------------------
// token quantiser
// ---------------------------------------------------------------------------
// W warps share a row; a lane keeps its first kQChunks 16-byte chunks in
// registers between the maximum and the rounding (longer rows read the rest
// again). The maximum is taken over the 15-bit magnitudes as integers, so an
// infinity or NaN wins it: such a token gets codes of 0 and a NaN scale.
constexpr int kQChunks = 8;
constexpr int kQThreads = 256;

// nearest integers (ties to even) of the fp32 quotients v / s of four values,
// one byte each: t = v * (1 / s) is within 1.5 ulp of the quotient, so only a t
// that close to a tie is divided for. In packed pairs, as the instructions per
// value, not the bytes, bound a long row otherwise.
EE_DEV uint32_t quant_word(uint64_t v01, uint64_t v23, float s, uint64_t inv2) {
  const uint64_t magic = both(12582912.f), back = both(-12582912.f);  // 1.5 * 2^23: the sum's rounding is rint(t)
  const uint64_t t01 = mul2f(v01, inv2), t23 = mul2f(v23, inv2);
  uint64_t r01 = add2f(t01, magic), r23 = add2f(t23, magic);
  // rint(t) - t, exact and at most 1/2
  const uint64_t d01 = fma2f(t01, both(-1.f), add2f(r01, back)), d23 = fma2f(t23, both(-1.f), add2f(r23, back));
  uint32_t d[4], b[4];
  unpack64(d01, d[0], d[1]);
  unpack64(d23, d[2], d[3]);
  const float far = fmaxf(fmaxf(fabsf(__uint_as_float(d[0])), fabsf(__uint_as_float(d[1]))),
                          fmaxf(fabsf(__uint_as_float(d[2])), fabsf(__uint_as_float(d[3]))));
  unpack64(r01, b[0], b[1]);
  unpack64(r23, b[2], b[3]);
  if (far > 0.49993896484375f) {  // 1/2 - 2^-14
    uint32_t v[4];
    unpack64(v01, v[0], v[1]);
    unpack64(v23, v[2], v[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fdiv_rn(__uint_as_float(v[e]), s) + 12582912.f);
  }
  return prmt(prmt(b[0], b[1], 0x0040u), prmt(b[2], b[3], 0x0040u), 0x5410u);
}

template <typename T, int W>
__global__ void __launch_bounds__(kQThreads) quantize_tokens_kernel(const T* __restrict__ x, int8_t* __restrict__ xq,
                                                                    float* __restrict__ sx, long long rows, int cols,
                                                                    long long ldx) {
  pdl_entry();
  constexpr int RPB = kQThreads / (32 * W);  // rows per CTA
  __shared__ uint32_t part[kQThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * RPB + warp / W;
  const bool live = row < rows;
  const int c0 = (warp % W) * 32 + lane, nch = cols >> 3;
  const T* xr = x + (live ? row : 0) * ldx;
  uint4 q[kQChunks];
  uint32_t mx = 0;
  auto magnitude = [&](const uint4& w) {
    mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu),
                               __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));  // of the two halves by themselves
  };
#pragma unroll
  for (int i = 0; i < kQChunks; ++i) {
    const int c = c0 + i * 32 * W;
    q[i] = c < nch && live ? *reinterpret_cast<const uint4*>(xr + 8 * c) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < kQChunks; ++i) magnitude(q[i]);
  if (live)
    for (int c = c0 + kQChunks * 32 * W; c < nch; c += 32 * W) magnitude(*reinterpret_cast<const uint4*>(xr + 8 * c));
  mx = __reduce_max_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16));
  if (W > 1) {
    if (lane == 0) part[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) mx = max(mx, part[warp / W * W + i]);
  }
  if (!live) return;
  const float amax = Act<T>::unpack2(mx).x;
  const bool finite = amax <= 3.4028234e38f;  // false for infinities and NaN
  const float s = fmaxf(__fdiv_rn(amax, 127.f), 1e-8f);
  const uint64_t inv2 = both(finite ? __frcp_rn(s) : 0.f);
  if (c0 == 0) sx[row] = finite ? s : __int_as_float(0x7fffffff);
  int8_t* qr = xq + row * cols;
  auto store = [&](const uint4& w, int c) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    uint32_t o[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 f = Act<T>::unpack2(ws[2 * h]), g = Act<T>::unpack2(ws[2 * h + 1]);
      o[h] = finite ? quant_word(pack64(__float_as_uint(f.x), __float_as_uint(f.y)),
                                 pack64(__float_as_uint(g.x), __float_as_uint(g.y)), s, inv2)
                    : 0u;
    }
    *reinterpret_cast<uint2*>(qr + 8 * c) = make_uint2(o[0], o[1]);
  };
#pragma unroll
  for (int i = 0; i < kQChunks; ++i) {
    const int c = c0 + i * 32 * W;
    if (c < nch) store(q[i], c);
  }
  for (int c = c0 + kQChunks * 32 * W; c < nch; c += 32 * W) store(*reinterpret_cast<const uint4*>(xr + 8 * c), c);
}

template <typename T>
static int launch_quantize(const T* x, int8_t* xq, float* sx, long long rows, int cols, long long ldx, cudaStream_t s) {
  // warps per row: enough that a row stays in registers (52224 x 2048: 54 us, 6.0 TB/s, with one; a fifth more with
  // two), and while the rows alone leave the GPU empty more of them, as long as each lane has a chunk (one row of 2048:
  // 3.6 us with one, 1.9 with four). In between a warp has one row and stops: 6528 x 2048 takes 10.4 us for 40 MB, 816
  // CTAs in 592 places with no next row in flight
  const int per = 32 * kQChunks, nch = cols / 8;
  int w = nch <= per ? 1 : (nch <= 2 * per ? 2 : (nch <= 4 * per ? 4 : 8));
  while (w < 8 && rows * w <= 8 * device_sms() && nch > 32 * w) w *= 2;
  const long long rpb = kQThreads / (32 * w);
  const dim3 grid((unsigned)((rows + rpb - 1) / rpb)), blk(kQThreads);
  cudaError_t e;
  if (w == 1) e = launch_pdl(quantize_tokens_kernel<T, 1>, grid, blk, 0, s, x, xq, sx, rows, cols, ldx);
  else if (w == 2) e = launch_pdl(quantize_tokens_kernel<T, 2>, grid, blk, 0, s, x, xq, sx, rows, cols, ldx);
  else if (w == 4) e = launch_pdl(quantize_tokens_kernel<T, 4>, grid, blk, 0, s, x, xq, sx, rows, cols, ldx);
  else e = launch_pdl(quantize_tokens_kernel<T, 8>, grid, blk, 0, s, x, xq, sx, rows, cols, ldx);
  return e == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------
constexpr unsigned long long kI8TimeoutNs = 1000000000ull;

int* gemm_status_ptr();  // ee_ops.cu: the status word of the GEMM kernels on the current device

template <typename T, bool GELU>
static int launch_pair(Int8Args a, const int8_t* xq, const int8_t* w, cudaStream_t s) {
  auto fn = int8_pair_kernel<T, GELU>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  const DevProps* dp = device_props();
  if (!dp) return EE_ERR_DEVICE;
  CUtensorMap tx, tw, ty{};
  if (!make_tmap_2d(&tx, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, a.K, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&tw, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.N, a.K, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      (a.vec && !make_tmap_2d(&ty, a.out, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, a.N, a.M, (uint64_t)a.N * 2, 64, 32,
                              CU_TENSOR_MAP_SWIZZLE_128B)))
    return EE_ERR_LAUNCH;
  a.tiles_m = (a.M + 255) / 256;
  a.tiles_n = (a.N + 255) / 256;
  const long long tiles = (long long)a.tiles_m * a.tiles_n;
  if (tiles > 0x7fffffff) return EE_ERR_SHAPE;
  const int pairs = (int)(tiles < dp->sms / 2 ? tiles : dp->sms / 2);
  return launch_pdl(fn, dim3(2 * pairs), dim3(kI8PairThreads), kI8PairSmem, s, tx, tw, ty, a) == cudaSuccess
             ? EE_OK
             : EE_ERR_LAUNCH;
}

// Ring stages of a CTA that takes kbc k-blocks. Clusters of 4 or 8 find room on
// the GPU at once when two CTAs share an SM (50 x 2048 x 8192: 19 us with rings
// of 200 KB, 10 with 100); alone or in pairs, CTAs are better off with the
// deeper ring (2000 x 1024 x 4096: 27 and 25)
template <int NT>
static int few_stages(int k, int split) {
  const int nkb = (k + 127) / 128, kbc = (nkb + split - 1) / split;
  const int fit = (int)((split >= 4 ? 100u : 200u) * 1024u / i8_few_stage<NT>());
  return kbc < fit ? kbc : fit;
}

template <typename T, int NT, bool GELU>
static int launch_few(Int8Args a, const int8_t* xq, const int8_t* w, int split, cudaStream_t s) {
  auto fn = int8_few_kernel<T, NT, GELU>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  CUtensorMap tx, tw;
  if (!make_tmap_2d(&tx, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, a.K, 128, NT, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tmap_2d(&tw, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.N, a.K, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return EE_ERR_LAUNCH;
  a.split = split;
  a.ns = few_stages<NT>(a.K, split);
  const size_t smem = i8_few_smem<NT>(a.ns);
  const long long units = (long long)((a.N + 127) / 128) * ((a.M + NT - 1) / NT);
  if (units * split > 0x7fffffff) return EE_ERR_SHAPE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * split));
  cfg.blockDim = dim3(kI8FewThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  unsigned int n = 1;
  add_pdl_attr(attr, n);
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, fn, tx, tw, a) == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}

// Which kernel: the token tile NT (0: the pair kernel) and the K split, by a
// cost in microseconds fitted to measurements of both kernels: a fixed part
// (launch, first loads, epilogue) and, per wave of CTAs and 128-byte k-block,
// the time its operands take to arrive. It tells 18 from 34 us (1000 x 4096 x
// 4096: pairs, few), 10 from 12 (1600 x 1024 x 1024: pairs, few), 16 from 10
// (512 x 1024 x 4096: pairs, few over 4 slices of K) and 10 from 9 (1023 x
// 1000 x 1040: 128-token tiles, 64-token tiles).
struct Int8Plan { int nt, split; };
static Int8Plan int8_plan(int m, int n, int k, int sms) {
  const int nkb = (k + 127) / 128, tiles_n = (n + 127) / 128;
  auto waves = [](double items, double slots) { return std::ceil(items / slots); };
  Int8Plan best{0, 1};
  double cost = 7.4 + 0.275 * nkb * waves(std::ceil(m / 256.0) * std::ceil(n / 256.0), sms / 2);
  if (m <= 64) cost = 1e30;  // a quarter of a pair's tokens or fewer: the other kernel's tiles fit
  static const struct { int nt; double fixed; } tiles[4] = {{16, 5.4}, {32, 6.3}, {64, 7.2}, {128, 8.3}};
  for (const auto& t : tiles) {
    const double units = (double)tiles_n * std::ceil(m / (double)t.nt), per = 0.28 * (16 + t.nt / 8.0) / 32;
    for (int s = 1; s <= 8 && s <= nkb && (s == 1 || units * s <= sms); s *= 2) {
      const double c = t.fixed + (s > 1 ? 0.4 : 0.0) + per * waves(units * s, sms) * ((nkb + s - 1) / s);
      if (c < cost) {
        cost = c;
        best = {t.nt, s};
      }
    }
  }
  return best;
}

// shared memory that a CTA of the plan asks for
static size_t int8_plan_smem(const Int8Plan& p, int k) {
  switch (p.nt) {
    case 16: return i8_few_smem<16>(few_stages<16>(k, p.split));
    case 32: return i8_few_smem<32>(few_stages<32>(k, p.split));
    case 64: return i8_few_smem<64>(few_stages<64>(k, p.split));
    case 128: return i8_few_smem<128>(few_stages<128>(k, p.split));
  }
  return kI8PairSmem;
}

template <typename T, bool GELU>
static int launch_int8_g(const Int8Args& a, const int8_t* xq, const int8_t* w, cudaStream_t s) {
  const Int8Plan p = int8_plan(a.M, a.N, a.K, device_sms());
  switch (p.nt) {
    case 16: return launch_few<T, 16, GELU>(a, xq, w, p.split, s);
    case 32: return launch_few<T, 32, GELU>(a, xq, w, p.split, s);
    case 64: return launch_few<T, 64, GELU>(a, xq, w, p.split, s);
    case 128: return launch_few<T, 128, GELU>(a, xq, w, p.split, s);
  }
  return launch_pair<T, GELU>(a, xq, w, s);
}
template <typename T>
static int launch_int8(const Int8Args& a, const int8_t* xq, const int8_t* w, cudaStream_t s) {
  return (a.epi & I8_GELU) ? launch_int8_g<T, true>(a, xq, w, s) : launch_int8_g<T, false>(a, xq, w, s);
}

static int check_product(const void* weight, const void* w_scales, const void* bias, const void* residual, void* y,
                         int64_t m, int64_t n, int64_t k, int32_t scale_dtype, int32_t act_dtype, int32_t epilogue) {
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  if (scale_dtype != EE_F32 && scale_dtype != EE_F16) return EE_ERR_DTYPE;
  if ((epilogue & ~(EE_EPI_BIAS | EE_EPI_GELU | EE_EPI_RESIDUAL)) != 0) return EE_ERR_ARG;
  if ((epilogue & EE_EPI_GELU) && (epilogue & EE_EPI_RESIDUAL)) return EE_ERR_ARG;
  // an int32 sum holds 131071 products of two codes (2^31 / 2^14)
  if (m < 0 || n < 0 || k < 16 || (k % 16) != 0 || k > 131056 || m > 0x7fffff00 || n > 0x7fffff00) return EE_ERR_SHAPE;
  if (m == 0 || n == 0) return EE_OK;
  if (!weight || !w_scales || !y) return EE_ERR_ARG;
  if (((epilogue & EE_EPI_BIAS) && !bias) || ((epilogue & EE_EPI_RESIDUAL) && !residual)) return EE_ERR_ARG;
  if (!aligned16(weight) || !aligned16(y) || !aligned16(w_scales) || (bias && !aligned16(bias)) ||
      (residual && !aligned16(residual)))
    return EE_ERR_ALIGN;
  return EE_OK;
}

static int int8_product(const int8_t* xq, const float* sx, const void* weight, const void* w_scales, const void* bias,
                        const void* residual, void* y, int64_t m, int64_t n, int64_t k, int32_t scale_dtype,
                        int32_t act_dtype, int32_t epilogue, bool early, cudaStream_t s) {
  Int8Args a{};
  a.sx = sx;
  a.sw = w_scales;
  a.bias = bias; a.resid = residual; a.out = y;
  a.M = (int)m; a.N = (int)n; a.K = (int)k;
  a.sw_f16 = scale_dtype == EE_F16;
  a.epi = epilogue;
  a.vec = n % 8 == 0;
  a.early = early && EE_PDL;
  a.status = gemm_status_ptr();
  a.timeout_ns = kI8TimeoutNs;
  if (!a.status) return EE_ERR_DEVICE;
  const int8_t* w = reinterpret_cast<const int8_t*>(weight);
  return act_dtype == EE_BF16 ? launch_int8<__nv_bfloat16>(a, xq, w, s) : launch_int8<__half>(a, xq, w, s);
}

}  // namespace ee

using namespace ee;

extern "C" {

int ee_quantize_tokens(const void* x, int64_t ldx, int8_t* xq, float* x_scales, int64_t m, int64_t k,
                       int32_t act_dtype, ee_stream_t stream) {
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  if (m < 0 || m > 0x7fffff00 || k < 16 || (k % 16) != 0 || k > 131056 || ldx < k || (ldx % 8) != 0)
    return EE_ERR_SHAPE;
  if (m == 0) return EE_OK;
  if (!x || !xq || !x_scales) return EE_ERR_ARG;
  if (!aligned16(x) || !aligned16(xq) || !aligned16(x_scales)) return EE_ERR_ALIGN;
  const int rc = check_device();
  if (rc) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  return act_dtype == EE_BF16
             ? launch_quantize(reinterpret_cast<const __nv_bfloat16*>(x), xq, x_scales, m, (int)k, ldx, s)
             : launch_quantize(reinterpret_cast<const __half*>(x), xq, x_scales, m, (int)k, ldx, s);
}

int ee_int8_gemm(const int8_t* xq, const float* x_scales, const void* weight, const void* w_scales, const void* bias,
                 const void* residual, void* y, int64_t m, int64_t n, int64_t k, int32_t scale_dtype,
                 int32_t act_dtype, int32_t epilogue, ee_stream_t stream) {
  int rc = check_product(weight, w_scales, bias, residual, y, m, n, k, scale_dtype, act_dtype, epilogue);
  if (rc || m == 0 || n == 0) return rc;
  if (!xq || !x_scales) return EE_ERR_ARG;
  if (!aligned16(xq) || !aligned16(x_scales)) return EE_ERR_ALIGN;
  rc = check_device();
  if (rc) return rc;
  return int8_product(xq, x_scales, weight, w_scales, bias, residual, y, m, n, k, scale_dtype, act_dtype, epilogue,
                      false, (cudaStream_t)stream);
}

int ee_int8_plan(int64_t m, int64_t n, int64_t k, int32_t sms, int32_t* tokens, int32_t* ctas, size_t* smem_bytes) {
  if (!tokens || !ctas || !smem_bytes || sms < 2) return EE_ERR_ARG;
  if (m < 1 || n < 1 || k < 16 || (k % 16) != 0 || k > 131056 || m > 0x7fffff00 || n > 0x7fffff00) return EE_ERR_SHAPE;
  const Int8Plan p = int8_plan((int)m, (int)n, (int)k, sms);
  *tokens = p.nt ? p.nt : 256;
  *ctas = p.nt ? p.split : 2;
  *smem_bytes = int8_plan_smem(p, (int)k);
  return EE_OK;
}

size_t ee_int8_linear_workspace_bytes(int64_t m, int64_t k) {
  if (m < 0 || k < 0 || m > 0x7fffff00 || k > 131056) return 0;
  return (((size_t)m * (size_t)k + 15) & ~(size_t)15) + (size_t)m * 4;
}

int ee_int8_linear(const void* x, int64_t ldx, const void* weight, const void* w_scales, const void* bias,
                   const void* residual, void* y, void* workspace, size_t workspace_bytes, int64_t m, int64_t n,
                   int64_t k, int32_t scale_dtype, int32_t act_dtype, int32_t epilogue, ee_stream_t stream) {
  int rc = check_product(weight, w_scales, bias, residual, y, m, n, k, scale_dtype, act_dtype, epilogue);
  if (rc || m == 0 || n == 0) return rc;
  if (!workspace || workspace_bytes < ee_int8_linear_workspace_bytes(m, k)) return EE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return EE_ERR_ALIGN;
  int8_t* xq = reinterpret_cast<int8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(xq + (((size_t)m * (size_t)k + 15) & ~(size_t)15));
  rc = ee_quantize_tokens(x, ldx, xq, sx, m, k, act_dtype, stream);
  if (rc) return rc;
  // the quantiser starts after everything before it, so the weights are final while it runs
  return int8_product(xq, sx, weight, w_scales, bias, residual, y, m, n, k, scale_dtype, act_dtype, epilogue, true,
                      (cudaStream_t)stream);
}

}  // extern "C"
