// ee_int8_tc.cuh -- the 8-bit integer product on the 5th-generation tensor
// cores (tcgen05.mma kind::i8: int8 x int8, exact int32 sums in TMEM).
//
//   y[m][n] = epi( (sum_k xq[m][k] * w[n][k]) * sx[m] * sw[n] + bias[n] )
//
// Both operands are K-major rows of bytes, so a 128-byte swizzled line holds
// 128 k and one MMA takes 32 of them. Bytes past K, M or N are zero-filled by
// the TMA loads: the sums are exact at any size.
//
// Two kernels, by how much there is to do (int8_plan in ee_int8.cu):
//   int8_pair_kernel  many tokens: persistent CTA pairs, 256 x 256 outputs
//                     per pair (cta_group::2), bound by the tensor cores
//   int8_few_kernel   few tokens: weight rows as the MMA's 128 lanes, K split
//                     over a cluster, bound by the weights' bytes and latency
#pragma once

#include "ee_common.cuh"
#include "ee_tma.cuh"
#include "ee_umma.cuh"

namespace ee {

struct Int8Args {
  const float* sx;       // [M]
  const void* sw;        // [N] fp32 or fp16
  const void *bias, *resid;
  void* out;
  int M, N, K;
  int sw_f16, epi;
  int vec;               // N % 8 == 0: rows of 16-byte pieces
  int tiles_m, tiles_n;  // pair kernel: 256 x 256 output tiles
  int split, ns;         // few kernel: CTAs per cluster (K slices), ring stages
  int* status;
  unsigned long long timeout_ns;
};
enum { I8_BIAS = 1, I8_GELU = 2, I8_RESID = 4 };

// kind::i8 instruction descriptor: D int32 (2 in bits [4,6)), A and B signed
// 8-bit (1 in bits [7,10) and [10,13)), both K-major, N >> 3, M >> 4.
__host__ __device__ constexpr uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int CG>
EE_DEV void umma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

EE_DEV float i8_wscale(const Int8Args& a, int n) {
  return a.sw_f16 ? __half2float(__ldg(reinterpret_cast<const __half*>(a.sw) + n))
                  : __ldg(reinterpret_cast<const float*>(a.sw) + n);
}

// GELU(z) = max(z, 0) - |z| Phi(-|z|), with Phi(-a) = e^(-a^2/2) t P(t),
// t = 1 / (1 + 0.35 a): Hastings' form, its degree-7 polynomial fitted here
// by weighted minimax (|error| of Phi below 4e-8, relative below 4e-6). About
// 16 instructions, where erff costs twice that: the epilogue of a 256 x 256
// tile has to keep up with the tensor cores.
EE_DEV float i8_gelu(float z) {
  const float a = fabsf(z);
  float t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.35f, a, 1.f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * z * -0.72134752f));
  float p = fmaf(t, 0.044615f, -0.18442732f);
  p = fmaf(t, p, 0.21107948f);
  p = fmaf(t, p, 0.00892954f);
  p = fmaf(t, p, 0.14315536f);
  p = fmaf(t, p, 0.13687154f);
  p = fmaf(t, p, 0.13977644f);
  return fmaf(-fminf(a, 3.0e38f), p * t * e, fmaxf(z, 0.f));  // the fminf: 0 instead of inf * 0
}

// ---------------------------------------------------------------------------
// pair primitives (cta_group::2)
// ---------------------------------------------------------------------------
EE_DEV void tmem_alloc2(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
EE_DEV void tmem_dealloc2(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// arrive on the barrier at this shared-memory offset in both CTAs of the pair
// when the pair MMAs issued so far have completed
EE_DEV void umma_commit2(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((unsigned short)3)
      : "memory");
}
// 2-D tiled TMA load into this CTA's shared memory, completing on an mbarrier
// of either CTA of the pair (a shared::cluster address)
EE_DEV void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
EE_DEV void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
EE_DEV void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
EE_DEV void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
EE_DEV void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
EE_DEV void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
EE_DEV void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// ---------------------------------------------------------------------------
// many tokens
// ---------------------------------------------------------------------------
// A pair's tile is 256 tokens x 256 features: each CTA holds 128 token rows
// (the MMA's A) and 128 weight rows (half of B) per 128-byte k-block, 32 KB a
// stage, so a k-block's 512 MMA cycles take 64 bytes a cycle from L2 -- half
// of what one CTA alone would need for 128 x 256. Roles (10 warps): TMA
// producer, MMA issuer (the pair's first CTA issues for both), eight epilogue
// warps. Two accumulators of 256 TMEM columns, so a tile's epilogue runs under
// the next tile's MMAs. Outputs are staged as swizzled [32 rows][64 columns]
// blocks and stored by TMA.
constexpr int kI8Stages = 5;
constexpr int kI8EpiWarps = 8;
constexpr int kI8PairThreads = 32 * (2 + kI8EpiWarps);
constexpr uint32_t kI8Stage = 32768;
constexpr uint32_t kI8OffEpi = kI8Stages * kI8Stage;              // 4 KB per epilogue warp
constexpr uint32_t kI8OffCol = kI8OffEpi + kI8EpiWarps * 4096;    // [2][256] scales and biases
constexpr uint32_t kI8OffBar = kI8OffCol + 2 * 2 * 256 * 4;
constexpr uint32_t kI8PairSmem = kI8OffBar + 8 * (2 * kI8Stages + 4) + 16 + 1024;

template <typename T, bool GELU>
__global__ void __launch_bounds__(kI8PairThreads, 1) __cluster_dims__(2, 1, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                     const __grid_constant__ CUtensorMap ty, const __grid_constant__ Int8Args a) {
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cl_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = a.tiles_m * a.tiles_n, nkb = (a.K + 127) / 128;
  const uint32_t bar_full = sb + kI8OffBar, bar_empty = bar_full + 8 * kI8Stages;
  const uint32_t bar_accf = bar_empty + 8 * kI8Stages, bar_acce = bar_accf + 16;
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tx);
    tma_prefetch_map(&tw);
    tma_prefetch_map(&ty);
    for (int s = 0; s < kI8Stages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_accf + 8 * b, 1);
      mbar_init(bar_acce + 8 * b, 2 * kI8EpiWarps);
    }
    mbar_fence_init();
  }
  pdl_entry();
  if (warp == 1) tmem_alloc2(sb + kI8OffBar + 8 * (2 * kI8Stages + 4), 512);
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + kI8OffBar + 8 * (2 * kI8Stages + 4));
  // tiles in bands of 8 token tiles, so that the tiles in flight share rows of both operands in L2
  auto tile_at = [&](int t, int& tm, int& tn) {
    const int band = t / (8 * a.tiles_n), in = t - band * 8 * a.tiles_n;
    const int h = min(8, a.tiles_m - band * 8);
    tn = in / h;
    tm = band * 8 + in - tn * h;
  };

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t lead_full = mapa(bar_full, 0);
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int tm, tn;
        tile_at(t, tm, tn);
        const int m0 = tm * 256 + 128 * (int)rank, n0 = tn * 256 + 128 * (int)rank;
        for (int kb = 0; kb < nkb; ++kb) {
          if (issued >= kI8Stages && !mbar_wait(bar_empty + 8 * s, ph ^ 1, a.timeout_ns)) {
            ok = false;
            break;
          }
          const uint32_t st = sb + s * kI8Stage;
          if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, 2 * kI8Stage);
          tma_load_2d_pair(st, &tx, kb * 128, m0, lead_full + 8 * s);
          tma_load_2d_pair(st + 16384, &tw, kb * 128, n0, lead_full + 8 * s);
          ++issued;
          if (++s == kI8Stages) { s = 0; ph ^= 1; }
        }
      }
      // the last stages have been read (so have landed) before the CTA may exit
      for (int g = max(issued - kI8Stages, 0); g < issued; ++g)
        if (!mbar_wait(bar_empty + 8 * (g % kI8Stages), (uint32_t)((g / kI8Stages) & 1), a.timeout_ns)) ok = false;
      if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = i8_idesc(256, 256);
      int s = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, ++i) {
        const int buf = i & 1;
        if (i >= 2 && !mbar_wait(bar_acce + 8 * buf, (uint32_t)(((i >> 1) - 1) & 1), a.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < nkb; ++kb) {
          if (!mbar_wait(bar_full + 8 * s, ph, a.timeout_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t st = sb + s * kI8Stage;
          const uint64_t ad = umma_desc_sw128(st), bd = umma_desc_sw128(st + 16384);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_i8<2>(tmem + buf * 256, ad + 2 * kk, bd + 2 * kk, idesc, (kb | kk) != 0 ? 1u : 0u);
          umma_commit2(bar_empty + 8 * s);
          if (++s == kI8Stages) { s = 0; ph ^= 1; }
        }
        if (ok) umma_commit2(bar_accf + 8 * buf);
      }
      if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    }
    __syncwarp();
  } else {
    const int ew = warp - 2, q4 = warp & 3, half = ew >> 2;  // lanes 32 q4 .. of TMEM, columns 128 half ..
    const uint32_t stg = sb + kI8OffEpi + ew * 4096;
    const uint32_t acce = mapa(bar_acce, 0);
    int i = 0;
    bool ok = true;
    for (int t = pair; t < tiles; t += pairs, ++i) {  // all tiles even after a failed wait: the warps meet in each
      int tm, tn;
      tile_at(t, tm, tn);
      const int buf = i & 1, m0 = tm * 256 + 128 * (int)rank + 32 * q4, n0 = tn * 256;
      const int m = m0 + lane;
      // the tile's column scales and biases, staged while the MMAs run
      float* col = reinterpret_cast<float*>(smem + kI8OffCol) + buf * 512;
      {
        const int c = ew * 32 + lane, n = n0 + c;
        col[c] = n < a.N ? i8_wscale(a, n) : 0.f;
        col[256 + c] = (n < a.N && (a.epi & I8_BIAS)) ? ld_param(reinterpret_cast<const T*>(a.bias) + n) : 0.f;
      }
      const float sx = m < a.M ? __ldg(a.sx + m) : 0.f;
      named_sync(1, 32 * kI8EpiWarps);
      if (ok && !mbar_wait(bar_accf + 8 * buf, (uint32_t)((i >> 1) & 1), a.timeout_ns)) {
        if (lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
#pragma unroll 1
      for (int c0 = half * 128; c0 < half * 128 + 128 && ok; c0 += 64) {
        uint32_t v[2][32];
        tmem_ld32(tmem + buf * 256 + ((uint32_t)(32 * q4) << 16) + c0, v[0]);
        tmem_ld32(tmem + buf * 256 + ((uint32_t)(32 * q4) << 16) + c0 + 32, v[1]);
        tmem_wait_ld();
        if (c0 == half * 128 + 64) {  // this warp's last read of the buffer
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acce + 8 * buf);
        }
        if (lane == 0) bulk_wait_read();  // the previous block has left the staging buffer
        __syncwarp();
        const T* res = reinterpret_cast<const T*>(a.resid) + (size_t)m * a.N + n0 + c0;
#pragma unroll
        for (int g = 0; g < 8; ++g) {  // 8 columns: one 16-byte piece of the row
          uint4 rq = make_uint4(0, 0, 0, 0);
          const bool rv = !GELU && (a.epi & I8_RESID) && m < a.M;
          if (rv && a.vec && n0 + c0 + 8 * g < a.N) rq = *reinterpret_cast<const uint4*>(res + 8 * g);
          const uint32_t rw[4] = {rq.x, rq.y, rq.z, rq.w};
          float wv[8], bv[8];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            *reinterpret_cast<float4*>(wv + 4 * e) = *reinterpret_cast<const float4*>(col + c0 + 8 * g + 4 * e);
            *reinterpret_cast<float4*>(bv + 4 * e) = *reinterpret_cast<const float4*>(col + 256 + c0 + 8 * g + 4 * e);
          }
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = 8 * g + 2 * e;
            float y0 = fmaf((float)(int)v[c >> 5][c & 31] * sx, wv[2 * e], bv[2 * e]);
            float y1 = fmaf((float)(int)v[c >> 5][(c & 31) + 1] * sx, wv[2 * e + 1], bv[2 * e + 1]);
            if (GELU) {
              y0 = i8_gelu(y0);
              y1 = i8_gelu(y1);
            } else if (rv) {
              float2 r = Act<T>::unpack2(rw[e]);
              if (!a.vec) {
                r.x = n0 + c0 + c < a.N ? ld_param(res + c) : 0.f;
                r.y = n0 + c0 + c + 1 < a.N ? ld_param(res + c + 1) : 0.f;
              }
              y0 += r.x;
              y1 += r.y;
            }
            o[e] = Act<T>::pack2(y0, y1);
          }
          sts16(stg + sw128(lane, g), o[0], o[1], o[2], o[3]);
        }
        if (a.vec) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && m0 < a.M && n0 + c0 < a.N) {
            tma_store_2d(&ty, n0 + c0, m0, stg);
            bulk_commit();
          }
        } else {  // rows off the 16-byte boundaries TMA needs: two columns a lane, row by row
          __syncwarp();
          for (int r = 0; r < 32 && m0 + r < a.M; ++r) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + (stg - sb) + sw128(r, lane >> 2) + (lane & 3) * 4);
            T* out = reinterpret_cast<T*>(a.out) + (size_t)(m0 + r) * a.N;
            const int n = n0 + c0 + 2 * lane;
            const unsigned short h[2] = {(unsigned short)w, (unsigned short)(w >> 16)};
            if (n < a.N) reinterpret_cast<unsigned short*>(out)[n] = h[0];
            if (n + 1 < a.N) reinterpret_cast<unsigned short*>(out)[n + 1] = h[1];
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait();
    __syncwarp();
  }
  tc_fence_before();
  cluster_sync();  // both CTAs: every load has landed, every MMA completed, every TMEM read and remote arrival done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// few tokens
// ---------------------------------------------------------------------------
// One cluster per 128 features x NT tokens, its CTAs each a slice of K: the
// weights are the MMA's 128 lanes (A), the tokens its N, so a call of one
// token wastes lanes of nothing but the tensor core. Six warps: TMA producer,
// MMA issuer, four that move the int32 partial sums to shared memory as
// [token][feature]; then every CTA adds its share of the features over the
// cluster's partials (integers: exact in any order) and writes them.
constexpr int kI8FewThreads = 192;
template <int NT> constexpr uint32_t i8_few_stage() { return 16384u + NT * 128u; }
template <int NT> constexpr uint32_t i8_few_part() { return NT * 128u * 4u; }

template <typename T, int NT, bool GELU>
__global__ void __launch_bounds__(kI8FewThreads)
    int8_few_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                    const __grid_constant__ Int8Args a) {
  constexpr uint32_t STAGE = i8_few_stage<NT>();
  constexpr uint32_t COLS = NT < 32 ? 32 : NT;
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = a.split;
  const uint32_t rank = S > 1 ? cl_rank() : 0;
  const int unit = blockIdx.x / S, n_units = (a.N + 127) / 128;
  const int n0 = (unit % n_units) * 128, m0 = (unit / n_units) * NT;
  const int nkb = (a.K + 127) / 128;
  const int kb0 = nkb * (int)rank / S, kb1 = nkb * ((int)rank + 1) / S;
  uint32_t ring = a.ns * STAGE;
  if (ring < i8_few_part<NT>()) ring = i8_few_part<NT>();
  const uint32_t bar_full = sb + ring, bar_empty = bar_full + 8 * a.ns, bar_acc = bar_empty + 8 * a.ns;
  const uint32_t off_tm = bar_acc + 8 - sb;
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tx);
    tma_prefetch_map(&tw);
    for (int s = 0; s < a.ns; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_acc, 1);
    mbar_fence_init();
  }
  pdl_entry();
  if (warp == 1) {
    tmem_alloc(sb + off_tm, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + off_tm);
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int issued = 0, s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (issued >= a.ns && !mbar_wait(bar_empty + 8 * s, ph ^ 1, a.timeout_ns)) {
          ok = false;
          break;
        }
        const uint32_t st = sb + s * STAGE, fb = bar_full + 8 * s;
        mbar_arrive_expect_tx(fb, STAGE);
        tma_load_2d(st, &tw, kb * 128, n0, fb);
        tma_load_2d(st + 16384, &tx, kb * 128, m0, fb);
        ++issued;
        if (++s == a.ns) { s = 0; ph ^= 1; }
      }
      for (int g = max(issued - a.ns, 0); g < issued; ++g)
        if (!mbar_wait(bar_full + 8 * (g % a.ns), (uint32_t)((g / a.ns) & 1), a.timeout_ns)) ok = false;
      if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = i8_idesc(128, NT);
      bool ok = true;
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(bar_full + 8 * s, ph, a.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t st = sb + s * STAGE;
        const uint64_t ad = umma_desc_sw128(st), bd = umma_desc_sw128(st + 16384);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_i8<1>(tmem, ad + 2 * kk, bd + 2 * kk, idesc, (kb != kb0 || kk) ? 1u : 0u);
        umma_commit(bar_empty + 8 * s);
        if (++s == a.ns) { s = 0; ph ^= 1; }
      }
      if (ok) umma_commit(bar_acc);
      else atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    }
    __syncwarp();
  }
  // every MMA has completed: the stages are free for the partial sums
  const bool done = mbar_wait(bar_acc, 0, a.timeout_ns);
  if (!done && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
  __syncthreads();
  tc_fence_after();
  if (warp >= 2) {
    const int q4 = warp & 3;
#pragma unroll
    for (int c0 = 0; c0 < NT; c0 += 16) {
      uint32_t v[16];
      tmem_ld16(tmem + ((uint32_t)(32 * q4) << 16) + c0, v);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e)
        *reinterpret_cast<uint32_t*>(smem + ((c0 + e) * 128 + 32 * q4 + lane) * 4) = v[e];
    }
  }
  tc_fence_before();
  if (S > 1) cluster_sync(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
  // this CTA's features rank * (128 / S) ..: groups of 4 of one token
  const int fg = 32 / S;  // feature groups of 4 per CTA
  for (int i = threadIdx.x; i < NT * fg && done; i += kI8FewThreads) {
    const int tok = i / fg, f = ((int)rank * fg + i % fg) * 4;
    const int m = m0 + tok, n = n0 + f;
    if (m >= a.M || n >= a.N) continue;
    int4 acc = make_int4(0, 0, 0, 0);
    const uint32_t at = sb + (tok * 128 + f) * 4;
    if (S > 1) {
#pragma unroll 4
      for (int r = 0; r < S; ++r) {
        const float4 p = ld_dsmem_f4(mapa(at, r));
        acc.x += __float_as_int(p.x);
        acc.y += __float_as_int(p.y);
        acc.z += __float_as_int(p.z);
        acc.w += __float_as_int(p.w);
      }
    } else {
      acc = *reinterpret_cast<const int4*>(smem + (at - sb));
    }
    const float sx = __ldg(a.sx + m);
    const int s4[4] = {acc.x, acc.y, acc.z, acc.w};
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = 0.f;
      if (n + e < a.N) {
        const float b = (a.epi & I8_BIAS) ? ld_param(reinterpret_cast<const T*>(a.bias) + n + e) : 0.f;
        y[e] = fmaf((float)s4[e] * sx, i8_wscale(a, n + e), b);
        if (GELU) y[e] = i8_gelu(y[e]);
        else if (a.epi & I8_RESID) y[e] += ld_param(reinterpret_cast<const T*>(a.resid) + (size_t)m * a.N + n + e);
      }
    }
    T* out = reinterpret_cast<T*>(a.out) + (size_t)m * a.N + n;
    if (a.vec) {
      *reinterpret_cast<uint2*>(out) = make_uint2(Act<T>::pack2(y[0], y[1]), Act<T>::pack2(y[2], y[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) out[e] = Act<T>::from_f(y[e]);
    }
  }
  if (S > 1) cluster_sync();  // the partials stay until every CTA of the cluster has read them
}

}  // namespace ee
