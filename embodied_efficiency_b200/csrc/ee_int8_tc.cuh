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
  int early;             // launched behind the call's own quantiser: the weights may be read before it has finished
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
// 11 instructions a value in packed pairs, where erff costs 30: the epilogue
// of a 256 x 256 tile has to keep up with the tensor cores.
EE_DEV uint64_t i8_gelu2(uint64_t z) {
  uint32_t z0, z1, d0, d1, e0, e1;
  unpack64(z, z0, z1);
  const uint64_t a = pack64(z0 & 0x7FFFFFFFu, z1 & 0x7FFFFFFFu);
  unpack64(fma2f(a, both(0.35f), both(1.f)), d0, d1);
  unpack64(mul2f(mul2f(z, z), both(-0.72134752f)), e0, e1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+r"(d0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+r"(d1));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+r"(e0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+r"(e1));
  const uint64_t t = pack64(d0, d1);
  uint64_t p = fma2f(t, both(-0.044615f), both(0.18442732f));  // -P: the final product is subtracted
  p = fma2f(t, p, both(-0.21107948f));
  p = fma2f(t, p, both(-0.00892954f));
  p = fma2f(t, p, both(-0.14315536f));
  p = fma2f(t, p, both(-0.13687154f));
  p = fma2f(t, p, both(-0.13977644f));
  p = mul2f(mul2f(p, t), pack64(e0, e1));
  unpack64(a, d0, d1);
  // the fminf: 0 instead of inf * 0
  return fma2f(pack64(__float_as_uint(fminf(__uint_as_float(d0), 3.0e38f)), __float_as_uint(fminf(__uint_as_float(d1), 3.0e38f))),
               p, pack64(__float_as_uint(fmaxf(__uint_as_float(z0), 0.f)), __float_as_uint(fmaxf(__uint_as_float(z1), 0.f))));
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
// Measured, single passes after a pause: 52224 x 8192 x 2048: 582 us, 3.0 POP/s
// (with the GELU 650; back to back, at the power limit's clocks, 790), 8192^3:
// 333 us, 3.3 POP/s, twice the measured 16-bit GEMM rate. (16 epilogue warps and
// a stage less were slower with the GELU: 677 us.)
constexpr int kI8Stages = 5, kI8EpiWarps = 8;
constexpr int kI8PairThreads = 32 * (2 + kI8EpiWarps);
constexpr uint32_t kI8Stage = 32768;
constexpr uint32_t kI8OffEpi = kI8Stages * kI8Stage;            // 4 KB per epilogue warp
constexpr uint32_t kI8OffCol = kI8OffEpi + kI8EpiWarps * 4096;  // [2][256] scales and biases
constexpr uint32_t kI8OffBar = kI8OffCol + 2 * 2 * 256 * 4;
constexpr uint32_t kI8PairUsed = kI8OffBar + 8 * (2 * kI8Stages + 4) + 16 + 1024;

// The other kernel's CTAs: a ring of stages (128 weight rows and NT tokens of
// a k-block) that the partial sums take over, two barriers a stage, one for the
// sums, the TMEM address.
template <int NT> constexpr uint32_t i8_few_stage() { return 16384u + NT * 128u; }
template <int NT> constexpr uint32_t i8_few_part() { return NT * 128u * 4u; }
template <int NT> constexpr uint32_t i8_few_ring(int ns) {
  return ns * i8_few_stage<NT>() > i8_few_part<NT>() ? ns * i8_few_stage<NT>() : i8_few_part<NT>();
}
template <int NT> constexpr uint32_t i8_few_smem(int ns) { return 1024u + i8_few_ring<NT>(ns) + 16u * ns + 16u; }

// A pair takes all TMEM columns of two SMs, and one of its CTAs can have its
// columns while the other waits for a CTA of another stream's launch. So that
// none which waits for a CTA elsewhere can be that one, no CTA of a cluster of
// int8_few_kernel fits beside a pair's: the pair asks for more shared memory
// than it uses. (All of an SM's would keep every other stream's kernels out.)
constexpr uint32_t kSmShared = 228 * 1024, kCtaReserve = 1024;  // of an SM; per CTA, beside what it asks for
constexpr uint32_t kI8PairAlone = (kSmShared - 2 * kCtaReserve - i8_few_smem<16>(1)) / 1024 * 1024 + 1024;
constexpr uint32_t kI8PairSmem = kI8PairUsed > kI8PairAlone ? kI8PairUsed : kI8PairAlone;
static_assert(kI8PairSmem + kCtaReserve <= kSmShared, "a pair's CTA fits");
static_assert(kI8PairSmem + i8_few_smem<16>(1) + 2 * kCtaReserve > kSmShared, "and nothing of the other kernel beside it");

template <typename T, bool GELU>
__global__ void __launch_bounds__(kI8PairThreads, 1) __cluster_dims__(2, 1, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                     const __grid_constant__ CUtensorMap ty, const __grid_constant__ Int8Args a) {
  constexpr int NS = kI8Stages, EW = kI8EpiWarps;
  constexpr uint32_t OFF_BAR = kI8OffBar;
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cl_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = a.tiles_m * a.tiles_n, nkb = (a.K + 127) / 128;
  const uint32_t bar_full = sb + OFF_BAR, bar_empty = bar_full + 8 * NS;
  const uint32_t bar_accf = bar_empty + 8 * NS, bar_acce = bar_accf + 16;
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tx);
    tma_prefetch_map(&tw);
    tma_prefetch_map(&ty);
    for (int s = 0; s < NS; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_accf + 8 * b, 1);
      mbar_init(bar_acce + 8 * b, 2 * EW);
    }
    mbar_fence_init();
  }
  if (!a.early) pdl_entry();
  if (warp == 1) tmem_alloc2(sb + OFF_BAR + 8 * (2 * NS + 4), 512);
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + OFF_BAR + 8 * (2 * NS + 4));
  // tiles in bands of 8 token tiles, so that the tiles in flight share rows of both operands in L2
  auto tile_at = [&](int t, int& tm, int& tn) {
    const int band = t / (8 * a.tiles_n), in = t - band * 8 * a.tiles_n;
    const int h = min(8, a.tiles_m - band * 8);
    tn = in / h;
    tm = band * 8 + in - tn * h;
  };

  const uint32_t lead_full = mapa(bar_full, 0);
  int pre = 0;  // stages whose weights are on their way before the tokens are ready
  if (a.early) {
    if (warp == 0 && lane == 0 && pair < tiles) {
      int tm, tn;
      tile_at(pair, tm, tn);
      for (; pre < NS && pre < nkb; ++pre) {
        if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * pre, 2 * kI8Stage);
        tma_load_2d_pair(sb + pre * kI8Stage + 16384, &tw, pre * 128, tn * 256 + 128 * (int)rank, lead_full + 8 * pre);
      }
    }
    __syncwarp();
    pdl_entry();
  }
  if (warp == 0) {
    if (lane == 0) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int tm, tn;
        tile_at(t, tm, tn);
        const int m0 = tm * 256 + 128 * (int)rank, n0 = tn * 256 + 128 * (int)rank;
        for (int kb = 0; kb < nkb; ++kb) {
          if (issued >= NS && !mbar_wait(bar_empty + 8 * s, ph ^ 1, a.timeout_ns)) {
            ok = false;
            break;
          }
          const uint32_t st = sb + s * kI8Stage;
          if (issued >= pre) {
            if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, 2 * kI8Stage);
            tma_load_2d_pair(st + 16384, &tw, kb * 128, n0, lead_full + 8 * s);
          }
          tma_load_2d_pair(st, &tx, kb * 128, m0, lead_full + 8 * s);
          ++issued;
          if (++s == NS) { s = 0; ph ^= 1; }
        }
      }
      // the last stages have been read (so have landed) before the CTA may exit
      for (int g = max(issued - NS, 0); g < issued; ++g)
        if (!mbar_wait(bar_empty + 8 * (g % NS), (uint32_t)((g / NS) & 1), a.timeout_ns)) ok = false;
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
          if (++s == NS) { s = 0; ph ^= 1; }
        }
        if (ok) umma_commit2(bar_accf + 8 * buf);
      }
      if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    }
    __syncwarp();
  } else {
    constexpr int CW = 256 / (EW / 4);  // columns per epilogue warp
    const int ew = warp - 2, q4 = warp & 3, cbeg = (ew >> 2) * CW;  // lanes 32 q4 .. of TMEM, columns cbeg ..
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
      for (int c = ew * 32 + lane; c < 512; c += 32 * EW) {
        const int n = n0 + (c & 255);
        float w = 0.f;
        if (n < a.N) {
          if (c < 256) w = i8_wscale(a, n);
          else if (a.epi & I8_BIAS) w = ld_param(reinterpret_cast<const T*>(a.bias) + n);
        }
        col[c] = w;
      }
      const float sx = m < a.M ? __ldg(a.sx + m) : 0.f;
      named_sync(1, 32 * EW);
      if (ok && !mbar_wait(bar_accf + 8 * buf, (uint32_t)((i >> 1) & 1), a.timeout_ns)) {
        if (lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      const uint64_t sx2 = both(sx);
#pragma unroll 1
      for (int c0 = cbeg; c0 < cbeg + CW && ok; c0 += 64) {
        if (lane == 0) bulk_wait_read();  // the previous block has left the staging buffer
        __syncwarp();
        const T* res = reinterpret_cast<const T*>(a.resid) + (size_t)m * a.N + n0 + c0;
        const bool rv = !GELU && (a.epi & I8_RESID) && m < a.M;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t v[32];
          tmem_ld32(tmem + buf * 256 + ((uint32_t)(32 * q4) << 16) + c0 + 32 * h, v);
          tmem_wait_ld();
          if (h == 1 && c0 + 64 == cbeg + CW) {  // this warp's last read of the buffer
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acce + 8 * buf);
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {  // 8 columns: one 16-byte piece of the row
            const int c = 32 * h + 8 * g;
            uint4 rq = make_uint4(0, 0, 0, 0);
            if (rv && a.vec && n0 + c0 + c < a.N) rq = *reinterpret_cast<const uint4*>(res + c);
            const uint32_t rw[4] = {rq.x, rq.y, rq.z, rq.w};
            uint4 w4[2], b4[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              w4[e] = *reinterpret_cast<const uint4*>(col + c0 + c + 4 * e);
              b4[e] = *reinterpret_cast<const uint4*>(col + 256 + c0 + c + 4 * e);
            }
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint4 wq = w4[e >> 1], bq = b4[e >> 1];
              const uint64_t w2 = (e & 1) ? pack64(wq.z, wq.w) : pack64(wq.x, wq.y);
              const uint64_t b2 = (e & 1) ? pack64(bq.z, bq.w) : pack64(bq.x, bq.y);
              const uint64_t s2 = pack64(__float_as_uint((float)(int)v[8 * g + 2 * e]),
                                         __float_as_uint((float)(int)v[8 * g + 2 * e + 1]));
              uint64_t y = fma2f(mul2f(s2, sx2), w2, b2);
              if (GELU) y = i8_gelu2(y);
              uint32_t y0, y1;
              unpack64(y, y0, y1);
              float f0 = __uint_as_float(y0), f1 = __uint_as_float(y1);
              if (rv) {
                float2 r = Act<T>::unpack2(rw[e]);
                if (!a.vec) {
                  r.x = n0 + c0 + c + 2 * e < a.N ? ld_param(res + c + 2 * e) : 0.f;
                  r.y = n0 + c0 + c + 2 * e + 1 < a.N ? ld_param(res + c + 2 * e + 1) : 0.f;
                }
                f0 += r.x;
                f1 += r.y;
              }
              o[e] = Act<T>::pack2(f0, f1);
            }
            sts16(stg + sw128(lane, 4 * h + g), o[0], o[1], o[2], o[3]);
          }
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
// token wastes lanes of nothing but the tensor core. TMA producer, MMA issuer,
// four warps that move the int32 partial sums to shared memory as
// [token][feature]; then all warps of every CTA add its share of the features over the
// cluster's partials (integers: exact in any order) and writes them.
// TMEM is given back before the CTA waits for its cluster: a CTA that holds
// columns waits for its own loads only, so whoever waits for them gets them.
constexpr int kI8FewThreads = 256;

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
  const uint32_t bar_full = sb + i8_few_ring<NT>(a.ns), bar_empty = bar_full + 8 * a.ns, bar_acc = bar_empty + 8 * a.ns;
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
  if (!a.early) pdl_entry();
  if (warp == 1) {
    tmem_alloc(sb + off_tm, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + off_tm);
  int pre = 0;  // stages whose weights are on their way before the tokens are ready
  if (a.early) {
    if (warp == 0 && lane == 0) {
      for (; pre < a.ns && kb0 + pre < kb1; ++pre) {
        mbar_arrive_expect_tx(bar_full + 8 * pre, STAGE);
        tma_load_2d(sb + pre * STAGE, &tw, (kb0 + pre) * 128, n0, bar_full + 8 * pre);
      }
    }
    __syncwarp();
    pdl_entry();
  }
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
        if (issued >= pre) {
          mbar_arrive_expect_tx(fb, STAGE);
          tma_load_2d(st, &tw, kb * 128, n0, fb);
        }
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
  if (warp >= 4) {
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
    tc_fence_before();
  }
  if (warp == 1 || warp >= 4) named_sync(1, 32 * 5);  // the sums are out of TMEM
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, COLS);
  }
  if (S > 1) cluster_sync(); else __syncthreads();
  // this CTA's features rank * (128 / S) ..: 4 of one token at a time, the same 4 for all of a thread's tokens
  const int fg = 32 / S;
  static_assert(kI8FewThreads % 32 == 0, "a thread's features do not change");
  const int f = ((int)rank * fg + (int)threadIdx.x % fg) * 4, n = n0 + f;
  float sw[4], bias[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    sw[e] = n + e < a.N ? i8_wscale(a, n + e) : 0.f;
    bias[e] = n + e < a.N && (a.epi & I8_BIAS) ? ld_param(reinterpret_cast<const T*>(a.bias) + n + e) : 0.f;
  }
#pragma unroll 2
  for (int tok = threadIdx.x / fg; tok < NT; tok += kI8FewThreads / fg) {
    const int m = m0 + tok;
    if (m >= a.M || n >= a.N || !done) break;
    const float sx = __ldg(a.sx + m);
    int4 acc = make_int4(0, 0, 0, 0);
    const uint32_t at = sb + (tok * 128 + f) * 4;
    if (S > 1) {
#pragma unroll 8
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
    float y[4] = {(float)acc.x, (float)acc.y, (float)acc.z, (float)acc.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e] * sx, sw[e], bias[e]);
    if (GELU) {
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        uint32_t g0, g1;
        unpack64(i8_gelu2(pack64(__float_as_uint(y[e]), __float_as_uint(y[e + 1]))), g0, g1);
        y[e] = __uint_as_float(g0);
        y[e + 1] = __uint_as_float(g1);
      }
    }
    const size_t o = (size_t)m * a.N + n;
    const T* res = reinterpret_cast<const T*>(a.resid) + o;
    T* out = reinterpret_cast<T*>(a.out) + o;
    if (a.vec) {
      if (!GELU && (a.epi & I8_RESID)) {
        const uint2 r = *reinterpret_cast<const uint2*>(res);
        const float2 r0 = Act<T>::unpack2(r.x), r1 = Act<T>::unpack2(r.y);
        y[0] += r0.x; y[1] += r0.y; y[2] += r1.x; y[3] += r1.y;
      }
      *reinterpret_cast<uint2*>(out) = make_uint2(Act<T>::pack2(y[0], y[1]), Act<T>::pack2(y[2], y[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) {
          if (!GELU && (a.epi & I8_RESID)) y[e] += ld_param(res + e);
          out[e] = Act<T>::from_f(y[e]);
        }
    }
  }
  if (S > 1) cluster_sync();  // the partials stay until every CTA of the cluster has read them
}

}  // namespace ee
