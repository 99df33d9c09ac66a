// ee_prompt_tc.cuh -- attention over long packed prompts on the 5th-generation
// tensor cores.
//
// A CTA takes two tiles of 128 query rows that read the same key head -- two
// heads of a group at the same rows, or two neighbouring row blocks of one
// head -- and walks the keys in blocks of 128, one pass with a running
// maximum and sum:
//   S = Q K^T       tcgen05.mma, both operands from shared memory, S in TMEM
//   P = 2^(c S - m) one thread per row: the whole row of S in registers, no
//                   exchange between threads; P goes back over S as 16-bit
//   O += P V        tcgen05.mma, A = P from TMEM, B = V (rows are keys: the
//                   MN-major operand), O in TMEM for the whole walk
// While one tile's threads are in the softmax, the tensor cores run the other
// tile's two products: per 128 x 128 block and tile 2 x 128^2 hd MACs (1024
// cycles at hd 128) against 128^2 exponentials (1024 cycles of the MUFU), so
// both are near their limit at hd 128 and the exponentials lead at hd 64.
//
// The running maximum m is a reference, not the exact maximum: it moves only
// when a row's maximum exceeds it by more than 2^8, so O is rarely rescaled
// (the weights stay below 2^8 and the result O / l does not depend on m). S(j)
// of a tile is issued after its O += P(j-1) V(j-1), so the wait for S(j) also
// says that O may be rescaled.
//
// Warps 0-3 and 4-7: softmax and output of tile 0 and 1; warp 8: TMA loads;
// warp 9: MMA issue (10 and 11 only fill their warpgroup). Waits are bounded; a timeout leaves EE_ERR_TIMEOUT in
// the GEMM status word.
#pragma once

#include "ee_prompt.cuh"
#include "ee_tma.cuh"
#include "ee_umma.cuh"

namespace ee {

struct PromptTcArgs {
  PromptArgs p;
  int pair_heads;  // 1: the tiles are two heads of a group, 0: two row blocks
  int head_items;  // items per row block (or pair of them): n_q / 2 or n_q
  int* status;
  unsigned long long timeout_ns;
};

constexpr int kPtThreads = 384;
// registers: 384 threads launch with 168 each; the four warps of loads and MMAs
// give theirs up to 72 and the softmax warps take 216 (256 x 216 + 128 x 72 =
// 384 x 168), so that a whole row of S stays in registers
constexpr int kPtRegsLaunch = 168, kPtRegsSoft = 216, kPtRegsRest = 72;
static_assert(256 * kPtRegsSoft + 128 * kPtRegsRest <= kPtThreads * kPtRegsLaunch, "the register shares fit the launch");
constexpr int kPtKeys = 128;
template <int HD> constexpr int pt_slots() { return HD == 128 ? 5 : 8; }
template <int HD> constexpr uint32_t pt_tile() { return 128u * HD * 2; }
template <int HD> constexpr uint32_t pt_off_bar() { return (2 + pt_slots<HD>()) * pt_tile<HD>(); }
template <int HD> constexpr uint32_t pt_smem() { return pt_off_bar<HD>() + 8 * (2 * pt_slots<HD>() + 8) + 64 + 1024; }

EE_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
// Descriptor of an MN-major, 128-byte-swizzled tile: lines of 64 elements of
// the MN dimension, one per k; eight k per 1024-byte atom (stride byte offset),
// the next 64 MN elements `panel` bytes on (leading byte offset).
EE_DEV uint64_t umma_desc_mn128(uint32_t saddr, uint32_t panel) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((panel >> 4) & 0x3FFFu) << 16) | ((uint64_t)64u << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
constexpr uint32_t kIdescBMajorMN = 1u << 16;

EE_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kPtThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptTcArgs a) {
  constexpr int NS = pt_slots<HD>();
  constexpr uint32_t TILE = pt_tile<HD>(), PANEL = 128 * 128;  // a panel: 64 columns of 128 rows
  constexpr int PANELS = HD / 64;
  extern __shared__ __align__(1024) char smem_raw[];
  __shared__ int sh[kPtThreads / 32 + 2];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sQ = sb, sKV = sb + 2 * TILE;
  const uint32_t b_full = sb + pt_off_bar<HD>(), b_empty = b_full + 8 * NS;
  const uint32_t b_q = b_empty + 8 * NS, b_s = b_q + 8, b_p = b_s + 16, b_o = b_p + 16, b_fix = b_o + 16;
  const uint32_t off_tm = b_fix + 8 - sb;
  if (warp == 8 && lane == 0) {
    tma_prefetch_map(&mq);
    tma_prefetch_map(&mk);
    tma_prefetch_map(&mv);
    for (int s = 0; s < NS; ++s) {
      mbar_init(b_full + 8 * s, 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    mbar_init(b_q, 1);
    mbar_init(b_fix, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(b_s + 8 * t, 1);
      mbar_init(b_p + 8 * t, 4);
      mbar_init(b_o + 8 * t, 1);
    }
    mbar_fence_init();
  }
  pdl_entry();
  // this CTA's item: later row blocks (more keys under the causal mask) first
  const PromptArgs& p = a.p;
  const int units = gridDim.x / a.head_items;
  const int unit = units - 1 - (int)blockIdx.x / a.head_items, hi = (int)blockIdx.x % a.head_items;
  PromptSeq s;
  if (!prompt_find(p, unit, 1, a.pair_heads ? 128 : 256, kPtThreads, sh, s)) return;
  const int h0 = a.pair_heads ? 2 * hi : hi, kvh = h0 / p.group;
  const int r0 = s.blk * (a.pair_heads ? 128 : 256);
  int nb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = a.pair_heads ? r0 : r0 + 128 * t;
    const int kend = p.causal ? min(max(s.klen - s.qlen + min(r + 128, s.qlen), 0), s.klen) : s.klen;
    nb[t] = r < s.qlen ? (kend + kPtKeys - 1) / kPtKeys : 0;
  }
  const int nbm = max(nb[0], nb[1]);
  if (warp == 9) {
    tmem_alloc(sb + off_tm, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + off_tm);
  // TMEM columns: S (P over its first half) of tile t at 128 t, O at 256 + 128 t
  // keys past the sequence's end in its last block: zeroed in V before their product with weights of 0
  const int tail = nbm > 0 && nbm * kPtKeys > s.klen ? s.klen - (nbm - 1) * kPtKeys : kPtKeys;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsRest));
   if (warp == 8) {
    bool ok = true;
    int n = 0;
    if (lane == 0 && nbm > 0) {
      mbar_arrive_expect_tx(b_q, (nb[0] > 0 ? TILE : 0) + (nb[1] > 0 ? TILE : 0));
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (nb[t] > 0)
          for (int c = 0; c < PANELS; ++c)
            tma_load_3d(sQ + t * TILE + c * PANEL, &mq, 64 * c, a.pair_heads ? h0 + t : h0,
                        s.q0 + (a.pair_heads ? r0 : r0 + 128 * t), b_q);
      for (; n < 2 * nbm; ++n) {  // K(0) V(0) K(1) V(1) ...
        const int sl = n % NS, k0 = s.k0 + (n >> 1) * kPtKeys;
        if (n >= NS && !mbar_wait(b_empty + 8 * sl, (uint32_t)((n / NS - 1) & 1), a.timeout_ns)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(b_full + 8 * sl, TILE);
        for (int c = 0; c < PANELS; ++c)
          tma_load_3d(sKV + sl * TILE + c * PANEL, (n & 1) ? &mv : &mk, 64 * c, kvh, k0, b_full + 8 * sl);
      }
    }
    __syncwarp();
    n = __shfl_sync(0xffffffffu, n, 0);
    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    // everything issued lands before the CTA may exit; the last of it is V's last block
    for (int g = max(n - NS, 0); g < n; ++g)
      if (!mbar_wait(b_full + 8 * (g % NS), (uint32_t)((g / NS) & 1), a.timeout_ns)) ok = false;
    if (nbm > 0 && !mbar_wait(b_q, 0, a.timeout_ns)) ok = false;
    if (ok && tail < kPtKeys) {
      const uint32_t v = sKV + (uint32_t)((2 * nbm - 1) % NS) * TILE;
      for (int i = lane; i < (kPtKeys - tail) * 8 * PANELS; i += 32) {
        const int row = tail + i / (8 * PANELS), c = i % (8 * PANELS);
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + (c >> 3) * PANEL + row * 128 + (c & 7) * 16),
                     "r"(0)
                     : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_fix);
    }
    if (!ok && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
   } else if (warp == 9) {
    if (lane == 0 && nbm > 0) {
      constexpr uint32_t id_s = umma_idesc<T>(128, 128), id_o = umma_idesc<T>(128, HD) | kIdescBMajorMN;
      bool ok = mbar_wait(b_q, 0, a.timeout_ns);
      auto wait_slot = [&](int n) { return mbar_wait(b_full + 8 * (n % NS), (uint32_t)((n / NS) & 1), a.timeout_ns); };
      auto scores = [&](int t, int j) {  // S_t = Q_t K(j)^T
        const uint32_t kt = sKV + (uint32_t)((2 * j) % NS) * TILE;
        const uint64_t qd = umma_desc_sw128(sQ + t * TILE), kd = umma_desc_sw128(kt);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint64_t o = (uint64_t)(((kk >> 2) * PANEL + (kk & 3) * 32) >> 4);
          umma_f16(tmem + 128 * t, qd + o, kd + o, id_s, kk ? 1u : 0u);
        }
        umma_commit(b_s + 8 * t);
      };
      if (ok) ok = wait_slot(0);
      tc_fence_after();
      if (ok) {
        if (nb[0] > 0) scores(0, 0);
        if (nb[1] > 0) scores(1, 0);
        umma_commit(b_empty + 0);  // K(0): slot 0
      }
      for (int j = 0; j < nbm && ok; ++j) {
        const int vs = (2 * j + 1) % NS;
        const uint32_t vt = sKV + (uint32_t)vs * TILE;
        ok = wait_slot(2 * j + 1) && (j + 1 < nbm ? wait_slot(2 * j + 2) : (tail == kPtKeys || mbar_wait(b_fix, 0, a.timeout_ns)));
        const uint64_t vd = umma_desc_mn128(vt, PANEL);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || j >= nb[t]) continue;
          ok = mbar_wait(b_p + 8 * t, (uint32_t)(j & 1), a.timeout_ns);
          if (!ok) continue;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kPtKeys / 16; ++kk)  // O_t += P_t V(j), 16 keys at a time
            umma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * kk, vd + (uint64_t)((kk * 2048) >> 4), id_o,
                        (j | kk) ? 1u : 0u);
          if (j + 1 < nb[t]) scores(t, j + 1);
          else umma_commit(b_o + 8 * t);
        }
        if (ok) {
          umma_commit(b_empty + 8 * vs);
          if (j + 1 < nbm) umma_commit(b_empty + 8 * ((2 * j + 2) % NS));
        }
      }
      if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    }
    __syncwarp();
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPtRegsSoft));
    const int t = warp >> 2, q4 = warp & 3;
    const int row = (a.pair_heads ? r0 : r0 + 128 * t) + 32 * q4 + lane;
    const int head = a.pair_heads ? h0 + t : h0;
    const uint32_t ts = tmem + 128 * t + ((uint32_t)(32 * q4) << 16), to = ts - 128 * t + 256 + 128 * t;
    const int lim = p.causal ? min(s.klen, s.klen - s.qlen + row + 1) : s.klen;  // keys this row sees
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nb[t] && ok; ++j) {
      ok = mbar_wait(b_s + 8 * t, (uint32_t)(j & 1), a.timeout_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, v[c]);
      tmem_wait_ld();
      const int left = lim - j * kPtKeys;
      if (__any_sync(0xffffffffu, left < kPtKeys)) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * c + e >= left) v[c][e] = 0xff800000u;
      }
      float x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = __uint_as_float(v[c][0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) x[c] = fmaxf(x[c], __uint_as_float(v[c][e]));
      }
      const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * p.scale_log2;
      float f = 1.f;
      if (mx > m + 8.f) {  // also from -inf, with f = 0: nothing to rescale yet
        f = ex2(m - mx);
        m = mx;
      }
      if (__any_sync(0xffffffffu, f != 1.f) && j > 0) {
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st32(to + 32 * c, o);
        }
        tmem_wait_st();
      }
      const float neg = m == -INFINITY ? 0.f : -m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float p0 = ex2(fmaf(__uint_as_float(v[c][e]), p.scale_log2, neg));
          const float p1 = ex2(fmaf(__uint_as_float(v[c][e + 1]), p.scale_log2, neg));
          sum[c] += p0 + p1;
          v[c >> 1][(c & 1) * 16 + e / 2] = Act<T>::pack2(p0, p1);
        }
        if (c & 1) tmem_st32(ts + 32 * (c >> 1), v[c >> 1]);
      }
      l = l * f + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(b_p + 8 * t);
    }
    if (ok && nb[t] > 0) ok = mbar_wait(b_o + 8 * t, 0, a.timeout_ns);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
    tc_fence_after();
    const bool mine = ok && row < s.qlen && (a.pair_heads || r0 + 128 * t < s.qlen);
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
    T* out = reinterpret_cast<T*>(p.out) + (long long)(s.q0 + row) * p.o_tok + head * p.o_head;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t o[32];
      if (nb[t] > 0) {
        tmem_ld32(to + 32 * c, o);
        tmem_wait_ld();
      }
      if (mine) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = l == 0.f ? 0u
                            : Act<T>::pack2(__uint_as_float(o[e + 2 * i]) * inv, __uint_as_float(o[e + 2 * i + 1]) * inv);
          *reinterpret_cast<uint4*>(out + 32 * c + e) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();  // every MMA has completed (the outputs waited for them) and every TMEM read is done
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ee
