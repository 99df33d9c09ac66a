// ee_prompt_tc.cuh -- attention over long packed prompts on the 5th-generation
// tensor cores.
//
// An item is two neighbouring tiles of up to 128 query rows of one sequence
// and key head; a row is (token, head of the key head's group), so a group
// shares its keys' loads and a tile of G heads covers 128 / G tokens. The keys
// are walked in blocks of 128, one pass with a running maximum and sum:
//   S = Q K^T       tcgen05.mma, both operands from shared memory, S in TMEM
//   P = 2^(c S - m) one thread per row: the whole row of S in registers, no
//                   exchange between threads; P goes back over S as 16-bit
//   O += P V        tcgen05.mma, A = P from TMEM, B = V (rows are keys: the
//                   MN-major operand), O in TMEM for the whole walk
// While one tile's threads are in the softmax, the tensor cores run the other
// tile's two products: per 128 x 128 block and tile 2 x 128^2 hd MACs (1024
// cycles at hd 128) against 128^2 exponentials (1024 cycles of the MUFU), so
// both are near their limit at hd 128 and the exponentials lead at hd 64. (A
// share of the exponentials as polynomials on the FMA pipe was slower at every
// share: 411 -> 428 / 472 / 530 us at hd 64 for 1/8, 1/4, 1/2 of them.)
//
// P is rounded to 16 bits, as the product takes it, while the sum l keeps the
// unrounded weights: half a step each, in either direction, which over many
// keys leaves 1.3 times the error of a plain fp32 form (fp16, heads of 64:
// 2.8e-4 to 2.1e-4 relative); a second product for the low bits would double P V.
//
// Measured: 8192 causal tokens, 16 / 4 heads of 128: 225 us in a single pass
// after a pause, 1220 TFLOP/s, 0.76 of the measured GEMM rate (back to back, at
// lower clocks, 257); 16 / 4 heads of 64 without a mask: 410 us, the MUFU 74 %
// busy while an SM has work. What bounds it is one thread's row: 3000 cycles
// per pair of blocks at hd 64 where the MUFU needs 2048. (Two threads a row
// need 130 registers and have 104: 470 -> 720 us at hd 128.)
// A last tile without a neighbour leaves its item's second half idle; halving
// its keys over both halves and joining the sums was slower (128 prompts of
// 257 to 816 tokens, hd 64: 395 -> 415 us).
//
// The running maximum m is a reference, not the exact maximum: it moves only
// when a row's maximum exceeds the one that set it by more than 8 (a factor of
// 2^8), so O is rarely rescaled (the weights stay below 2^8, for fp16 2^15, see
// prompt_reference, and the result O / l does not depend on m). S(j) of a tile
// is issued after its O += P(j-1) V(j-1), so the wait for S(j) also says that O
// may be rescaled.
//
// Persistent: one CTA per SM takes items c, 2G - 1 - c, 2G + c, ... of the G
// CTAs (a snake, longest items first), and the next item's loads and first
// scores run under the current one's last products and output. Warps 0-3 and
// 4-7: softmax and output of tile 0 and 1; warp 8: finds the items, publishes
// them in a shared-memory ring and loads Q, K and V by TMA; warp 9: MMA issue;
// warp 10: zeroes V's rows past a sequence's end (their weights are 0, but
// 0 * NaN is not); warp 11 only fills the warpgroup.
//
// Waits are bounded, each by what it waits for: a block's loads, scores,
// weights or products by timeout_ns, an item's whole walk by timeout_ns without
// a block started (wait_walk). A wait that gives up leaves EE_ERR_TIMEOUT in
// the GEMM status word and ends its role; the others then give up too, every
// load lands and every MMA completes before the CTA returns its memory.
#pragma once

#include "ee_prompt.cuh"
#include "ee_tma.cuh"
#include "ee_umma.cuh"

namespace ee {

struct PromptTcArgs {
  PromptArgs p;
  int tpt;  // tokens per tile: 128 / group
  int* status;
  unsigned long long timeout_ns;
};

constexpr int kPtThreads = 384;
// registers: 384 threads launch with 168 each; the four warps of loads and MMAs
// give theirs up to 88 and the softmax warps take 208 (256 x 208 + 128 x 88 =
// 384 x 168), so that a whole row of S stays in registers
constexpr int kPtRegsLaunch = 168, kPtRegsSoft = 208, kPtRegsRest = 88;
static_assert(256 * kPtRegsSoft + 128 * kPtRegsRest <= kPtThreads * kPtRegsLaunch, "the register shares fit the launch");
constexpr int kPtKeys = 128, kPtInfo = 4, kPtLoads = 8;  // keys per block; items published, loads of K / V ahead
constexpr unsigned long long kPtDrainNs = 1000000000ull;  // for loads and MMAs already issued, whatever timeout_ns is
template <int HD> constexpr int pt_slots() { return HD == 128 ? 4 : 8; }
template <int HD> constexpr uint32_t pt_tile() { return 128u * HD * 2; }
template <int HD> constexpr uint32_t pt_off_out() { return (2 + pt_slots<HD>()) * pt_tile<HD>(); }  // 4 KB per softmax warp
template <int HD> constexpr uint32_t pt_off_bar() { return pt_off_out<HD>() + 8 * 4096; }
// barriers: full / empty per load of K / V, Q full / empty, S / P (two halves) / S free / O / O free per tile, V to fix /
// fixed, item full / empty, MMAs done after a failure
template <int HD> constexpr uint32_t pt_off_info() { return pt_off_bar<HD>() + 8 * (2 * kPtLoads + 17 + 2 * kPtInfo) + 8; }
template <int HD> constexpr uint32_t pt_off_beat() { return pt_off_info<HD>() + kPtInfo * 64; }  // blocks the MMA warp has come to
template <int HD> constexpr uint32_t pt_smem() { return pt_off_beat<HD>() + 16 + 1024; }

// One published item (16 words)
struct PromptItem {
  int q0, qlen, k0, klen;  // the sequence (k0: its first key row)
  int tok, kvh, part;      // first token of tile 0, key head, part of the keys
  int key0;                // first key of this part
  int n[2];                // key blocks of the tiles in this part
  int tail;                // valid keys of the part's last block (128: all)
  int nbm;                 // max(n[0], n[1]); -1: no more items
  int pad[4];
};

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

// The 32 sequences in which the last item was found: a CTA's items come in
// order of descending units, so the search only ever moves down from there.
struct PromptWindow {
  int base, before;  // first sequence; units before it
};
// The window's sequences, one a lane, and the units up to and including each.
EE_DEV int prompt_window(const PromptTcArgs& a, const PromptWindow& w, PromptSeq& s, int& nu) {
  const int lane = threadIdx.x & 31, b = w.base + lane;
  s = PromptSeq{};
  if (b < a.p.n_seq) s = prompt_seq(a.p, b);
  nu = (s.qlen + 2 * a.tpt - 1) / (2 * a.tpt);
  int inc = nu;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  return inc;
}

// Item `idx` (unit-major from the last unit down, key heads and parts inside),
// by the whole warp. False past the last item.
EE_DEV bool prompt_item(const PromptTcArgs& a, int idx, int units, PromptWindow& w, PromptItem& it) {
  const PromptArgs& p = a.p;
  const int per = p.n_kv * p.splits;
  const int unit = units - 1 - idx / per;
  if (unit < 0) return false;
  it.kvh = idx % per / p.splits;
  it.part = idx % p.splits;
  PromptSeq s;
  int nu, inc = prompt_window(a, w, s, nu);
  while (unit < w.before && w.base > 0) {
    w.base -= 32;
    inc = prompt_window(a, w, s, nu);
    w.before -= __shfl_sync(0xffffffffu, inc, 31);
  }
  inc += w.before;
  const unsigned hit = __ballot_sync(0xffffffffu, unit >= inc - nu && unit < inc);
  if (!hit) return false;  // the offsets have changed meanwhile
  const int src = __ffs(hit) - 1;
  it.q0 = __shfl_sync(0xffffffffu, s.q0, src);
  it.qlen = __shfl_sync(0xffffffffu, s.qlen, src);
  it.k0 = __shfl_sync(0xffffffffu, s.k0, src);
  it.klen = __shfl_sync(0xffffffffu, s.klen, src);
  it.tok = (unit - __shfl_sync(0xffffffffu, inc - nu, src)) * 2 * a.tpt;
  int nb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = it.tok + t * a.tpt, last = min(first + a.tpt, it.qlen);
    const int kend = p.causal ? min(max(it.klen - it.qlen + last, 0), it.klen) : it.klen;
    nb[t] = first < it.qlen ? (kend + kPtKeys - 1) / kPtKeys : 0;
  }
  const int all = max(nb[0], nb[1]);
  const int j0 = (int)((long long)all * it.part / p.splits), j1 = (int)((long long)all * (it.part + 1) / p.splits);
  it.key0 = j0 * kPtKeys;
  it.n[0] = max(min(nb[0], j1) - j0, 0);
  it.n[1] = max(min(nb[1], j1) - j0, 0);
  it.nbm = max(it.n[0], it.n[1]);
  it.tail = it.nbm > 0 ? min(it.klen - (j0 + it.nbm - 1) * kPtKeys, kPtKeys) : kPtKeys;
  return true;
}

EE_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kPtThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptTcArgs a) {
  constexpr int NS = pt_slots<HD>(), NP = kPtLoads;
  static_assert(NS <= NP, "a barrier per load that the slots can hold");
  constexpr uint32_t TILE = pt_tile<HD>(), PANEL = 128 * 128;  // a panel: 64 columns of 128 rows
  constexpr int PANELS = HD / 64;
  // hd 64 leaves TMEM for P beside S, so the next scores are computed during the softmax
  constexpr bool SEP = HD == 64;
  // pieces in which a block's weights are handed over (in one piece, hd 64: 501 instead of 411 us for 8192 tokens)
  constexpr int PARTS = 2;
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sQ = sb, sKV = sb + 2 * TILE;
  const uint32_t b_full = sb + pt_off_bar<HD>(), b_empty = b_full + 8 * NP;
  const uint32_t b_qf = b_empty + 8 * NP, b_qe = b_qf + 8, b_s = b_qe + 8, b_p = b_s + 16, b_sf = b_p + 32, b_o = b_sf + 16;
  const uint32_t b_of = b_o + 16, b_req = b_of + 16, b_fix = b_req + 8, b_if = b_fix + 8, b_ie = b_if + 8 * kPtInfo;
  const uint32_t b_end = b_ie + 8 * kPtInfo, off_tm = b_end + 8 - sb;
  volatile PromptItem* ring = reinterpret_cast<volatile PromptItem*>(smem + pt_off_info<HD>());
  volatile uint32_t* beat = reinterpret_cast<volatile uint32_t*>(smem + pt_off_beat<HD>());
  const PromptArgs& p = a.p;
  if (warp == 8 && lane == 0) {
    tma_prefetch_map(&mq);
    tma_prefetch_map(&mk);
    tma_prefetch_map(&mv);
    for (int s = 0; s < NP; ++s) {
      mbar_init(b_full + 8 * s, 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    mbar_init(b_req, 1);
    mbar_init(b_fix, 1);
    mbar_init(b_qf, 1);
    mbar_init(b_qe, 1);
    mbar_init(b_end, 1);
    *beat = 0;
    for (int t = 0; t < 2; ++t) {
      mbar_init(b_s + 8 * t, 1);
      mbar_init(b_p + 8 * t, 4);
      mbar_init(b_p + 16 + 8 * t, 4);
      mbar_init(b_sf + 8 * t, 4);
      mbar_init(b_o + 8 * t, 1);
      mbar_init(b_of + 8 * t, 4);
    }
    for (int i = 0; i < kPtInfo; ++i) {
      mbar_init(b_if + 8 * i, 1);
      mbar_init(b_ie + 8 * i, 10);  // 8 softmax warps, the MMA warp, the fixing warp
    }
    mbar_fence_init();
  }
  pdl_entry();
  if (warp == 9) {
    tmem_alloc(sb + off_tm, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + off_tm);
  // TMEM columns: S of tile t at 128 t, O at 256 + 128 t (SEP: 256 + 64 t), P over S (SEP: at 384 + 64 t)
  constexpr uint32_t OC = SEP ? 64 : 128;
  // A wait that may take an item's walk over its keys: given up when timeout_ns pass without a block begun.
  auto wait_walk = [&](uint32_t bar, uint32_t parity) {
    uint32_t seen = *beat;
    while (!mbar_wait(bar, parity, a.timeout_ns)) {
      const uint32_t now = *beat;
      if (now == seen) return false;
      seen = now;
    }
    return true;
  };
  // The consumers' view of the item ring: wait for item i, read it; release when done with it. A tile that has no
  // blocks of the item before comes here while the other one walks them.
  auto item_wait = [&](int i) { return wait_walk(b_if + 8 * (i % kPtInfo), (uint32_t)((i / kPtInfo) & 1)); };
  auto item_done = [&](int i) { mbar_arrive(b_ie + 8 * (i % kPtInfo)); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsRest));
    if (warp == 8) {
      // ---------------- items and loads ----------------
      bool ok = true;
      int units = 0, n = 0, nq = 0, sl = 0;  // K / V tiles and Q loads issued so far, next slot
      uint32_t g = 0, slot_load[NS];         // loads (barrier phases) of K / V so far, and each slot's last one
#pragma unroll 4
      for (int b = lane; b < p.n_seq; b += 32) units += (prompt_seq(p, b).qlen + 2 * a.tpt - 1) / (2 * a.tpt);
      units = __reduce_add_sync(0xffffffffu, units);
      PromptWindow window{(p.n_seq - 1) / 32 * 32, 0};
      {
        PromptSeq s;
        int nu;
        window.before = units - __shfl_sync(0xffffffffu, prompt_window(a, window, s, nu), 31);
      }
      const uint32_t qbytes = (uint32_t)(p.group * a.tpt) * 128u * PANELS;
      for (int i = 0;; ++i) {
        const long long idx = (long long)i * gridDim.x + ((i & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        PromptItem it{};
        const bool more = ok && idx < (long long)units * p.n_kv * p.splits && prompt_item(a, (int)idx, units, window, it);
        if (lane == 0 && i >= kPtInfo)  // the slot's item has been read by all; if not, it stays as it is
          ok = mbar_wait(b_ie + 8 * (i % kPtInfo), (uint32_t)((i / kPtInfo - 1) & 1), a.timeout_ns);
        if (lane == 0 && ok) {
          volatile PromptItem* r = ring + i % kPtInfo;
          r->q0 = it.q0; r->qlen = it.qlen; r->klen = it.klen;
          r->tok = it.tok; r->kvh = it.kvh; r->part = it.part; r->key0 = it.key0;
          r->n[0] = it.n[0]; r->n[1] = it.n[1]; r->tail = it.tail;
          r->nbm = more ? it.nbm : -1;
          mbar_arrive(b_if + 8 * (i % kPtInfo));
          // tile w of the item (K(0) V(0) K(1) V(1) ...) into the next slot, on the load's barrier, which expects
          // what has been issued and no more: `loaded` ends its phase, after a failure too
          auto load_kv = [&](int w) {
            if (n >= NS) {  // the load that used the slot before has been consumed
              const uint32_t was = slot_load[sl];
              if (!mbar_wait(b_empty + 8 * (was % NP), (was / NP) & 1, a.timeout_ns)) {
                ok = false;
                return;
              }
            }
            slot_load[sl] = g;
            mbar_expect_tx(b_full + 8 * (g % NP), TILE);
            for (int c = 0; c < PANELS; ++c)
              tma_load_3d(sKV + sl * TILE + c * PANEL, (w & 1) ? &mv : &mk, 64 * c, it.kvh,
                          it.k0 + it.key0 + (w >> 1) * kPtKeys, b_full + 8 * (g % NP));
            ++n;
            if (++sl == NS) sl = 0;
          };
          auto loaded = [&]() {
            mbar_arrive(b_full + 8 * (g % NP));
            ++g;
          };
          if (more && it.nbm > 0) {
            load_kv(0);
            loaded();
            // Q: its buffers are free when the last scores of the previous item are done
            if (ok && nq > 0 && !mbar_wait(b_qe, (uint32_t)((nq - 1) & 1), a.timeout_ns)) ok = false;
            if (ok) {
              mbar_arrive_expect_tx(b_qf, (it.n[0] > 0 ? qbytes : 0) + (it.n[1] > 0 ? qbytes : 0));
              for (int t = 0; t < 2; ++t)
                if (it.n[t] > 0)
                  for (int c = 0; c < PANELS; ++c)
                    tma_load_3d(sQ + t * TILE + c * PANEL, &mq, 64 * c, it.kvh * p.group, it.q0 + it.tok + t * a.tpt, b_qf);
              ++nq;
            }
            for (int j = 0; j < it.nbm && ok; ++j) {  // V(j) and K(j + 1)
              load_kv(2 * j + 1);
              if (j + 1 < it.nbm && ok) load_kv(2 * j + 2);
              loaded();
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!more || !ok) break;
      }
      // everything issued lands before the CTA may exit, whatever has failed; if nothing has, it is used too, and the
      // MMA warp's arrivals that say so have come
      if (lane == 0) {
        const uint32_t e0 = g > NP ? g - NP : 0;
        bool landed = true;
        for (uint32_t e = e0; e < g; ++e) landed &= mbar_wait(b_full + 8 * (e % NP), (e / NP) & 1, kPtDrainNs);
        if (nq > 0) landed &= mbar_wait(b_qf, (uint32_t)((nq - 1) & 1), kPtDrainNs);
        ok = ok && landed;
        for (uint32_t e = e0; e < g && ok; ++e) ok = mbar_wait(b_empty + 8 * (e % NP), (e / NP) & 1, a.timeout_ns);
        if (ok && nq > 0) ok = mbar_wait(b_qe, (uint32_t)((nq - 1) & 1), a.timeout_ns);
        if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---------------- MMA issue (all lanes run the loops, see elect_one) ----------------
      // The tensor cores queue about two MMAs beyond the running one and a wait costs 100 cycles or more even when
      // it is over, so the issuer's waits are few: one for V(j) and K(j + 1) together, then the weights.
      constexpr uint32_t id_s = umma_idesc<T>(128, 128), id_o = umma_idesc<T>(128, HD) | kIdescBMajorMN;
      const uint64_t q_desc = umma_desc_sw128(sQ), k_desc = umma_desc_sw128(sKV), v_desc = umma_desc_mn128(sKV, PANEL);
      auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.timeout_ns)); };
      bool ok = true;
      int sl = 0;                         // slot of the next K / V tile
      uint32_t g = 0, nq = 0, nfix = 0;   // loads of K / V, Q loads and fixed tails so far
      uint32_t np[2] = {0, 0}, no[2] = {0, 0};  // P blocks and outputs of each tile so far
      auto scores = [&](int t, int slot) {      // S_t = Q_t K^T
        const uint64_t qd = q_desc + (uint64_t)(t * (TILE >> 4)), kd = k_desc + (uint64_t)(slot * (TILE >> 4));
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t o = (uint64_t)(((kk >> 2) * PANEL + (kk & 3) * 32) >> 4);
            umma_f16(tmem + 128 * t, qd + o, kd + o, id_s, kk ? 1u : 0u);
          }
          umma_commit(b_s + 8 * t);
        }
        __syncwarp();
      };
      for (int i = 0; ok; ++i) {
        ok = __all_sync(0xffffffffu, item_wait(i));
        if (!ok) break;
        const volatile PromptItem* r = ring + i % kPtInfo;
        const int nbm = __shfl_sync(0xffffffffu, r->nbm, 0), n0 = __shfl_sync(0xffffffffu, r->n[0], 0);
        const int n1 = __shfl_sync(0xffffffffu, r->n[1], 0), tail = __shfl_sync(0xffffffffu, r->tail, 0);
        if (lane == 0) item_done(i);
        __syncwarp();
        if (nbm < 0) break;
        if (nbm == 0) continue;
        ok = wait(b_qf, nq & 1) && wait(b_full + 8 * (g % NP), (g / NP) & 1);
        if (!ok) break;
        ++nq;
        tc_fence_after();
        if (n0 > 0) scores(0, sl);
        if (n1 > 0) scores(1, sl);
        if (elect_one()) {
          umma_commit(b_empty + 8 * (g % NP));
          if (nbm == 1) umma_commit(b_qe);
        }
        __syncwarp();
        ++g;
        for (int j = 0; j < nbm; ++j, ++g) {
          const int vs = sl + 1 == NS ? 0 : sl + 1, ks = vs + 1 == NS ? 0 : vs + 1;  // V(j) and K(j + 1)
          ok = wait(b_full + 8 * (g % NP), (g / NP) & 1);
          if (!ok) break;
          if (lane == 0) *beat = g;
          bool fix = j + 1 == nbm && tail < kPtKeys;
          if (fix && lane == 0) mbar_arrive(b_req);
          __syncwarp();
          const uint64_t vd = v_desc + (uint64_t)(vs * (TILE >> 4));
          if (SEP) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (!ok || j + 1 >= (t ? n1 : n0)) continue;
              ok = wait(b_sf + 8 * t, np[t] & 1);  // S(j) is in the softmax's registers
              tc_fence_after();
              if (ok) scores(t, ks);
            }
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int nt = t ? n1 : n0;
            if (!ok || j >= nt) continue;
            // O of the tile's previous item has been read
            if (j == 0 && no[t] > 0) ok = wait(b_of + 8 * t, (no[t] - 1) & 1);
            if (ok && fix) {
              ok = wait(b_fix, nfix & 1);
              ++nfix;
              fix = false;
            }
#pragma unroll
            for (int h = 0; h < PARTS; ++h) {  // O_t += P_t V(j)
              ok = ok && wait(b_p + 16 * h + 8 * t, np[t] & 1);
              tc_fence_after();
              if (ok && elect_one()) {
#pragma unroll
                for (int kk = 8 / PARTS * h; kk < 8 / PARTS * (h + 1); ++kk)
                  umma_f16_ts(tmem + 256 + OC * t, tmem + (SEP ? 384 + 64 * t : 128 * t) + 8 * kk,
                              vd + (uint64_t)((kk * 2048) >> 4), id_o, (j | kk) ? 1u : 0u);
                if (h == PARTS - 1 && (SEP || j + 1 == nt)) umma_commit(b_o + 8 * t);
              }
              __syncwarp();
            }
            ++np[t];
            if (ok && !SEP && j + 1 < nt) scores(t, ks);
            if (j + 1 == nt) ++no[t];
          }
          if (!ok) break;
          if (elect_one()) {
            umma_commit(b_empty + 8 * (g % NP));
            if (j + 2 == nbm) umma_commit(b_qe);
          }
          __syncwarp();
          sl = ks;
        }
      }
      if (!ok) {  // what has been issued completes before the memory it works on is given back
        if (lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
        __syncwarp();
        if (elect_one()) umma_commit(b_end);
        mbar_wait(b_end, 0, kPtDrainNs);
        __syncwarp();
      }
    } else if (warp == 10) {
      // ---------------- V rows past the sequence's end ----------------
      int n = 0, nfix = 0;
      uint32_t g = 0;
      for (int i = 0;; ++i) {
        bool ok = item_wait(i);
        const volatile PromptItem* r = ring + i % kPtInfo;
        const int nbm = r->nbm, tail = r->tail;
        __syncwarp();
        if (lane == 0) item_done(i);
        if (!__all_sync(0xffffffffu, ok) || nbm < 0) break;
        if (nbm == 0) continue;
        n += 2 * nbm;
        g += nbm + 1;
        if (tail == kPtKeys) continue;
        // not before the MMA warp has come to the block: earlier, the barrier's parity may be an older load's
        ok = wait_walk(b_req, (uint32_t)(nfix++ & 1)) &&
             mbar_wait(b_full + 8 * ((g - 1) % NP), ((g - 1) / NP) & 1, a.timeout_ns);
        if (!__all_sync(0xffffffffu, ok)) break;
        const uint32_t v = sKV + (uint32_t)((n - 1) % NS) * TILE;
        for (int e = lane; e < (kPtKeys - tail) * 8 * PANELS; e += 32) {
          const int row = tail + e / (8 * PANELS), c = e % (8 * PANELS);
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + (c >> 3) * PANEL + row * 128 + (c & 7) * 16),
                       "r"(0)
                       : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(b_fix);
      }
    }
  } else {
    // ---------------- softmax and output ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPtRegsSoft));
    const int t = warp >> 2, q4 = warp & 3, r = 32 * q4 + lane;
    const int rtok = r / p.group, rhead = r - rtok * p.group;
    const uint32_t ts = tmem + 128 * t + ((uint32_t)(32 * q4) << 16), to = tmem + 256 + OC * t + ((uint32_t)(32 * q4) << 16);
    const uint32_t tp = SEP ? tmem + 384 + 64 * t + ((uint32_t)(32 * q4) << 16) : ts;
    int ns = 0, no = 0;  // score blocks and commits of O (per block when SEP, else per item) so far
    bool ok = true;
    for (int i = 0; ok; ++i) {
      ok = __all_sync(0xffffffffu, item_wait(i));
      if (!ok) break;
      const volatile PromptItem* it = ring + i % kPtInfo;
      if (it->nbm < 0) break;
      const int nt = it->n[t], qlen = it->qlen, klen = it->klen, key0 = it->key0;
      const int tok = it->tok + t * a.tpt + rtok, head = it->kvh * p.group + rhead;
      const int out_row = it->q0 + tok;
      const int part = it->part;
      __syncwarp();
      if (lane == 0) item_done(i);
      const bool mine = rtok < a.tpt && tok < qlen;
      const int lim = (p.causal ? min(klen, klen - qlen + tok + 1) : klen) - key0;  // keys of this part the row sees
      float m = -INFINITY, top = -INFINITY, l = 0.f;  // top: the score at which m moves
      for (int j = 0; j < nt; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(b_s + 8 * t, (uint32_t)(ns & 1), a.timeout_ns));
        if (!ok) break;
        ++ns;
        tc_fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, v[c]);
        tmem_wait_ld();
        if (SEP) {  // the whole of S is in registers: the next scores may be written
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(b_sf + 8 * t);
        }
        const int left = lim - j * kPtKeys;
        if (__any_sync(0xffffffffu, left < kPtKeys)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int n = left - 32 * c;
            if (__any_sync(0xffffffffu, n < 32)) {  // a bit per key: one predicated move a value instead of a comparison too
              const uint32_t seen = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen >> e & 1u)) v[c][e] = 0xff800000u;
            }
          }
        }
        float x[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[c] = fmaxf(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]));
#pragma unroll
          for (int e = 2; e < 32; e += 2) x[c] = max3(x[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
        }
        const float mx = fmaxf(max3(x[0], x[1], x[2]), x[3]) * p.scale_log2;
        float f = 1.f;
        if (mx > top) {  // also from -inf, with f = 0: nothing to rescale yet
          const float to = prompt_reference<T, 7>(mx);
          f = ex2(m - to);
          m = to;
          top = mx + 8.f;
        }
        const bool rescale = __any_sync(0xffffffffu, f != 1.f) && j > 0;
        if (SEP && j > 0) {  // O += P(j-1) V(j-1) is done: P may be written, O rescaled
          ok = __all_sync(0xffffffffu, mbar_wait(b_o + 8 * t, (uint32_t)((no - 1) & 1), a.timeout_ns));
          if (!ok) break;
          tc_fence_after();
        }
        if (SEP) ++no;
        if (rescale) {
#pragma unroll 1
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(to + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(to + 16 * c, o);
          }
          tmem_wait_st();
        }
        const float neg = m == -INFINITY ? 0.f : -m;
        const uint64_t sc2 = both(p.scale_log2), neg2 = both(neg);
        uint64_t sum[4] = {0, 0, 0, 0};
        // weights of the block, 64 keys at a time: the products with the first half start under the second
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            uint32_t y0, y1;
            unpack64(fma2f(pack64(v[c][e], v[c][e + 1]), sc2, neg2), y0, y1);
            const float w0 = ex2(__uint_as_float(y0)), w1 = ex2(__uint_as_float(y1));
            sum[c] = add2f(sum[c], pack64(__float_as_uint(w0), __float_as_uint(w1)));
            v[c >> 1][(c & 1) * 16 + e / 2] = Act<T>::pack2(w0, w1);
          }
          if (c & 1) tmem_st32(tp + 32 * (c >> 1), v[c >> 1]);
          if (c == 3 || (PARTS == 2 && c == 1)) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_p + 16 * (PARTS - 1 ? c >> 1 : 0) + 8 * t);
          }
        }
        {
          const uint64_t s2 = add2f(add2f(sum[0], sum[1]), add2f(sum[2], sum[3]));
          uint32_t s0, s1;
          unpack64(s2, s0, s1);
          l = l * f + (__uint_as_float(s0) + __uint_as_float(s1));
        }
      }
      if (!ok) break;
      if (nt > 0) {
        if (!SEP) ++no;
        ok = __all_sync(0xffffffffu, mbar_wait(b_o + 8 * t, (uint32_t)((no - 1) & 1), a.timeout_ns));
        if (!ok) break;
      }
      tc_fence_after();
      const bool whole = p.splits == 1;
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
      const long long at = ((long long)part * p.tq + out_row) * p.n_q + head;
      if (!whole && mine) *reinterpret_cast<float2*>(p.stat + 2 * at) = make_float2(m, l);
      // the element a lane's row starts at, -1 for a row that is not there
      const long long row_at = mine ? (long long)out_row * p.o_tok + head * p.o_head : -1;
      const uint32_t stg = sb + pt_off_out<HD>() + warp * 4096;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          if (nt > 0) {
            tmem_ld32(to + 64 * c + 32 * h, o);
            tmem_wait_ld();
            if (c == HD / 64 - 1 && h == 1) {  // O has been read: the next item may start over
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(b_of + 8 * t);
            }
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = l == 0.f ? 0u
                                : Act<T>::pack2(__uint_as_float(o[8 * e + 2 * k]) * inv,
                                                __uint_as_float(o[8 * e + 2 * k + 1]) * inv);
              asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stg + sw128(lane, 4 * h + e)), "r"(w[0]),
                           "r"(w[1]), "r"(w[2]), "r"(w[3])
                           : "memory");
            }
          } else if (mine && l != 0.f) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(p.part + at * HD + 64 * c + 32 * h + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (whole) {
          // 64 columns of the warp's rows from shared memory: a lane's own row would be 16 bytes of 32 lines a store
          __syncwarp();
          long long base[8];
          uint4 line[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int rr = 4 * e + (lane >> 3);
            base[e] = __shfl_sync(0xffffffffu, row_at, rr);
            line[e] = lds16(stg + sw128(rr, lane & 7));
          }
          T* out = reinterpret_cast<T*>(p.out) + 64 * c + 8 * (lane & 7);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (base[e] >= 0) *reinterpret_cast<uint4*>(out + base[e]) = line[e];
          __syncwarp();
        }
      }
    }
    if (!ok && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();  // every MMA has completed (the outputs or the MMA warp waited for them) and every TMEM read is done
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ee
