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
// CTAs (a snake, from the last sequence's last rows up: longest items first within
// a causal prompt, but a batch's sequences in their order, whatever their lengths),
// and the next item's loads and first
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

#include "ee_cache.cuh"
#include "ee_prompt.cuh"
#include "ee_tma.cuh"
#include "ee_umma.cuh"

namespace ee {

struct PromptTcArgs {
  PromptArgs p;
  int tpt;  // tokens per tile: 128 / group
  int* status;
  unsigned long long timeout_ns;
  CacheView c;  // keys and values in a cache
  const float *k_steps, *v_steps;
  PromptMore more;  // JOIN
};

// registers: 384 threads launch with 168 each; the four warps of loads and MMAs
// give theirs up to 88 and the softmax warps take 208 (256 x 208 + 128 x 88 =
// 384 x 168), so that a whole row of S stays in registers. With four more warps
// that decode a cache's codes 512 threads launch with 128, and the shares are
// 200, 72 and 40.
template <int BITS> struct PtThreads {
  static constexpr int N = BITS ? 512 : 384, LAUNCH = BITS ? 128 : 168;
  static constexpr int SOFT = BITS ? 200 : 208, REST = BITS ? 72 : 88, DECODE = BITS ? 40 : 0;
  static_assert(256 * SOFT + 128 * REST + 128 * DECODE <= N * LAUNCH, "the register shares fit the launch");
};
constexpr int kPtKeys = 128, kPtInfo = 4, kPtLoads = 8;  // keys per block; items published, loads of K / V ahead
constexpr unsigned long long kPtDrainNs = 1000000000ull;  // for loads and MMAs already issued, whatever timeout_ns is
// Shared memory: Q of both tiles, the slots of K / V, output staging of every
// softmax warp, barriers, published items; for a cache also the ring of codes
// as they come, and the steps of the blocks.
template <int HD, int BITS> constexpr int pt_slots() { return BITS ? 4 : (HD == 128 ? 4 : 8); }
constexpr int kPtSlotsK = 2;  // of a cache's: K, the others V
template <int BITS> constexpr int pt_tiles() { return BITS ? 1 : 2; }  // tiles of rows in an item
template <int HD> constexpr uint32_t pt_tile() { return 128u * HD * 2; }
template <int BITS> constexpr uint32_t pt_stage() { return BITS ? 0u : 4096u; }  // bytes of a warp's output staging
template <int HD, int BITS> constexpr uint32_t pt_raw() { return 128u * HD * BITS / 8; }  // codes of a tile
// tiles of codes on their way: 40 to 48 KB where they are large (with 32 KB an SM waited for them)
template <int HD, int BITS> constexpr int pt_raws() { return !BITS ? 0 : HD * BITS == 1024 ? 3 : HD * BITS == 512 ? 5 : 6; }
constexpr int kPtSteps = 4;  // blocks whose steps are held: of K, of V, and the powers of two that fp16 values take
constexpr uint32_t kPtStepBytes = 3 * 128 * 4;
template <int HD, int BITS> constexpr uint32_t pt_off_raw() { return (pt_tiles<BITS>() + pt_slots<HD, BITS>()) * pt_tile<HD>(); }
template <int HD, int BITS> constexpr uint32_t pt_off_out() { return pt_off_raw<HD, BITS>() + pt_raws<HD, BITS>() * pt_raw<HD, BITS>(); }
template <int HD, int BITS> constexpr uint32_t pt_off_rawsteps() { return pt_off_out<HD, BITS>() + 8 * pt_stage<BITS>(); }
template <int HD, int BITS> constexpr uint32_t pt_off_steps() { return pt_off_rawsteps<HD, BITS>() + pt_raws<HD, BITS>() * 1024u; }
template <int HD, int BITS> constexpr uint32_t pt_off_bar() { return pt_off_steps<HD, BITS>() + (BITS ? kPtSteps * kPtStepBytes : 0u); }
// barriers: full / empty per load of K / V, Q full / empty, S / P (two halves) / S free / O / O free per tile, V to fix /
// fixed, item full / empty, MMAs done after a failure; of a cache the other half's sums (twice), steps full, codes full /
// empty. (There full / empty are a slot's, K and V by themselves.)
template <int HD, int BITS> constexpr uint32_t pt_off_info() {
  return pt_off_bar<HD, BITS>() + 8 * (2 * kPtLoads + 19 + kPtSteps + 2 * kPtInfo + 2 * pt_raws<HD, BITS>()) + 8;
}
template <int HD, int BITS> constexpr uint32_t pt_off_beat() { return pt_off_info<HD, BITS>() + kPtInfo * 64; }  // blocks the MMA warp has come to
// which keys of a block are there (4 words a block), which pieces of a tile of codes
template <int HD, int BITS> constexpr uint32_t pt_off_there() { return pt_off_beat<HD, BITS>() + 16; }
template <int HD, int BITS> constexpr uint32_t pt_off_odd() {  // which values of a block leave other factors to the weight than below 2
  return pt_off_there<HD, BITS>() + (BITS ? kPtSteps * 16 + (pt_raws<HD, BITS>() * 4 + 15) / 16 * 16 : 0);
}
template <int HD, int BITS> constexpr uint32_t pt_off_half() {  // one tile's maxima and sums for the other, of two items
  return pt_off_odd<HD, BITS>() + (BITS ? kPtSteps * 16 : 0);
}
template <int HD, int BITS> constexpr uint32_t pt_smem() { return pt_off_half<HD, BITS>() + (BITS ? 2048 : 0) + 1024; }

// One published item (16 words)
struct PromptItem {
  int q0, qlen, k0, klen;  // the sequence (k0: its first key row)
  int tok, kvh, part;      // first token of tile 0, key head, part of the keys
  int key0;                // first key of this part
  int n[2];                // key blocks of the tiles in this part
  int tail;                // valid keys of the part's last block (128: all)
  int nbm;                 // blocks of keys: max(n[0], n[1]), or their sum where the tiles alternate; -1: no more items
  int turn;                // a cache's items: block j is for the softmax and the columns of "tile" (j + turn) mod 2
  int pad[3];
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
template <int BITS>
EE_DEV int prompt_window(const PromptTcArgs& a, const PromptWindow& w, PromptSeq& s, int& nu) {
  const int lane = threadIdx.x & 31, b = w.base + lane;
  s = PromptSeq{};
  if (b < a.p.n_seq) s = prompt_seq(a.p, b);
  nu = (s.qlen + pt_tiles<BITS>() * a.tpt - 1) / (pt_tiles<BITS>() * a.tpt);
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
template <int BITS>
EE_DEV bool prompt_item(const PromptTcArgs& a, int idx, int units, PromptWindow& w, PromptItem& it) {
  const PromptArgs& p = a.p;
  const int per = p.n_kv * p.splits;
  const int unit = units - 1 - idx / per;
  if (unit < 0) return false;
  it.kvh = idx % per / p.splits;
  it.part = idx % p.splits;
  PromptSeq s;
  int nu, inc = prompt_window<BITS>(a, w, s, nu);
  while (unit < w.before && w.base > 0) {
    w.base -= 32;
    inc = prompt_window<BITS>(a, w, s, nu);
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
  it.tok = (unit - __shfl_sync(0xffffffffu, inc - nu, src)) * pt_tiles<BITS>() * a.tpt;
  int nb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = it.tok + t * a.tpt, last = min(first + a.tpt, it.qlen);
    const int kend = p.causal ? min(max(it.klen - it.qlen + last, 0), it.klen) : it.klen;
    nb[t] = t < pt_tiles<BITS>() && first < it.qlen ? (kend + kPtKeys - 1) / kPtKeys : 0;
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

// BITS 0: K and V of 16 bits. 8 or 4: codes from a paged cache, with 512 threads.
// Warp 10 finds the items; warp 8 looks up their pages and brings codes (TMA, a
// box per piece of a page) and steps (bulk copies) into a ring, 128 keys at a
// time; warps 12-15 turn them into 16-bit tiles in the slots, exactly, two of K
// and two of V, and hand on the steps. A key's step multiplies its column of S,
// a value's its column of P after the sum is taken, so the weights that P V
// rounds are the products. That product is in fp16 whatever the call's type, for
// the weights' 11 bits: the values are code times a power of two, exactly, and the
// weights take what that leaves of the step, a factor below 2 (or, for values
// beyond fp16's largest number and far below its smallest, the rest too: see where
// the reference moves). In bf16 the result's rounding is eight times the weights',
// with weights in bf16 the two together were 1.4 times it, and in rows of few keys
// one factor for all dims; in fp16 the two are of one size. Weights that end below
// 2^-14 lose up to 2^-25 each beside a largest one of 2^7 or more. (Weights in bf16
// took 119 and 179 us where these take 116 and 187; two products of them, 139 and 217.)
//
// There an item is one tile, as a call's sequences rarely have two (50 tokens a
// turn): its blocks take turns on the two halves' softmax warps and columns of
// TMEM, from where the item before stopped, so one half's softmax runs under the
// other's products as two tiles' would; the half with the last block adds the
// other's sums and finishes the rows. (Items of two tiles, the second's half at
// the first's keys where it is empty: 150 and 207 us where this took 129 and 184
// in the first two cases below.)
//
// Measured, heads of 128, 8 bits: 64 x 50 tokens behind 257 to 816, 16 heads: 116
// us; 4 x 500 to 1024 behind 1 to 4096, 16 / 4 heads: 187, 525 TFLOP/s; with keys
// and values in 16 bits: 88 and 134. Without decoding, steps and exponentials the
// rest takes 86 and 117: what bounds it is the round trip of scores, softmax and
// products of a lone tile, whose 50 rows are two warps of four, then the decoding
// (2 x 128 x 128 codes a block by four warps) and the steps' multiplications; and
// the uneven end: the fullest CTA has 42 blocks where 35.2 are the mean, and 100 where
// 81.4 are. Not
// faster: K and V decoded by two warps each (118 -> 136), S read twice by halves,
// without spills (118 -> 130, 179 -> 200).
//
// JOIN: the call's rows as one sequence over 16-bit keys, and other sums of theirs
// (a.more, left by the kernel before this one) are added where they are finished.
template <typename T, int HD, int BITS = 0, bool JOIN = false>
__global__ void __launch_bounds__(PtThreads<BITS>::N, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptTcArgs a) {
  constexpr int NS = pt_slots<HD, BITS>(), NP = kPtLoads, NR = pt_raws<HD, BITS>(), KS = kPtSlotsK, VS = NS - KS;
  static_assert(NS <= NP, "a barrier per load that the slots can hold");
  static_assert(pt_smem<HD, BITS>() <= 227 * 1024, "an SM's shared memory");
  constexpr uint32_t TILE = pt_tile<HD>(), PANEL = 128 * 128;  // a panel: 64 columns of 128 rows
  constexpr int PANELS = HD / 64;
  // hd 64 leaves TMEM for P beside S, so the next scores are computed during the softmax
  constexpr bool SEP = HD == 64;
  // pieces in which a block's weights are handed over (in one piece, hd 64: 501 instead of 411 us for 8192 tokens)
  constexpr int PARTS = 2;
  using PT = typename std::conditional<BITS != 0, __half, T>::type;  // what P and V are in their product
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sQ = sb, sKV = sb + pt_tiles<BITS>() * TILE;
  const uint32_t b_full = sb + pt_off_bar<HD, BITS>(), b_empty = b_full + 8 * NP;
  const uint32_t b_qf = b_empty + 8 * NP, b_qe = b_qf + 8, b_s = b_qe + 8, b_p = b_s + 16, b_sf = b_p + 32, b_o = b_sf + 16;
  const uint32_t b_of = b_o + 16, b_req = b_of + 16, b_fix = b_req + 8, b_if = b_fix + 8, b_ie = b_if + 8 * kPtInfo;
  const uint32_t b_end = b_ie + 8 * kPtInfo, b_half = b_end + 8, b_st = b_half + 16, b_rf = b_st + 8 * kPtSteps, b_re = b_rf + 8 * NR, off_tm = b_re + 8 * NR - sb;
  volatile PromptItem* ring = reinterpret_cast<volatile PromptItem*>(smem + pt_off_info<HD, BITS>());
  volatile uint32_t* beat = reinterpret_cast<volatile uint32_t*>(smem + pt_off_beat<HD, BITS>());
  const PromptArgs& p = a.p;
  if (warp == 8 && lane == 0) {
    tma_prefetch_map(&mq);
    tma_prefetch_map(&mk);
    tma_prefetch_map(&mv);
    for (int s = 0; s < NP; ++s) {
      mbar_init(b_full + 8 * s, BITS ? 4 : 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    for (int s = 0; s < NR; ++s) {
      mbar_init(b_rf + 8 * s, 1);
      mbar_init(b_re + 8 * s, 4);
    }
    mbar_init(b_req, 1);
    mbar_init(b_fix, 1);
    mbar_init(b_qf, 1);
    mbar_init(b_qe, 1);
    mbar_init(b_end, 1);
    mbar_init(b_half, 4);
    mbar_init(b_half + 8, 4);
    for (int i = 0; i < kPtSteps; ++i) mbar_init(b_st + 8 * i, 4);
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
      mbar_init(b_ie + 8 * i, BITS ? 14 : 10);  // 8 softmax warps, the MMA warp, the fixing warp or the loading and decoding ones
    }
    mbar_fence_init();
  }
  // JOIN: what is read before the rows are finished is older than the kernel this one follows, which waited for it. A
  // CTA's first item runs beside that kernel's last ones; its end, however far, is waited for without a limit by every
  // warp before its second item (the softmax warps: before they finish rows), so no bounded wait counts it
  if (JOIN) pdl_release();
  else pdl_entry();
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

  if (BITS > 0 && warp >= 12) {
    if constexpr (BITS > 0) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PtThreads<BITS>::DECODE));
      // ---------------- codes into 16-bit tiles: 32 keys of each by a warp ----------------
      constexpr int RB = HD * BITS / 8;                    // bytes of a row of codes
      constexpr int PER_ROW = RB < 64 ? RB / 16 : 4;       // lanes on a row; a row of 128 bytes takes two of its pieces
      constexpr int ROWS = 32 / PER_ROW, HALVES = RB / 16 / PER_ROW, PIECES = 32 / ROWS * HALVES;
      // pieces under way at once, in a loop: unrolled whole, the two ways of decoding and the softmax do not fit the
      // instruction cache together (bf16, heads of 128: 64 x 50 tokens 137 us, 4 x 500..1024 192; so 116 and 187; of 64
      // with one, 99 and 167, with two 102 and 165)
      constexpr int BATCH = PIECES < 8 ? 1 : 2;
      const int quarter = warp - 12, row0 = 32 * quarter + lane / PER_ROW, q0 = lane % PER_ROW;
      const uint32_t from = sb + pt_off_raw<HD, BITS>() + row0 * RB + q0 * 16;
      uint32_t to[16 / BITS];  // where the 16-bit pieces of the lane's first piece go
#pragma unroll
      for (int k = 0; k < 16 / BITS; ++k) {
        const int c = q0 * (16 / BITS) + k;
        to[k] = sKV + (c >> 3) * PANEL + sw128(row0, c & 7);
      }
      uint32_t rt = 0, nk = 0, nv = 0;  // tiles of codes, of K and of V so far
      bool ok = true;
      for (int i = 0;; ++i) {
        ok = __all_sync(0xffffffffu, item_wait(i));
        if (!ok) break;
        const volatile PromptItem* r = ring + i % kPtInfo;
        const int nbm = r->nbm, klen = r->klen, key0 = r->key0;
        __syncwarp();
        if (lane == 0) item_done(i);
        if (nbm < 0) break;
        for (int x = 0; x < 2 * nbm && ok; ++x) {  // K(0) K(1) V(0) K(2) V(1) ... V(nbm - 1)
          const bool isv = x == 2 * nbm - 1 || (x > 0 && (x & 1) == 0);
          const uint32_t rs = rt % NR, blk = isv ? nv : nk, slots = isv ? VS : KS, at = isv ? KS + blk % VS : blk % KS;
          const int j = (x + 1) / 2;  // K's block
          ok = mbar_wait(b_rf + 8 * rs, (rt / NR) & 1, a.timeout_ns);
          // the products of the tile that used the slot before are done
          if (ok && blk >= slots) ok = mbar_wait(b_empty + 8 * at, (blk / slots - 1) & 1, a.timeout_ns);
          float* steps = reinterpret_cast<float*>(smem + pt_off_steps<HD, BITS>() + (blk % kPtSteps) * kPtStepBytes);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (!isv) {
            const float* raw_steps = reinterpret_cast<const float*>(smem + pt_off_rawsteps<HD, BITS>() + rs * 1024);
            const uint32_t there = *reinterpret_cast<volatile uint32_t*>(smem + pt_off_there<HD, BITS>() + kPtSteps * 16 + rs * 4);
            const int shift = min(a.c.shift, 7);
            const int key = 32 * quarter + lane;
            const bool have = key0 + j * kPtKeys + key < klen && (there >> (key >> shift) & 1);
            float ks = have ? raw_steps[key] : 0.f, vs = have ? raw_steps[128 + key] : 0.f;
            // a value's step that is no number must reach the rows that see it and no others: as its key's
            if (!(fabsf(vs) <= 3.4028234e38f)) {
              ks = __int_as_float(0x7fffffff);
              vs = 0.f;
            }
            steps[key] = ks * (p.scale_log2 * code_unit<T, BITS>());
            // 2^e to the values, exactly: e from -24, where fp16 ends, to where its largest number holds any code
            const int e = min(max(((__float_as_int(vs) >> 23) & 0xff) - 127, -24), BITS == 8 ? 8 : 12);
            const __half2 v2 = __float2half2_rn(__int_as_float((127 + e) << 23));
            vs *= __int_as_float((127 - e) << 23);
            steps[128 + key] = vs;
            steps[256 + key] = __uint_as_float(*reinterpret_cast<const uint32_t*>(&v2));
            const uint32_t all = __ballot_sync(0xffffffffu, have);
            const uint32_t odd = __ballot_sync(0xffffffffu, fabsf(vs) >= 2.f || (fabsf(vs) < 0.00390625f && vs != 0.f));
            if (lane == 0) {
              *reinterpret_cast<volatile uint32_t*>(smem + pt_off_there<HD, BITS>() + (blk % kPtSteps) * 16 + quarter * 4) = all;
              *reinterpret_cast<volatile uint32_t*>(smem + pt_off_odd<HD, BITS>() + (blk % kPtSteps) * 16 + quarter * 4) = odd;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(b_st + 8 * (blk % kPtSteps));
          }
          const uint32_t raw = from + rs * pt_raw<HD, BITS>(), dst = at * TILE;
          auto decode = [&](auto type, auto value) {
            using U = decltype(type);
#pragma unroll 1
            for (int e0 = 0; e0 < PIECES; e0 += BATCH) {
              uint4 x[BATCH];
#pragma unroll
              for (int u = 0; u < BATCH; ++u) x[u] = lds16(raw + (e0 + u) / HALVES * (ROWS * RB) + (e0 + u) % HALVES * 64);
              uint32_t by[BATCH];
#pragma unroll
              for (int u = 0; u < BATCH; ++u)
                if (decltype(value)::value) by[u] = __float_as_uint(steps[256 + row0 + (e0 + u) / HALVES * ROWS]);
#pragma unroll
              for (int u = 0; u < BATCH; ++u) {
                const int e = e0 + u;
                const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                uint32_t o[64 / BITS];  // pairs
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  if (BITS == 8) {
                    const uint32_t f = xw[k] ^ 0x80808080u;
                    o[2 * k] = code_pair8<U>(f, 0);
                    o[2 * k + 1] = code_pair8<U>(f, 1);
                  } else {
#pragma unroll
                    for (int b = 0; b < 4; ++b) o[4 * k + b] = code_pair4<U>(xw[k], xw[k] >> 4, b);
                  }
                }
                if (decltype(value)::value) {
#pragma unroll
                  for (int k = 0; k < 64 / BITS; ++k) o[k] = fma2<U>(o[k], by[u], 0u);
                }
#pragma unroll
                for (int k = 0; k < 16 / BITS; ++k)
                  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to[k] + dst + e / HALVES * (ROWS * 128) +
                                                                                e % HALVES * PANEL),
                               "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]), "r"(o[4 * k + 3])
                               : "memory");
              }
            }
          };
          if (isv) decode(PT(), std::true_type());
          else decode(T(), std::false_type());
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(b_re + 8 * rs);
            mbar_arrive(b_full + 8 * at);
          }
          ++rt;
          if (isv) ++nv; else ++nk;
        }
        if (!ok) break;
      }
      // the MMA warp's arrivals that say the tiles are used have come
      if (quarter == 0 && lane == 0) {
        for (int v = 0; v < 2; ++v) {
          const uint32_t slots = v ? VS : KS, n = v ? nv : nk;
          for (uint32_t e = n > slots ? n - slots : 0; e < n && ok; ++e)
            ok = mbar_wait(b_empty + 8 * ((v ? KS : 0) + e % slots), (e / slots) & 1, a.timeout_ns);
        }
      }
      if (!ok && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
      __syncwarp();
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PtThreads<BITS>::REST));
    if (warp == (BITS ? 10 : 8)) {
      // ---------------- items, and loads but for a cache's ----------------
      bool ok = true;
      int units = 0, n = 0, nq = 0, sl = 0;  // K / V tiles and Q loads issued so far, next slot
      int bs = 0;                            // blocks so far (cache)
      uint32_t g = 0, slot_load[NS];         // loads (barrier phases) of K / V so far, and each slot's last one
#pragma unroll 4
      for (int b = lane; b < p.n_seq; b += 32) units += (prompt_seq(p, b).qlen + pt_tiles<BITS>() * a.tpt - 1) / (pt_tiles<BITS>() * a.tpt);
      units = __reduce_add_sync(0xffffffffu, units);
      PromptWindow window{(p.n_seq - 1) / 32 * 32, 0};
      {
        PromptSeq s;
        int nu;
        window.before = units - __shfl_sync(0xffffffffu, prompt_window<BITS>(a, window, s, nu), 31);
      }
      const uint32_t qbytes = (uint32_t)(p.group * a.tpt) * 128u * PANELS;
      for (int i = 0;; ++i) {
        if (JOIN && i == 1) pdl_wait();
        const long long idx = (long long)i * gridDim.x + ((i & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        PromptItem it{};
        const bool more = ok && idx < (long long)units * p.n_kv * p.splits && prompt_item<BITS>(a, (int)idx, units, window, it);
        if (BITS) {  // the blocks of one item after another take turns on the tiles' softmax warps and columns
          it.turn = bs & 1;
          it.n[it.turn] = (it.nbm + 1) / 2;
          it.n[1 - it.turn] = it.nbm / 2;
          bs += it.nbm;
        }
        if (lane == 0 && i >= kPtInfo)  // the slot's item has been read by all; if not, it stays as it is
          ok = BITS ? wait_walk(b_ie + 8 * (i % kPtInfo), (uint32_t)((i / kPtInfo - 1) & 1))
                    : mbar_wait(b_ie + 8 * (i % kPtInfo), (uint32_t)((i / kPtInfo - 1) & 1), a.timeout_ns);
        if (lane == 0 && ok) {
          volatile PromptItem* r = ring + i % kPtInfo;
          r->q0 = it.q0; r->qlen = it.qlen; r->klen = it.klen;
          if (BITS) r->k0 = it.k0;
          r->tok = it.tok; r->kvh = it.kvh; r->part = it.part; r->key0 = it.key0;
          r->n[0] = it.n[0]; r->n[1] = it.n[1]; r->tail = it.tail;
          r->turn = it.turn;
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
          if (BITS == 0 && more && it.nbm > 0) {
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
      if (BITS && lane == 0 && !ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
      if (BITS == 0 && lane == 0) {
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
    } else if (BITS > 0 && warp == 8) {
      // ---------------- loads of Q and of the tiles' codes ----------------
      if constexpr (BITS > 0) {
      // K(0) K(1) V(0) K(2) V(1) ..., in pieces of a page; a block's steps come with its K. A lane per piece looks its page
      // up, two blocks and an item ahead.
      const int shift = min(a.c.shift, 7), pieces = kPtKeys >> shift;
      constexpr uint32_t RB = HD * BITS / 8;
      const uint32_t qbytes = (uint32_t)(p.group * a.tpt) * 128u * PANELS;
      uint32_t g = 0;  // tiles of codes so far
      int nq = 0;      // loads of Q
      bool ok = true;
      struct At {
        int q0, tok, kvh, k0, klen, key0, nbm;
      };
      auto item_at = [&](int i) {
        At x{0, 0, 0, 0, 0, 0, -1};
        ok = __all_sync(0xffffffffu, ok && item_wait(i));
        if (!ok) return x;
        const volatile PromptItem* r = ring + i % kPtInfo;
        x = At{r->q0, r->tok, r->kvh, r->k0, r->klen, r->key0, r->nbm};
        __syncwarp();
        if (lane == 0) item_done(i);
        return x;
      };
      auto page_of = [&](const At& x, int j) {  // of this lane's piece of block j, -1 for none
        const int key = x.key0 + j * kPtKeys + (lane << shift);
        if (lane >= pieces || j >= x.nbm || key >= x.klen) return -1;
        return __ldg(a.c.table + (long long)x.k0 * a.c.table_row + (key >> a.c.shift));
      };
      auto codes = [&](const At& x, int w, int j, int page) {  // K (w = 0) or V of block j
        const bool there = (unsigned)page < (unsigned)a.c.pages;
        const uint32_t mask = __ballot_sync(0xffffffffu, there), slot = g % NR;
        if (g >= (uint32_t)NR) ok = __all_sync(0xffffffffu, ok && mbar_wait(b_re + 8 * slot, (g / NR - 1) & 1, a.timeout_ns));
        if (!ok) return;
        const uint32_t bar = b_rf + 8 * slot, dst = sb + pt_off_raw<HD, BITS>() + slot * pt_raw<HD, BITS>();
        const uint32_t steps = sb + pt_off_rawsteps<HD, BITS>() + slot * 1024;
        if (lane == 0) {
          *reinterpret_cast<volatile uint32_t*>(smem + pt_off_there<HD, BITS>() + kPtSteps * 16 + slot * 4) = mask;
          mbar_arrive_expect_tx(bar, __popc(mask) * ((RB << shift) + (w == 0 ? 8u << shift : 0u)));
        }
        __syncwarp();
        if (there) {
          const int key = x.key0 + j * kPtKeys + (lane << shift);
          const int row = ((page * a.c.n_kv + x.kvh) << a.c.shift) + (key & ((1 << a.c.shift) - 1));
          tma_load_2d(dst + lane * (RB << shift), w ? &mv : &mk, 0, row, bar);
          if (w == 0) {
            bulk_load(steps + lane * (4 << shift), a.k_steps + row, 4 << shift, bar);
            bulk_load(steps + 512 + lane * (4 << shift), a.v_steps + row, 4 << shift, bar);
          }
        }
        __syncwarp();
        ++g;
      };
      At it = item_at(0), nx = it;
      int page = page_of(it, 0), next = page_of(it, 1), page2 = -1, next2 = -1;
      for (int i = 0; ok && it.nbm >= 0; ++i) {
        if (it.nbm == 0) {
          nx = item_at(i + 1);
          page2 = page_of(nx, 0);
          next2 = page_of(nx, 1);
        }
        for (int j = 0; j < it.nbm && ok; ++j) {
          if (j == 0) {
            codes(it, 0, 0, page);
            // Q: its buffer is free when the last scores of the previous item are done
            if (nq > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait(b_qe, (uint32_t)((nq - 1) & 1), a.timeout_ns));
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(b_qf, qbytes);
              for (int c = 0; c < PANELS; ++c)
                tma_load_3d(sQ + c * PANEL, &mq, 64 * c, it.kvh * p.group, it.q0 + it.tok, b_qf);
            }
            ++nq;
          }
          const int after = page_of(it, j + 2);
          if (j + 1 < it.nbm) codes(it, 0, j + 1, next);
          if (j == max(it.nbm - 2, 0)) {  // the next item's first pages, under this one's last loads
            nx = item_at(i + 1);
            page2 = page_of(nx, 0);
            next2 = page_of(nx, 1);
          }
          if (ok) codes(it, 1, j, page);
          page = next;
          next = after;
        }
        it = nx;
        page = page2;
        next = next2;
      }
      // everything issued lands before the CTA may exit, whatever has failed; if nothing has, it is used too, and the MMA
      // warp's arrival that says so of Q has come
      if (lane == 0) {
        bool landed = true;
        for (uint32_t e = g > (uint32_t)NR ? g - NR : 0; e < g; ++e) landed &= mbar_wait(b_rf + 8 * (e % NR), (e / NR) & 1, kPtDrainNs);
        if (nq > 0) landed &= mbar_wait(b_qf, (uint32_t)((nq - 1) & 1), kPtDrainNs);
        ok = ok && landed;
        if (ok && nq > 0) ok = mbar_wait(b_qe, (uint32_t)((nq - 1) & 1), a.timeout_ns);
        if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
      }
      __syncwarp();
      }
    } else if (warp == 9) {
      // ---------------- MMA issue (all lanes run the loops, see elect_one) ----------------
      // The tensor cores queue about two MMAs beyond the running one and a wait costs 100 cycles or more even when
      // it is over, so the issuer's waits are few: one for V(j) and K(j + 1) together, then the weights.
      constexpr uint32_t id_s = umma_idesc<T>(128, 128), id_o = umma_idesc<PT>(128, HD) | kIdescBMajorMN;
      const uint64_t q_desc = umma_desc_sw128(sQ), k_desc = umma_desc_sw128(sKV), v_desc = umma_desc_mn128(sKV, PANEL);
      auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.timeout_ns)); };
      bool ok = true;
      int sl = 0;                         // slot of the next K / V tile
      uint32_t g = 0, nq = 0, nfix = 0;   // loads of K / V, Q loads and fixed tails so far
      uint32_t nk = 0, nv = 0;            // tiles of K and of V (cache)
      bool begun = false;                 // the item's first scores have been issued under the item before
      uint32_t np[2] = {0, 0}, no[2] = {0, 0};  // P blocks and outputs of each tile so far
      auto scores = [&](int t, int slot, int tq) {  // S_t = Q_tq K^T
        const uint64_t qd = q_desc + (uint64_t)(tq * (TILE >> 4)), kd = k_desc + (uint64_t)(slot * (TILE >> 4));
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
        if (JOIN && i == 1) pdl_wait();
        ok = __all_sync(0xffffffffu, item_wait(i));
        if (!ok) break;
        const volatile PromptItem* r = ring + i % kPtInfo;
        const int nbm = __shfl_sync(0xffffffffu, r->nbm, 0), n0 = __shfl_sync(0xffffffffu, r->n[0], 0);
        const int n1 = __shfl_sync(0xffffffffu, r->n[1], 0), tail = __shfl_sync(0xffffffffu, r->tail, 0);
        const int turn = BITS > 0 ? __shfl_sync(0xffffffffu, r->turn, 0) : 0;
        if (lane == 0) item_done(i);
        __syncwarp();
        if (nbm < 0) break;
        if (nbm == 0) continue;
        if constexpr (BITS > 0) {
          auto product = [&](int t, bool first, bool last) {  // O_t += P_t V, V in the next slot
            const uint32_t outs = t ? no[1] : no[0], ps = t ? np[1] : np[0];
            if (first && outs > 0) ok = wait(b_of + 8 * t, (outs - 1) & 1);  // O of the tile's previous item has been read
            const uint64_t vd = v_desc + (uint64_t)((KS + nv % VS) * (TILE >> 4));
#pragma unroll
            for (int h = 0; h < PARTS; ++h) {
              ok = ok && wait(b_p + 16 * h + 8 * t, ps & 1);
              tc_fence_after();
              if (ok && elect_one()) {
#pragma unroll
                for (int kk = 8 / PARTS * h; kk < 8 / PARTS * (h + 1); ++kk)
                  umma_f16_ts(tmem + 256 + OC * t, tmem + (SEP ? 384 + 64 * t : 128 * t) + 8 * kk,
                              vd + (uint64_t)((kk * 2048) >> 4), id_o, (!first || kk) ? 1u : 0u);
                if (h == PARTS - 1 && (SEP || last)) umma_commit(b_o + 8 * t);
              }
              __syncwarp();
            }
            if (t) ++np[1]; else ++np[0];
            if (last) {
              if (t) ++no[1]; else ++no[0];
            }
          };
          // S_t = Q K^T with the next K, whose slot is free when they are there; an item's last ones free Q
          auto next_scores = [&](int t, bool end) {
            ok = ok && wait(b_full + 8 * (nk % KS), (nk / KS) & 1);
            if (!ok) return;
            tc_fence_after();
            scores(t, nk % KS, 0);
            if (elect_one()) {
              umma_commit(b_empty + 8 * (nk % KS));
              if (end) umma_commit(b_qe);
            }
            __syncwarp();
            ++nk;
          };
          if (!begun) {
            ok = wait(b_qf, nq++ & 1);
            next_scores(turn, nbm == 1);
          }
          begun = false;
          for (int j = 0; j < nbm && ok; ++j) {
            if (lane == 0) *beat = *beat + 1;
            __syncwarp();
            // S(j + 1), or the next item's S(0), in the other tile's columns: its softmax runs before P(j) is there. (The
            // other tile's last weights have been waited for, so its last scores have been read.)
            const int t = (j + turn) & 1;
            if (j + 1 < nbm) {
              next_scores(1 - t, j + 2 == nbm);
            } else {
              ok = __all_sync(0xffffffffu, item_wait(i + 1));
              const int xn = __shfl_sync(0xffffffffu, ring[(i + 1) % kPtInfo].nbm, 0);
              if (ok && xn > 0) {
                ok = wait(b_qf, nq++ & 1);
                next_scores(1 - t, xn == 1);
                begun = true;
              }
            }
            ok = ok && wait(b_full + 8 * (KS + nv % VS), (nv / VS) & 1);
            if (!ok) break;
            tc_fence_after();
            product(t, j < 2, j + 2 >= nbm);
            if (!ok) break;
            if (elect_one()) umma_commit(b_empty + 8 * (KS + nv % VS));
            __syncwarp();
            ++nv;
          }
          continue;
        }
        ok = wait(b_qf, nq & 1) && wait(b_full + 8 * (g % NP), (g / NP) & 1);
        if (!ok) break;
        ++nq;
        tc_fence_after();
        if (n0 > 0) scores(0, sl, 0);
        if (n1 > 0) scores(1, sl, 1);
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
              if (ok) scores(t, ks, t);
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
            if (ok && !SEP && j + 1 < nt) scores(t, ks, t);
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
    } else if (BITS == 0 && warp == 10) {
      // ---------------- V rows past the sequence's end ----------------
      int n = 0, nfix = 0;
      uint32_t g = 0;
      for (int i = 0;; ++i) {
        if (JOIN && i == 1) pdl_wait();
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PtThreads<BITS>::SOFT));
    const int t = warp >> 2, q4 = warp & 3, r = 32 * q4 + lane;
    const int rtok = r / p.group, rhead = r - rtok * p.group;
    const uint32_t ts = tmem + 128 * t + ((uint32_t)(32 * q4) << 16), to = tmem + 256 + OC * t + ((uint32_t)(32 * q4) << 16);
    const uint32_t tp = SEP ? tmem + 384 + 64 * t + ((uint32_t)(32 * q4) << 16) : ts;
    int ns = 0, no = 0;  // score blocks and commits of O (per block when SEP, else per item) so far
    uint32_t bs = 0, nhalf = 0;  // blocks so far, items of more blocks than one that the tiles took turns on (cache)
    bool ok = true;
    for (int i = 0; ok; ++i) {
      ok = __all_sync(0xffffffffu, item_wait(i));
      if (!ok) break;
      const volatile PromptItem* it = ring + i % kPtInfo;
      if (it->nbm < 0) break;
      const int nt = it->n[t], qlen = it->qlen, klen = it->klen, key0 = it->key0, nbm = it->nbm;
      const int turn = it->turn;
      const int tok = it->tok + (BITS ? 0 : t) * a.tpt + rtok, head = it->kvh * p.group + rhead;
      const int out_row = it->q0 + tok;
      const int part = it->part;
      __syncwarp();
      if (lane == 0) item_done(i);
      const bool mine = rtok < a.tpt && tok < qlen;
      const int lim = (p.causal ? min(klen, klen - qlen + tok + 1) : klen) - key0;  // keys of this part the row sees
      const bool idle = BITS && !__any_sync(0xffffffffu, mine);
      float m = -INFINITY, top = -INFINITY, l = 0.f;  // top: the score at which m moves
      for (int i = 0; i < nt; ++i) {
        const int j = BITS ? 2 * i + ((t + turn) & 1) : i;
        ok = __all_sync(0xffffffffu, mbar_wait(b_s + 8 * t, (uint32_t)(ns & 1), a.timeout_ns));
        if (!ok) break;
        ++ns;
        tc_fence_after();
        if (BITS && idle) {  // no row of this warp is one of the item's: whatever P holds there stays there
          if (SEP) {
            if (lane == 0) mbar_arrive(b_sf + 8 * t);
            if (i > 0) ok = __all_sync(0xffffffffu, mbar_wait(b_o + 8 * t, (uint32_t)((no - 1) & 1), a.timeout_ns));
            if (!ok) break;
            ++no;
          }
          if (lane == 0) {
            mbar_arrive(b_p + 8 * t);
            mbar_arrive(b_p + 16 + 8 * t);
          }
          continue;
        }
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
        const float4* steps = reinterpret_cast<const float4*>(smem + pt_off_steps<HD, BITS>() + ((bs + j) % kPtSteps) * kPtStepBytes);
        uint32_t there[4];
        bool gaps = false;
        if constexpr (BITS > 0) {
          // the block's steps came before its K; four blocks on there are others
          ok = __all_sync(0xffffffffu, mbar_wait(b_st + 8 * ((bs + j) % kPtSteps), ((bs + j) / kPtSteps) & 1, a.timeout_ns));
          if (!ok) break;
          const volatile uint32_t* tw =
              reinterpret_cast<volatile uint32_t*>(smem + pt_off_there<HD, BITS>() + ((bs + j) % kPtSteps) * 16);
#pragma unroll
          for (int c = 0; c < 4; ++c) there[c] = tw[c];
          gaps = (there[0] & there[1] & there[2] & there[3]) != 0xffffffffu;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 k = steps[8 * c + e / 4];
              unpack64(mul2f(pack64(v[c][e], v[c][e + 1]), pack64(__float_as_uint(k.x), __float_as_uint(k.y))), v[c][e], v[c][e + 1]);
              unpack64(mul2f(pack64(v[c][e + 2], v[c][e + 3]), pack64(__float_as_uint(k.z), __float_as_uint(k.w))), v[c][e + 2],
                       v[c][e + 3]);
            }
        }
        if (gaps || __any_sync(0xffffffffu, left < kPtKeys)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int n = left - 32 * c;
            if (gaps || __any_sync(0xffffffffu, n < 32)) {  // a bit per key: one predicated move a value instead of a comparison too
              uint32_t seen = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
              if (BITS) seen &= there[c];
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
        float mx = fmaxf(max3(x[0], x[1], x[2]), x[3]) * (BITS ? 1.f : p.scale_log2);  // a cache's steps have it in them
        if constexpr (BITS > 0) {
          // steps that fp16 values do not take are the weights': the reference is the largest score with what is left in it,
          // so that the products with them stay in fp16's range
          const uint4 odd = lds16(sb + pt_off_odd<HD, BITS>() + ((bs + j) % kPtSteps) * 16);
          if (odd.x | odd.y | odd.z | odd.w) {
            mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float4 r = steps[32 + 8 * c + e / 4];
                auto with = [](uint32_t s, float y) {  // |y| < 2^(n + 1); a step of 0 takes little off, so that sums of weights fit fp32
                  return __uint_as_float(s) + (float)max(((__float_as_int(y) >> 23) & 0xff) - 127, -60);
                };
                mx = max3(mx, with(v[c][e], r.x), with(v[c][e + 1], r.y));
                mx = max3(mx, with(v[c][e + 2], r.z), with(v[c][e + 3], r.w));
              }
          }
        }
        float f = 1.f;
        if (mx > top) {  // also from -inf, with f = 0: nothing to rescale yet
          const float to = prompt_reference<PT, 7>(mx);
          f = ex2(m - to);
          m = to;
          top = mx + (BITS ? 7.f : 8.f);  // weights up to 2^15, with a factor below 2 from the values' steps 2^14 before it
        }
        const bool rescale = __any_sync(0xffffffffu, f != 1.f) && i > 0;
        if (SEP && i > 0) {  // O += P(j-1) V(j-1) is done: P may be written, O rescaled
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
        float4 vs4;
        // weights of the block, 64 keys at a time: the products with the first half start under the second
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            uint32_t y0, y1;
            const uint64_t x2 = pack64(v[c][e], v[c][e + 1]);
            unpack64(BITS ? add2f(x2, neg2) : fma2f(x2, sc2, neg2), y0, y1);
            float w0 = ex2(__uint_as_float(y0)), w1 = ex2(__uint_as_float(y1));
            sum[c] = add2f(sum[c], pack64(__float_as_uint(w0), __float_as_uint(w1)));
            if (BITS) {
              if (e % 4 == 0) vs4 = steps[32 + 8 * c + e / 4];
              uint32_t u0, u1;
              unpack64(mul2f(pack64(__float_as_uint(w0), __float_as_uint(w1)),
                             e % 4 == 0 ? pack64(__float_as_uint(vs4.x), __float_as_uint(vs4.y))
                                        : pack64(__float_as_uint(vs4.z), __float_as_uint(vs4.w))),
                       u0, u1);
              w0 = __uint_as_float(u0);
              w1 = __uint_as_float(u1);
            }
            v[c >> 1][(c & 1) * 16 + e / 2] = Act<PT>::pack2(w0, w1);
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
      if (BITS) bs += nbm;
      if (nt > 0) {
        if (!SEP) ++no;
        ok = __all_sync(0xffffffffu, mbar_wait(b_o + 8 * t, (uint32_t)((no - 1) & 1), a.timeout_ns));
        if (!ok) break;
      }
      tc_fence_after();
      const bool whole = p.splits == 1 && !p.sums;
      if (BITS && t != (nbm > 0 ? (nbm - 1 + turn) & 1 : 0)) {  // the other one, with the last block, finishes the rows
        if (nt > 0) {  // this one's sums, and O in the same lanes of tensor memory, are for it to take
          volatile float* sums = reinterpret_cast<volatile float*>(smem + pt_off_half<HD, BITS>() + 1024 * (nhalf & 1) + 8 * r);
          sums[0] = m;
          sums[1] = l;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(b_half + 8 * (nhalf & 1));
          ++nhalf;
        }
        continue;
      }
      float own = 1.f, own1 = 0.f;  // what O (and tile 1's) is multiplied by before the division
      bool merge = false;
      if (BITS && nbm > 1) {
        ok = __all_sync(0xffffffffu, mbar_wait(b_half + 8 * (nhalf & 1), (uint32_t)(nhalf / 2 & 1), a.timeout_ns));
        if (!ok) break;
        tc_fence_after();
        const volatile float* other = reinterpret_cast<volatile float*>(smem + pt_off_half<HD, BITS>() + 1024 * (nhalf & 1) + 8 * r);
        const float m1 = other[0], l1 = other[1];
        ++nhalf;
        const float ref = fmaxf(m, m1);
        merge = true;
        own = m == -INFINITY ? 0.f : ex2(m - ref);
        own1 = m1 == -INFINITY ? 0.f : ex2(m1 - ref);
        l = l * own + l1 * own1;
        m = ref;
      }
      float others = 0.f;  // JOIN: what the other sums are multiplied by, and O by own
      bool covered = mine, ours = true, theirs = false;
      const long long more_at = (long long)out_row * p.n_q + head;
      if (JOIN) {
        pdl_wait();
        covered = mine && out_row >= __ldg(a.more.cu_q) && out_row < __ldg(a.more.cu_q + a.more.n_seq);
        const float2 st = covered ? __ldg(reinterpret_cast<const float2*>(a.more.stat) + more_at) : make_float2(-INFINITY, 0.f);
        ours = l != 0.f;  // sums that have seen no key need not have been written
        theirs = st.y != 0.f;
        const float high = fmaxf(m, st.x), ref = high == -INFINITY ? 0.f : high;
        own = ours ? ex2(m - ref) : 0.f;
        others = theirs ? ex2(st.x - ref) : 0.f;
        l = (ours ? l * own : 0.f) + (theirs ? st.y * others : 0.f);
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
      const long long at = ((long long)part * p.tq + out_row) * p.n_q + head;
      if (!whole && mine) *reinterpret_cast<float2*>(p.stat + 2 * at) = make_float2(m, l);
      // the element a lane's row starts at, -1 for a row that is not there
      const long long row_at = covered ? (long long)out_row * p.o_tok + head * p.o_head : -1;
      const uint32_t stg = sb + pt_off_out<HD, BITS>() + warp * pt_stage<BITS>();
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          float4 x4[JOIN ? 8 : 1];
          if (JOIN) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              x4[e % (JOIN ? 8 : 1)] = theirs ? __ldg(reinterpret_cast<const float4*>(a.more.part + more_at * HD) + 16 * c + 8 * h + e)
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
          }
          if (nt > 0) {
            tmem_ld32(to + 64 * c + 32 * h, o);
            if (BITS && merge) {
              uint32_t x[32];
              tmem_ld32(to + (t ? 0u - OC : OC) + 64 * c + 32 * h, x);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * own + __uint_as_float(x[e]) * own1);
            } else {
              tmem_wait_ld();
            }
            if (c == HD / 64 - 1 && h == 1) {  // O has been read: the next item may start over
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(b_of + 8 * t);
                if (BITS && merge) mbar_arrive(b_of + 8 - 8 * t);
              }
            }
          }
          if (JOIN) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float4 x = x4[e / 4 % (JOIN ? 8 : 1)];
              const float add = e % 4 == 0 ? x.x : e % 4 == 1 ? x.y : e % 4 == 2 ? x.z : x.w;
              o[e] = __float_as_uint((ours ? __uint_as_float(o[e]) * own : 0.f) + add * others);
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
              if (BITS) {  // 16 bytes of a lane's own row: the ring of codes has taken the room to gather lines in
                if (mine)
                  *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + row_at + 64 * c + 32 * h + 8 * e) =
                      make_uint4(w[0], w[1], w[2], w[3]);
              } else {
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stg + sw128(lane, 4 * h + e)), "r"(w[0]),
                             "r"(w[1]), "r"(w[2]), "r"(w[3])
                             : "memory");
              }
            }
          } else if (mine && l != 0.f) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<uint4*>(p.part + at * HD + 64 * c + 32 * h + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (BITS == 0 && whole) {
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
  if (JOIN) pdl_wait();  // not to end before the kernel this one follows
  tc_fence_before();
  __syncthreads();  // every MMA has completed (the outputs or the MMA warp waited for them) and every TMEM read is done
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ee
