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
// both are near their limit at hd 128 and the exponentials lead at hd 64.
//
// The running maximum m is a reference, not the exact maximum: it moves only
// when a row's maximum exceeds it by more than 2^8, so O is rarely rescaled
// (the weights stay below 2^8 and the result O / l does not depend on m). S(j)
// of a tile is issued after its O += P(j-1) V(j-1), so the wait for S(j) also
// says that O may be rescaled.
//
// Persistent: one CTA per SM takes items c, 2G - 1 - c, 2G + c, ... of the G
// CTAs (a snake, longest items first), and the next item's loads and first
// scores run under the current one's last products and output. Warps 0-3 and
// 4-7: softmax and output of tile 0 and 1; warp 8: finds the items, publishes
// them in a shared-memory ring and loads Q, K and V by TMA; warp 9: MMA issue;
// warp 10: zeroes V's rows past a sequence's end (their weights are 0, but
// 0 * NaN is not); warp 11 only fills the warpgroup. Waits are bounded; a
// timeout leaves EE_ERR_TIMEOUT in the GEMM status word.
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
constexpr int kPtKeys = 128, kPtInfo = 4;  // keys per block; items published ahead
template <int HD> constexpr int pt_slots() { return HD == 128 ? 5 : 8; }
template <int HD> constexpr uint32_t pt_tile() { return 128u * HD * 2; }
template <int HD> constexpr uint32_t pt_off_bar() { return (2 + pt_slots<HD>()) * pt_tile<HD>(); }
// barriers: full / empty per slot, Q full / empty, S / P / O / O free per tile, V to fix / fixed, item full / empty
template <int HD> constexpr uint32_t pt_off_info() { return pt_off_bar<HD>() + 8 * (2 * pt_slots<HD>() + 12 + 2 * kPtInfo) + 8; }
template <int HD> constexpr uint32_t pt_smem() { return pt_off_info<HD>() + kPtInfo * 64 + 1024; }

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

// Item `idx` (unit-major from the last unit down, key heads and parts inside):
// the whole warp searches, 32 sequences at a time. False past the last item.
EE_DEV bool prompt_item(const PromptTcArgs& a, int idx, int units, PromptItem& it) {
  const PromptArgs& p = a.p;
  const int lane = threadIdx.x & 31, per = p.n_kv * p.splits;
  const int unit = units - 1 - idx / per;
  if (unit < 0) return false;
  it.kvh = idx % per / p.splits;
  it.part = idx % p.splits;
  int before = 0;
  for (int b0 = 0; b0 < p.n_seq; b0 += 32) {
    const int b = b0 + lane;
    PromptSeq s{};
    int nu = 0;
    if (b < p.n_seq) {
      s = prompt_seq(p, b);
      nu = (s.qlen + 2 * a.tpt - 1) / (2 * a.tpt);
    }
    int inc = nu;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    inc += before;
    const unsigned hit = __ballot_sync(0xffffffffu, unit >= inc - nu && unit < inc);
    if (hit) {
      const int src = __ffs(hit) - 1;
      it.q0 = __shfl_sync(0xffffffffu, s.q0, src);
      it.qlen = __shfl_sync(0xffffffffu, s.qlen, src);
      it.k0 = __shfl_sync(0xffffffffu, s.k0, src);
      it.klen = __shfl_sync(0xffffffffu, s.klen, src);
      it.tok = (unit - __shfl_sync(0xffffffffu, inc - nu, src)) * 2 * a.tpt;
      break;
    }
    before = __shfl_sync(0xffffffffu, inc, 31);
  }
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

template <typename T, int HD>
__global__ void __launch_bounds__(kPtThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ PromptTcArgs a) {
  constexpr int NS = pt_slots<HD>();
  constexpr uint32_t TILE = pt_tile<HD>(), PANEL = 128 * 128;  // a panel: 64 columns of 128 rows
  constexpr int PANELS = HD / 64;
  extern __shared__ __align__(1024) char smem_raw[];
  const uint32_t base0 = smem_u32(smem_raw);
  const uint32_t sb = (base0 + 1023u) & ~1023u;
  char* smem = smem_raw + (sb - base0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sQ = sb, sKV = sb + 2 * TILE;
  const uint32_t b_full = sb + pt_off_bar<HD>(), b_empty = b_full + 8 * NS;
  const uint32_t b_qf = b_empty + 8 * NS, b_qe = b_qf + 8, b_s = b_qe + 8, b_p = b_s + 16, b_o = b_p + 16;
  const uint32_t b_of = b_o + 16, b_req = b_of + 16, b_fix = b_req + 8, b_if = b_fix + 8, b_ie = b_if + 8 * kPtInfo;
  const uint32_t off_tm = b_ie + 8 * kPtInfo - sb;
  volatile PromptItem* ring = reinterpret_cast<volatile PromptItem*>(smem + pt_off_info<HD>());
  const PromptArgs& p = a.p;
  if (warp == 8 && lane == 0) {
    tma_prefetch_map(&mq);
    tma_prefetch_map(&mk);
    tma_prefetch_map(&mv);
    for (int s = 0; s < NS; ++s) {
      mbar_init(b_full + 8 * s, 1);
      mbar_init(b_empty + 8 * s, 1);
    }
    mbar_init(b_req, 1);
    mbar_init(b_fix, 1);
    mbar_init(b_qf, 1);
    mbar_init(b_qe, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(b_s + 8 * t, 1);
      mbar_init(b_p + 8 * t, 4);
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
  // TMEM columns: S (P over its first half) of tile t at 128 t, O at 256 + 128 t
  // The consumers' view of the item ring: wait for item i, read it; release when done with it.
  auto item_wait = [&](int i) { return mbar_wait(b_if + 8 * (i % kPtInfo), (uint32_t)((i / kPtInfo) & 1), a.timeout_ns); };
  auto item_done = [&](int i) { mbar_arrive(b_ie + 8 * (i % kPtInfo)); };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsRest));
    if (warp == 8) {
      // ---------------- items and loads ----------------
      bool ok = true;
      int units = 0, n = 0, nq = 0;  // K / V tiles and Q loads issued so far
      for (int b = lane; b < p.n_seq; b += 32) units += (prompt_seq(p, b).qlen + 2 * a.tpt - 1) / (2 * a.tpt);
      units = __reduce_add_sync(0xffffffffu, units);
      const uint32_t qbytes = (uint32_t)(p.group * a.tpt) * 128u * PANELS;
      for (int i = 0;; ++i) {
        const long long idx = (long long)i * gridDim.x + ((i & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        PromptItem it{};
        const bool more = ok && idx < (long long)units * p.n_kv * p.splits && prompt_item(a, (int)idx, units, it);
        if (lane == 0) {
          if (i >= kPtInfo && ok && !mbar_wait(b_ie + 8 * (i % kPtInfo), (uint32_t)((i / kPtInfo - 1) & 1), a.timeout_ns))
            ok = false;
          volatile PromptItem* r = ring + i % kPtInfo;
          r->q0 = it.q0; r->qlen = it.qlen; r->klen = it.klen;
          r->tok = it.tok; r->kvh = it.kvh; r->part = it.part; r->key0 = it.key0;
          r->n[0] = it.n[0]; r->n[1] = it.n[1]; r->tail = it.tail;
          r->nbm = more && ok ? it.nbm : -1;
          mbar_arrive(b_if + 8 * (i % kPtInfo));
          auto load_kv = [&](int w) {  // tile w of the item: K(0) V(0) K(1) V(1) ...
            const int sl = n % NS;
            if (n >= NS && !mbar_wait(b_empty + 8 * sl, (uint32_t)((n / NS - 1) & 1), a.timeout_ns)) {
              ok = false;
              return;
            }
            mbar_arrive_expect_tx(b_full + 8 * sl, TILE);
            for (int c = 0; c < PANELS; ++c)
              tma_load_3d(sKV + sl * TILE + c * PANEL, (w & 1) ? &mv : &mk, 64 * c, it.kvh,
                          it.k0 + it.key0 + (w >> 1) * kPtKeys, b_full + 8 * sl);
            ++n;
          };
          if (more && ok && it.nbm > 0) {
            load_kv(0);
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
            for (int w = 1; w < 2 * it.nbm && ok; ++w) load_kv(w);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!more || !ok) break;
      }
      // everything issued lands before the CTA may exit
      if (lane == 0) {
        for (int g = max(n - NS, 0); g < n; ++g)
          if (!mbar_wait(b_full + 8 * (g % NS), (uint32_t)((g / NS) & 1), a.timeout_ns)) ok = false;
        if (nq > 0 && !mbar_wait(b_qf, (uint32_t)((nq - 1) & 1), a.timeout_ns)) ok = false;
        if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ---------------- MMA issue ----------------
      if (lane == 0) {
        constexpr uint32_t id_s = umma_idesc<T>(128, 128), id_o = umma_idesc<T>(128, HD) | kIdescBMajorMN;
        bool ok = true;
        int n = 0, nq = 0, nfix = 0;   // K / V tiles, Q loads and fixed tails consumed so far
        int np[2] = {0, 0}, no[2] = {0, 0};  // P blocks and outputs of each tile so far
        auto wait_slot = [&](int g) { return mbar_wait(b_full + 8 * (g % NS), (uint32_t)((g / NS) & 1), a.timeout_ns); };
        auto scores = [&](int t, int g) {  // S_t = Q_t K^T, K in ring tile g
          const uint64_t qd = umma_desc_sw128(sQ + t * TILE), kd = umma_desc_sw128(sKV + (uint32_t)(g % NS) * TILE);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t o = (uint64_t)(((kk >> 2) * PANEL + (kk & 3) * 32) >> 4);
            umma_f16(tmem + 128 * t, qd + o, kd + o, id_s, kk ? 1u : 0u);
          }
          umma_commit(b_s + 8 * t);
        };
        for (int i = 0; ok; ++i) {
          if (!item_wait(i)) {
            ok = false;
            break;
          }
          const volatile PromptItem* r = ring + i % kPtInfo;
          const int nbm = r->nbm, n0 = r->n[0], n1 = r->n[1], tail = r->tail;
          item_done(i);
          if (nbm < 0) break;
          if (nbm == 0) continue;
          ok = mbar_wait(b_qf, (uint32_t)(nq & 1), a.timeout_ns) && wait_slot(n);
          if (!ok) break;
          ++nq;
          tc_fence_after();
          if (n0 > 0) scores(0, n);
          if (n1 > 0) scores(1, n);
          umma_commit(b_empty + 8 * (n % NS));
          if (nbm == 1) umma_commit(b_qe);
          for (int j = 0; j < nbm && ok; ++j) {
            const int vg = n + 2 * j + 1, vs = vg % NS;
            ok = wait_slot(vg);
            if (ok && j + 1 < nbm) ok = wait_slot(vg + 1);
            const bool fix = j + 1 == nbm && tail < kPtKeys;
            if (ok && fix) mbar_arrive(b_req);
            int fixed = fix ? 0 : 1;
            const uint64_t vd = umma_desc_mn128(sKV + (uint32_t)vs * TILE, PANEL);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int nt = t ? n1 : n0;
              if (!ok || j >= nt) continue;
              // O of the tile's previous item has been read
              if (j == 0 && no[t] > 0) ok = mbar_wait(b_of + 8 * t, (uint32_t)((no[t] - 1) & 1), a.timeout_ns);
              ok = ok && mbar_wait(b_p + 8 * t, (uint32_t)(np[t] & 1), a.timeout_ns);
              if (ok && !fixed) {
                ok = mbar_wait(b_fix, (uint32_t)(nfix & 1), a.timeout_ns);
                ++nfix;
                fixed = 1;
              }
              if (!ok) continue;
              ++np[t];
              tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < kPtKeys / 16; ++kk)  // O_t += P_t V(j), 16 keys at a time
                umma_f16_ts(tmem + 256 + 128 * t, tmem + 128 * t + 8 * kk, vd + (uint64_t)((kk * 2048) >> 4), id_o,
                            (j | kk) ? 1u : 0u);
              if (j + 1 < nt) {
                scores(t, vg + 1);
              } else {
                umma_commit(b_o + 8 * t);
                ++no[t];
              }
            }
            if (ok) {
              umma_commit(b_empty + 8 * vs);
              if (j + 1 < nbm) umma_commit(b_empty + 8 * ((vg + 1) % NS));
              if (j + 2 == nbm) umma_commit(b_qe);
            }
          }
          n += 2 * nbm;
        }
        if (!ok) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
      }
      __syncwarp();
    } else if (warp == 10) {
      // ---------------- V rows past the sequence's end ----------------
      int n = 0, nfix = 0;
      for (int i = 0;; ++i) {
        bool ok = item_wait(i);
        const volatile PromptItem* r = ring + i % kPtInfo;
        const int nbm = r->nbm, tail = r->tail;
        __syncwarp();
        if (lane == 0) item_done(i);
        if (!__all_sync(0xffffffffu, ok) || nbm < 0) break;
        n += 2 * nbm;
        if (nbm == 0 || tail == kPtKeys) continue;
        // not before the MMA warp has come to the block: earlier, the slot's parity may be an older load's
        const int g = n - 1;
        ok = mbar_wait(b_req, (uint32_t)(nfix++ & 1), a.timeout_ns) &&
             mbar_wait(b_full + 8 * (g % NS), (uint32_t)((g / NS) & 1), a.timeout_ns);
        if (!__all_sync(0xffffffffu, ok)) break;
        const uint32_t v = sKV + (uint32_t)(g % NS) * TILE;
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
    const uint32_t ts = tmem + 128 * t + ((uint32_t)(32 * q4) << 16), to = tmem + 256 + 128 * t + ((uint32_t)(32 * q4) << 16);
    int ns = 0, no = 0;  // score blocks and outputs so far
    bool ok = true;
    for (int i = 0; ok; ++i) {
      ok = __all_sync(0xffffffffu, item_wait(i));
      if (!ok) break;
      const volatile PromptItem* it = ring + i % kPtInfo;
      if (it->nbm < 0) break;
      const int nt = it->n[t], qlen = it->qlen, klen = it->klen, key0 = it->key0;
      const int tok = it->tok + t * a.tpt + rtok, head = it->kvh * p.group + rhead;
      const long long out_row = (long long)it->q0 + tok;
      const int part = it->part;
      __syncwarp();
      if (lane == 0) item_done(i);
      const bool mine = rtok < a.tpt && tok < qlen;
      const int lim = (p.causal ? min(klen, klen - qlen + tok + 1) : klen) - key0;  // keys of this part the row sees
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nt; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(b_s + 8 * t, (uint32_t)(ns & 1), a.timeout_ns));
        if (!ok) break;
        ++ns;
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
      if (!ok) break;
      if (nt > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(b_o + 8 * t, (uint32_t)(no & 1), a.timeout_ns));
        if (!ok) break;
        ++no;
      }
      tc_fence_after();
      const bool whole = p.splits == 1;
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
      T* out = reinterpret_cast<T*>(p.out) + out_row * p.o_tok + head * p.o_head;
      const long long at = ((long long)part * p.tq + out_row) * p.n_q + head;
      if (!whole && mine) *reinterpret_cast<float2*>(p.stat + 2 * at) = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        if (nt > 0) {
          tmem_ld32(to + 32 * c, o);
          tmem_wait_ld();
          if (c == HD / 32 - 1) {  // O has been read: the next item may start over
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_of + 8 * t);
          }
        }
        if (mine && whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = l == 0.f ? 0u
                              : Act<T>::pack2(__uint_as_float(o[e + 2 * k]) * inv, __uint_as_float(o[e + 2 * k + 1]) * inv);
            *reinterpret_cast<uint4*>(out + 32 * c + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (mine && l != 0.f) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(p.part + at * HD + 32 * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
    }
    if (!ok && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();  // every MMA has completed (the outputs waited for them) and every TMEM read is done
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace ee
