// ee_cache_attn.cuh -- attention of query rows over a paged cache of 8- or
// 4-bit keys and values.
//
// Few rows (up to 16 a sequence and key head; more: ee_prompt_tc.cuh). A row is
// (token, head of the key head's group); an item is 8 NT rows of one sequence
// and key head against the sequence's keys, cut into steps of 32. All items'
// steps form one list of which every warp takes an equal share (see
// ee_prompt_list.cuh); its steps' codes come by TMA into a ring in shared
// memory, one box of 32 rows each of keys and values, and 32 steps (fp32) of
// either by a bulk copy, on the stage's barrier.
//
// Both products are taken transposed, so that 8 rows are enough to fill an MMA:
//   S^T = K Q^T    A = codes of 16 keys x 16 dims, B = the rows' queries
//   O^T += V^T P   A = codes of 16 dims x 16 keys, B = the rows' weights
// The codes become 16-bit operands in registers, exactly (integers below 2^8):
// a 16-bit lane of an operand register takes its bits straight from a code's
// byte or half byte, OR-ed under the exponent of a power of two that one packed
// instruction takes off again (bytes in bf16: as its numbers below 2^-126, times
// 2^127, which leaves a 64th of them). ldmatrix moves pairs (4 bits: fours) of codes as
// its 16-bit elements; which dim or key a code then belongs to is a matter of
// naming, the same in both operands of a product, so nothing is shuffled: the
// words of K hold four (eight) dims of a key, of which bytes 0 and 2 make one
// pair and 1 and 3 the other; the words of V, transposed on the way, two (four)
// dims of two keys, whose low bytes are one row of V^T and the high ones the
// next. A key's step multiplies its scores; a value's step multiplies the
// weights, after their sum is taken.
//
// Queries go into the product as fp16, bf16 ones scaled by a power of two so
// that the row's largest lies in [1, 2): a value more than 2^14 below it loses
// up to 2^-25 of the largest, less than fp32 loses in the sum. The weights times
// the values' steps have fp32's range, so they are rounded to bf16, and a second
// product adds what that left (to 2^-16): without it a row of few keys is off by
// the same half step in all its dims, 1.6 times the result's own rounding (64 x 1
// token: 23.6 us, with it 24.4).
//
// HBM-bound where the call is large (64 x 1 token behind 4096, 8 key heads of 128,
// 8 bits: 5.5 TB/s; 4 bits, where the instructions on a code count: 3.9). In
// between, latency: 850 instructions a step and the second product by two warps a
// scheduler, whose issue slots are 23 % busy over the launch (64 x 1 behind 1 to
// 1632, 16 / 4 heads of 128, 8 bits: 24.5 us where the bytes take 9.6; twelve
// warps with rings two stages deep: 30.4 where eight took 28.7). A small call is
// two launches, the sums and the join of rows that a border cut, and in each the
// way through offsets, lengths and table to the codes: 9 us.
#pragma once

#include <atomic>
#include <type_traits>

#include "ee_cache.cuh"
#include "ee_host.h"
#include "ee_prompt_list.cuh"
#include "ee_prompt_tc.cuh"
#include "ee_tma.cuh"

namespace ee {

// ee_prompt.cu
bool prompt_head_map(CUtensorMap* map, const void* base, int hd, int heads, long long tokens, long long head, long long tok,
                     int bh, int bt);

struct CacheAttnArgs {
  CacheView c;
  const float *k_steps, *v_steps;
  const void* q;
  void* out;
  const int* cu_q;
  long long q_tok, q_head, o_tok, o_head;  // strides, elements
  int tq, n_q, group, causal;
  int rows, rows_log2;  // rows of an item
  float scale_log2;     // scale * log2(e)
  // sums of parts, [hd] each, and their maximum and weight: first of items that a border cuts, by worker ([workers][2]
  // [rows]); behind a prefix then of every whole item's rows ([tq][n_q]) and of the prefix ([pre_splits][tq][n_q])
  float *part, *stat;
  long long whole;      // the first of the whole items' rows
  int pre_splits;       // 0: no prefix
  int pre_ctas;         // of the kernel that sums it up
  int* status;
  unsigned long long timeout_ns;
};

struct CacheSeq {
  int q0, qlen, klen;
};
EE_DEV CacheSeq list_seq(const CacheAttnArgs& a, int b) {
  CacheSeq s;
  s.q0 = min(max(__ldg(a.cu_q + b), 0), a.tq);
  s.qlen = min(max(__ldg(a.cu_q + b + 1), s.q0), a.tq) - s.q0;
  s.klen = min(max(__ldg(a.c.k_lens + b), 0), a.c.width << a.c.shift);
  return s;
}
constexpr int kCaKeys = 32, kCaMinSteps = 6;  // keys of a step; steps that are worth a worker (2 x 1
                                               // token behind 30000, 4 bits: 21.4 us with 3, 19.8 with 6, 20.6 with 10)
EE_DEV long long list_steps(const CacheAttnArgs& a, const CacheSeq& s, int& per_item) {
  per_item = (s.klen + kCaKeys - 1) / kCaKeys;
  return (((long long)s.qlen * a.group + a.rows - 1) >> a.rows_log2) * a.c.n_kv * per_item;
}

// How the kernel is cut: workers (warps) per CTA and stages of their rings.
template <int HD, int BITS, int NT>
struct CaShape {
  static constexpr int RB = HD * BITS / 8;           // bytes of a row of codes
  static constexpr int TILE = kCaKeys * RB;
  static constexpr int STAGE = 2 * TILE + 2 * kCaKeys * 4;
  static constexpr int WORKERS = NT == 1 && STAGE < 8192 ? 16 : 8;
  static constexpr int FIT = 212 * 1024 / (WORKERS * STAGE);
  static constexpr int NS = FIT < 6 ? FIT : 6;
  static constexpr int THREADS = 32 * WORKERS;
  static constexpr int SMEM = WORKERS * NS * STAGE + 1024;
  static constexpr int ROWS = 8 * NT;
};

EE_DEV void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
EE_DEV float ca_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
EE_DEV uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Bytes 0 and 2 of a word (signed codes) as two fp16: the byte with its sign
// bit flipped under the exponent of 1024, less 1024 + 128.
EE_DEV uint32_t byte_pair_f16(uint32_t w) { return fma2<__half>(and_xor(w, 0x00FF00FFu, 0x64806480u), 0x3C003C00u, 0xE480E480u); }
// Half bytes 0 and 4 (LOW) or 1 and 5 of a word as two fp16: likewise, the upper
// ones 16 times as large before the multiplication.
template <bool LOW>
EE_DEV uint32_t half_pair_f16(uint32_t w) {
  return LOW ? fma2<__half>(and_xor(w, 0x000F000Fu, 0x64086408u), 0x3C003C00u, 0xE408E408u)   // less 1024 + 8
             : fma2<__half>(and_xor(w, 0x00F000F0u, 0x64806480u), 0x2C002C00u, 0xD480D480u);  // / 16, less 64 + 8
}
// Bytes 0 and 2 as two bf16, a 64th of them: the byte with its sign bit flipped
// is that many times 2^-133 (subnormal below 128, and linear on to 255); times
// 2^127, less 128 / 64.
EE_DEV uint32_t byte_pair_bf16(uint32_t w) {
  return fma2<__nv_bfloat16>(and_xor(w, 0x00FF00FFu, 0x00800080u), 0x7F007F00u, 0xC000C000u);
}
EE_DEV uint32_t half_pair_bf16(uint32_t w) {  // half bytes 0 and 4, less 128 + 8
  return fma2<__nv_bfloat16>(and_xor(w, 0x000F000Fu, 0x43084308u), 0x3F803F80u, 0xC308C308u);
}

// A place in the list: a step of an item of a sequence.
struct CaAt {
  int b, step, per_item;
  int r0, kvh;  // the item: its first row, its key head
  CacheSeq s;
  EE_DEV void enter(const CacheAttnArgs& a, int seq) {  // sequence `seq` or the next one that has steps
    for (b = seq; b < a.c.n_seq; ++b) {
      s = list_seq(a, b);
      if (list_steps(a, s, per_item) > 0) break;
    }
    r0 = kvh = step = 0;
  }
  EE_DEV bool next(const CacheAttnArgs& a) {  // true: another item
    if (++step < per_item) return false;
    step = 0;
    if (++kvh == a.c.n_kv) {
      kvh = 0;
      r0 += a.rows;
      if (r0 >= s.qlen * a.group) enter(a, b + 1);
    }
    return true;
  }
};

template <typename T, int HD, int BITS, int NT>
__global__ void __launch_bounds__(CaShape<HD, BITS, NT>::THREADS, 1)
    cache_rows_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                      const __grid_constant__ CacheAttnArgs a) {
  using S = CaShape<HD, BITS, NT>;
  constexpr int NTH = S::THREADS, NWK = S::WORKERS, NS = S::NS, RB = S::RB, TILE = S::TILE, R = S::ROWS;
  constexpr int CH = HD / 16;  // 16-dim pieces of a head: MMAs of K Q^T, tiles of O^T
  constexpr bool HALF = std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) char smem_raw[];
  __shared__ PrList<NTH> sh;
  __shared__ __align__(8) uint64_t bars[NWK][NS];
  __shared__ int none[NWK][NS];  // the stage's page does not exist: its keys do not either
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3, mi = lane >> 3;
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring = smem0 + warp * NS * 2 * TILE;
  const uint32_t steps0 = smem0 + NWK * NS * 2 * TILE + warp * NS * 2 * kCaKeys * 4;
  const uint32_t full = smem_u32(&bars[warp][0]);
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(full + 8 * i, 1);
    mbar_fence_init();
  }
  // What a CTA's way to its first load reads, one after another (offsets and lengths, table), is brought to L2 under the
  // kernel before this one.
  {
    const long long i = 32ll * ((long long)blockIdx.x * NTH + tid);
    if (i <= a.c.n_seq) prefetch_l2(a.cu_q + i);
    if (i < a.c.n_seq) prefetch_l2(a.c.k_lens + i);
    if (a.c.width > 0 && i < (a.c.n_seq - 1) * a.c.table_row + a.c.width) prefetch_l2(a.c.table + i);
  }
  // Behind a prefix the kernel before this one sums that up, from nothing that this one writes and for nothing that it
  // reads; it has itself waited for everything before the call, so this one need not wait for it but before it ends (the
  // join follows on this one).
  if (a.pre_splits) pdl_release();
  else pdl_entry();
  const int per = (a.c.n_seq + NTH - 1) / NTH;
  const long long total = pr_list<NTH>(a, &sh, per, a.c.n_seq, [](int, const CacheSeq&, long long) {});
  const long long share = pr_share(total, (int)gridDim.x * NWK, kCaMinSteps);
  const long long me = (long long)warp * gridDim.x + blockIdx.x;  // neighbours in the list on different SMs
  const long long first = me * share;
  if (first >= total) {
    pdl_wait();
    return;
  }
  int left = (int)(total - first < share ? total - first : share);  // steps to go
  CaAt at{};
  {
    int lo = 0;  // the last thread whose sequences begin at or before the share
#pragma unroll
    for (int o = NTH / 2; o > 0; o >>= 1)
      if (sh.before[lo + o] <= first) lo += o;
    long long x = first - sh.before[lo];
    at.enter(a, lo * per);
    while (at.b < a.c.n_seq) {
      int n;
      const long long steps = list_steps(a, at.s, n);
      if (x < steps) break;
      x -= steps;
      at.enter(a, at.b + 1);
    }
    if (at.b >= a.c.n_seq) {  // the lengths have changed meanwhile
      pdl_wait();
      return;
    }
    const int item = (int)pr_div(x, at.per_item);
    at.step = (int)(x - (long long)item * at.per_item);
    at.r0 = item / a.c.n_kv * R;
    at.kvh = item % a.c.n_kv;
  }
  // ---- loads: the place they have come to, its page ----
  CaAt ld = at;
  const int page_shift = a.c.shift - 5, page_mask = (1 << page_shift) - 1;  // steps per page
  auto page_of = [&](const CaAt& p) { return __ldg(a.c.table + p.b * a.c.table_row + (p.step >> page_shift)); };
  int page = page_of(ld);
  int issued = 0;
  auto load = [&](int buf) {  // step `ld` into stage buf, then on to the next step
    if (lane == 0) {
      const bool ok = (unsigned)page < (unsigned)a.c.pages;
      const int row = (((ok ? page : 0) * a.c.n_kv + ld.kvh) << a.c.shift) + (ld.step & page_mask) * kCaKeys;
      const uint32_t bar = full + 8 * buf, d = ring + buf * 2 * TILE, e = steps0 + buf * 2 * kCaKeys * 4;
      none[warp][buf] = !ok;
      mbar_arrive_expect_tx(bar, S::STAGE);
      tma_load_2d(d, &mk, 0, row, bar);
      tma_load_2d(d + TILE, &mv, 0, row, bar);
      bulk_load(e, a.k_steps + row, kCaKeys * 4, bar);
      bulk_load(e + kCaKeys * 4, a.v_steps + row, kCaKeys * 4, bar);
    }
    ++issued;
    const bool other = ld.next(a);
    if (ld.b < a.c.n_seq && (other || (ld.step & page_mask) == 0)) page = page_of(ld);
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i)
    if (i < left && ld.b < a.c.n_seq) load(i);
  // ldmatrix addresses of this lane within a tile: row of 16, 16-byte pieces as TMA's swizzle of this row length places
  // them
  uint32_t la[RB / 32];
  {
    const int row = (mi & 1) * 8 + (lane & 7), x = RB == 128 ? row & 7 : RB == 64 ? (row >> 1) & 3 : (row >> 2) & 1;
#pragma unroll
    for (int c = 0; c < RB / 32; ++c) la[c] = row * RB + (((2 * c + (mi >> 1)) ^ x) << 4);
  }
  uint32_t qf[NT][CH][2];
  float o[CH][NT][4];
  float m[NT][2], l[NT][2], crow[NT][2];
  int lim[NT][2];
  int rows = 0, lim_min = 0;
  bool fresh = true, head = true, ok = true;  // the item's first step of this share; no item of it finished yet
  int from = 0, buf = 0, done = 0;
  uint32_t phase = 0;
  auto row_at = [&](int r, int& tok, int& h) {  // token and head of row r, the last row's for those past it
    const int x = min(r, rows - 1);
    tok = x / a.group;
    h = at.kvh * a.group + x - tok * a.group;
  };
  for (; left > 0 && issued > done; --left) {
    if (fresh) {
      fresh = false;
      from = at.step;
      rows = at.s.qlen * a.group;
      int tok, h;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        row_at(at.r0 + 8 * j + g, tok, h);
        const T* src = reinterpret_cast<const T*>(a.q) + (long long)(at.s.q0 + tok) * a.q_tok + h * a.q_head;
        uint32_t w[CH][2];  // this lane's dims in the order of the codes
        if (BITS == 8) {
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const uint2 x = *reinterpret_cast<const uint2*>(src + 16 * c + 4 * t);
            w[c][0] = prmt(x.x, x.y, 0x5410u);
            w[c][1] = prmt(x.x, x.y, 0x7632u);
          }
        } else {
#pragma unroll
          for (int c = 0; c < CH / 2; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + 32 * c + 8 * t);
            w[2 * c][0] = prmt(x.x, x.z, 0x5410u);
            w[2 * c][1] = prmt(x.x, x.z, 0x7632u);
            w[2 * c + 1][0] = prmt(x.y, x.w, 0x5410u);
            w[2 * c + 1][1] = prmt(x.y, x.w, 0x7632u);
          }
        }
        float back = a.scale_log2;
        if (HALF) {
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            qf[j][c][0] = w[c][0];
            qf[j][c][1] = w[c][1];
          }
        } else {
          uint32_t mx = 0;
#pragma unroll
          for (int c = 0; c < CH; ++c) mx = __vmaxu2(mx, __vmaxu2(w[c][0] & 0x7FFF7FFFu, w[c][1] & 0x7FFF7FFFu));
          mx = max(mx & 0xFFFFu, mx >> 16);
          mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const int e = min(max((int)(mx >> 7), 1), 253);  // the largest value's exponent
          const float by = __int_as_float((254 - e) << 23);
          back *= __int_as_float(e << 23);
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 f = Act<T>::unpack2(w[c][i]);
              qf[j][c][i] = Act<__half>::pack2(f.x * by, f.y * by);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          crow[j][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
          row_at(at.r0 + 8 * j + 2 * t + e, tok, h);
          lim[j][e] = a.causal ? min(at.s.klen, at.s.klen - at.s.qlen + tok + 1) : at.s.klen;
          m[j][e] = -INFINITY;
          l[j][e] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][j][e] = 0.f;
      }
      row_at(at.r0, tok, h);
      lim_min = a.causal ? min(at.s.klen, at.s.klen - at.s.qlen + tok + 1) : at.s.klen;  // no row sees less than the first
    }
    // the step before this one has been read: its stage takes the next load
    if (left > NS - 1 && ld.b < a.c.n_seq) load(buf == 0 ? NS - 1 : buf - 1);
    ok = __all_sync(0xffffffffu, mbar_wait(full + 8 * buf, phase, a.timeout_ns));
    if (!ok) break;
    const uint32_t kt = ring + buf * 2 * TILE, vt = kt + TILE, st = steps0 + buf * 2 * kCaKeys * 4;
    const int key = at.step * kCaKeys;
    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][j][e] = 0.f;
#pragma unroll
      for (int c2 = 0; c2 < RB / 32; ++c2) {
        uint32_t r[4];
        pr_ldsm(kt + la[c2] + 16 * mt * RB, r);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint32_t x = r[2 * p], y = r[2 * p + 1];  // keys g and g + 8
          if (BITS == 8) {
            const int c = 2 * c2 + p;
            const uint32_t a0 = byte_pair_f16(x), a1 = byte_pair_f16(y), a2 = byte_pair_f16(x >> 8), a3 = byte_pair_f16(y >> 8);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma16816<__half>(s[mt][j], a0, a1, a2, a3, qf[j][c][0], qf[j][c][1]);
          } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int c = 2 * (2 * c2 + p) + q;
              const uint32_t xx = x >> (8 * q), yy = y >> (8 * q);
              const uint32_t a0 = half_pair_f16<true>(xx), a1 = half_pair_f16<true>(yy);
              const uint32_t a2 = half_pair_f16<false>(xx), a3 = half_pair_f16<false>(yy);
#pragma unroll
              for (int j = 0; j < NT; ++j) mma16816<__half>(s[mt][j], a0, a1, a2, a3, qf[j][c][0], qf[j][c][1]);
            }
          }
        }
      }
    }
    constexpr float UNIT = BITS == 8 ? 64.f : 1.f;  // what the bf16 codes leave out
    float ks[4], vs[4];                             // keys g, g + 8, g + 16, g + 24
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks[i]) : "r"(st + (g + 8 * i) * 4));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs[i]) : "r"(st + (kCaKeys + g + 8 * i) * 4));
      vs[i] *= UNIT;
    }
    const bool gone = *reinterpret_cast<volatile int*>(&none[warp][buf]) != 0;
    const bool masked = gone || key + kCaKeys > lim_min;
    float x0[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][j][e] = s[mt][j][e] * ks[2 * mt + (e >> 1)] * crow[j][e & 1];
      if (masked) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (gone || key + 16 * mt + 8 * (e >> 1) + g >= lim[j][e & 1]) s[mt][j][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) x0[j][e] = fmaxf(fmaxf(s[0][j][e], s[0][j][2 + e]), fmaxf(s[1][j][e], s[1][j][2 + e]));
    }
#pragma unroll
    for (int d = 4; d < 32; d <<= 1)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) x0[j][e] = fmaxf(x0[j][e], __shfl_xor_sync(0xffffffffu, x0[j][e], d));
    // m is a reference, not the exact maximum: it moves when a score is 8 above it (a weight of 2^8), so that O is
    // rarely rescaled
    bool moved = false;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) moved |= x0[j][e] > m[j][e] + 8.f;
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float n = fmaxf(m[j][e], x0[j][e]);
          const float f = n == -INFINITY ? 1.f : ca_ex2(m[j][e] - n);
          m[j][e] = n;
          l[j][e] *= f;
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            o[c][j][e] *= f;
            o[c][j][2 + e] *= f;
          }
        }
    }
    uint32_t pb[2][NT][2], pl[2][NT][2];  // weights of 16 keys as the product takes them, and what their rounding left
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float u0 = m[j][0] == -INFINITY ? 0.f : m[j][0], u1 = m[j][1] == -INFINITY ? 0.f : m[j][1];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = ca_ex2(s[mt][j][2 * i] - u0), p1 = ca_ex2(s[mt][j][2 * i + 1] - u1);
          l[j][0] += p0;
          l[j][1] += p1;
          float w0 = p0 * vs[2 * mt + i], w1 = p1 * vs[2 * mt + i];
          if (masked) {  // whatever the value's step is there
            if (s[mt][j][2 * i] == -INFINITY) w0 = 0.f;
            if (s[mt][j][2 * i + 1] == -INFINITY) w1 = 0.f;
          }
          const uint32_t hi = Act<__nv_bfloat16>::pack2(w0, w1);
          pb[mt][j][i] = movmatrix(hi);
          const float2 f = Act<__nv_bfloat16>::unpack2(hi);
          pl[mt][j][i] = movmatrix(Act<__nv_bfloat16>::pack2(w0 - f.x, w1 - f.y));
        }
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int c2 = 0; c2 < RB / 32; ++c2) {
        uint32_t r[4];
        pr_ldsm_t(vt + la[c2] + 16 * mt * RB, r);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint32_t x = r[2 * p], y = r[2 * p + 1];  // keys 2t, 2t + 1 and those 8 on
#pragma unroll
          for (int q = 0; q < (BITS == 8 ? 1 : 2); ++q) {
            uint32_t a0, a1, a2, a3;
            if (BITS == 8) {
              a0 = byte_pair_bf16(x), a1 = byte_pair_bf16(x >> 8), a2 = byte_pair_bf16(y), a3 = byte_pair_bf16(y >> 8);
            } else {
              a0 = half_pair_bf16(x >> (8 * q)), a1 = half_pair_bf16(x >> (8 * q + 4));
              a2 = half_pair_bf16(y >> (8 * q)), a3 = half_pair_bf16(y >> (8 * q + 4));
            }
            const int c = BITS == 8 ? 2 * c2 + p : 2 * (2 * c2 + p) + q;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma16816<__nv_bfloat16>(o[c][j], a0, a1, a2, a3, pb[mt][j][0], pb[mt][j][1]);
              mma16816<__nv_bfloat16>(o[c][j], a0, a1, a2, a3, pl[mt][j][0], pl[mt][j][1]);
            }
          }
        }
      }
    __syncwarp();  // every lane has read the stage before it is loaded again
    ++done;
    if (++buf == NS) {
      buf = 0;
      phase ^= 1;
    }
    const bool end = at.step + 1 == at.per_item;
    if (end || left == 1) {
      const bool whole = end && from == 0;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = l[j][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const int rr = 8 * j + 2 * t + e, r = at.r0 + rr;
          if (r >= rows) continue;
          int tok, h;
          row_at(r, tok, h);
          if (whole && !a.pre_splits) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees no key is zero
            T* out = reinterpret_cast<T*>(a.out) + (long long)(at.s.q0 + tok) * a.o_tok + h * a.o_head;
#pragma unroll
            for (int c = 0; c < CH; c += BITS == 8 ? 1 : 2) {
              const uint32_t w = Act<T>::pack2(o[c][j][e] * inv, o[c][j][2 + e] * inv);
              if (BITS == 8) *reinterpret_cast<uint32_t*>(out + 16 * c + 2 * g) = w;
              else
                *reinterpret_cast<uint2*>(out + 16 * c + 4 * g) =
                    make_uint2(w, Act<T>::pack2(o[c + 1][j][e] * inv, o[c + 1][j][2 + e] * inv));
            }
          } else {
            const long long slot = whole ? a.whole + (long long)(at.s.q0 + tok) * a.n_q + h
                                         : (me * 2 + (head ? 0 : 1)) * R + rr;  // at the share's front, or its end
#pragma unroll
            for (int c = 0; c < CH; c += BITS == 8 ? 1 : 2) {
              if (BITS == 8)
                *reinterpret_cast<float2*>(a.part + slot * HD + 16 * c + 2 * g) = make_float2(o[c][j][e], o[c][j][2 + e]);
              else
                *reinterpret_cast<float4*>(a.part + slot * HD + 16 * c + 4 * g) =
                    make_float4(o[c][j][e], o[c][j][2 + e], o[c + 1][j][e], o[c + 1][j][2 + e]);
            }
            if (g == 0) *reinterpret_cast<float2*>(a.stat + 2 * slot) = make_float2(m[j][e], sum);
          }
        }
      fresh = true;
      head = false;
    }
    at.next(a);
  }
  if (!ok && lane == 0) atomicCAS(a.status, 0, (int)EE_ERR_TIMEOUT);
  // whatever has been issued lands before the CTA ends
  for (int i = done; i < issued; ++i) mbar_wait(full + 8 * (i % NS), (uint32_t)(i / NS & 1), 1000000000ull);
  pdl_wait();
}

// The rows whose item a border cut, rows without keys of their own, and behind a
// prefix every row. A warp per (token, head), or a CTA (MANY).
template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(kPrJoin) cache_join_kernel(const __grid_constant__ CacheAttnArgs a, int most) {
  __shared__ PrList<kPrJoin> list;
  __shared__ JoinSmem<HD> sh;
  __shared__ CacheSeq seq;
  __shared__ long long seq_first;
  __shared__ int found;  // the token's sequence: the first that claims it, should a table that decreases have several
  const int tok = blockIdx.x;
  if (threadIdx.x == 0) found = 0x7fffffff;
  __syncthreads();
  const int per = (a.c.n_seq + kPrJoin - 1) / kPrJoin;
  CacheSeq hit{};
  int hit_b = -1;
  long long hit_at = 0;  // steps of the thread's own sequences before the token's
  const long long total = pr_list<kPrJoin>(a, &list, per, a.c.n_seq, [&](int b, const CacheSeq& s, long long before) {
    if (hit_b < 0 && tok >= s.q0 && tok < s.q0 + s.qlen) {
      hit = s;
      hit_b = b;
      hit_at = before;
      atomicMin(&found, b);
    }
  });
  if (hit_b >= 0 && hit_b == found) {
    seq = hit;
    seq_first = list.before[threadIdx.x] + hit_at;
  }
  __syncthreads();
  // what hangs on lengths and offsets alone, under the kernel before this one
  const bool there = found != 0x7fffffff;
  const int h = MANY ? blockIdx.y : blockIdx.y * (kPrJoin / 32) + (threadIdx.x >> 5);
  int r = 0;
  long long w0 = 0, n = 0, front = 0;  // parts of its own: their first worker, their number, where the first's lies
  if (there && h < a.n_q) {
    const CacheSeq s = seq;
    int steps;
    list_steps(a, s, steps);
    r = (tok - s.q0) * a.group + h % a.group;
    if (steps > 0) {
      const long long share = pr_share(total, most, kCaMinSteps);
      const long long first = seq_first + (long long)((r >> a.rows_log2) * a.c.n_kv + h / a.group) * steps;
      w0 = pr_div(first, share);
      n = pr_div(first + steps - 1, share) - w0 + 1;
      front = w0 * share == first ? 0 : a.rows;  // else the first part is at its share's end
    }
  }
  pdl_entry();  // by every thread, the ones that return too: this grid must not end before the one it follows
  if (!there || h >= a.n_q) return;  // rows outside the sequences stay as they were
  if (n == 1 && !a.pre_splits) return;  // in one share: written already
  const long long row = (long long)tok * a.n_q + h, hop = (long long)a.tq * a.n_q;
  r &= a.rows - 1;
  auto slot = [&](long long i) {
    if (i >= n) return a.whole + (1 + i - n) * hop + row;  // a part of the prefix
    if (n == 1) return a.whole + row;
    return (w0 + i) * 2 * a.rows + (i == 0 ? front : 0) + r;
  };
  T* out = reinterpret_cast<T*>(a.out) + (long long)tok * a.o_tok + h * a.o_head;
  if (MANY) join_row<T, HD>(a.part, a.stat, n + a.pre_splits, slot, out, &sh);
  else join_row_warp<T, HD>(a.part, a.stat, n + a.pre_splits, slot, out);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// The maps of the codes as rows of hd * bits / 8 bytes: in boxes of 32 rows,
// swizzled, for few rows; in boxes of a page (at most 128), plain, for many.
struct CacheMaps {
  CUtensorMap k, v;
};

// How a call runs: 8-row tiles a warp of the kernel for few rows, or (0) the
// tensor-core kernel and its parts of the keys.
struct CachePlan {
  int nt, splits;
};

template <typename T, int HD, int BITS, int NT>
int launch_cache_rows(const CacheMaps& m, const CacheAttnArgs& a, cudaStream_t s) {
  using S = CaShape<HD, BITS, NT>;
  auto fn = cache_rows_kernel<T, HD, BITS, NT>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  // beside the prefix's CTAs, where they leave half of the SMs or more
  const int sms = device_sms(), ctas = a.pre_ctas > 0 && 2 * a.pre_ctas <= sms ? sms - a.pre_ctas : sms, most = ctas * S::WORKERS;
  if (launch_pdl(fn, dim3(ctas), dim3(S::THREADS), S::SMEM, s, m.k, m.v, a) != cudaSuccess) return EE_ERR_LAUNCH;
  // parts of a row, on average: a CTA per row from 16 of its own on, or more than 32 of the prefix (64 x 16 rows with 16
  // of them: 8 us with a CTA a row, 4 with a warp)
  const long long blocks = (long long)a.tq * a.group / a.rows;
  const long long items = (blocks > a.c.n_seq ? blocks : a.c.n_seq) * a.c.n_kv;
  const cudaError_t e =
      most > 16 * items || a.pre_splits > 32
          ? launch_pdl(cache_join_kernel<T, HD, true>, dim3((unsigned)a.tq, a.n_q), dim3(kPrJoin), 0, s, a, most)
          : launch_pdl(cache_join_kernel<T, HD, false>, dim3((unsigned)a.tq, (a.n_q + kPrJoin / 32 - 1) / (kPrJoin / 32)),
                       dim3(kPrJoin), 0, s, a, most);
  return e == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}

template <typename T, int HD, int BITS>
int launch_cache_tc(const CacheMaps& m, const PromptTcArgs& a, cudaStream_t s) {
  auto fn = prompt_tc_kernel<T, HD, BITS>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  CUtensorMap mq;
  if (!prompt_head_map(&mq, a.p.q, HD, a.p.n_q, a.p.tq, a.p.q_head, a.p.q_tok, a.p.group, a.tpt)) return EE_ERR_SHAPE;
  // at most one partial tile per sequence beyond the rows' whole tiles
  const long long items = ((long long)a.p.tq / a.tpt + a.p.n_seq) * a.p.n_kv * a.p.splits;
  if (items > 0x7fffffff) return EE_ERR_SHAPE;
  const int sms = device_sms();
  const bool keys = a.c.width > 0;  // without, any map does: none of them is loaded by
  return launch_pdl(fn, dim3((unsigned)(items < sms ? items : sms)), dim3(PtThreads<BITS>::N), pt_smem<HD, BITS>(), s, mq,
                    keys ? m.k : mq, keys ? m.v : mq, a) == cudaSuccess
             ? EE_OK
             : EE_ERR_LAUNCH;
}

template <typename T, int HD>
int launch_cache_few(const CacheMaps& m, const CacheAttnArgs& a, const CachePlan& p, int bits, cudaStream_t s);
template <typename T, int HD>
int launch_cache_many(const CacheMaps& m, const PromptTcArgs& a, int bits, cudaStream_t s);

#define EE_CACHE_ATTN(T, HD)                                                                                           \
  template <>                                                                                                          \
  int launch_cache_few<T, HD>(const CacheMaps& m, const CacheAttnArgs& a, const CachePlan& p, int bits,                \
                              cudaStream_t s) {                                                                        \
    if (p.nt > 1)                                                                                                      \
      return bits == 8 ? launch_cache_rows<T, HD, 8, 2>(m, a, s) : launch_cache_rows<T, HD, 4, 2>(m, a, s);            \
    return bits == 8 ? launch_cache_rows<T, HD, 8, 1>(m, a, s) : launch_cache_rows<T, HD, 4, 1>(m, a, s);              \
  }                                                                                                                    \
  template <>                                                                                                          \
  int launch_cache_many<T, HD>(const CacheMaps& m, const PromptTcArgs& a, int bits, cudaStream_t s) {                  \
    return bits == 8 ? launch_cache_tc<T, HD, 8>(m, a, s) : launch_cache_tc<T, HD, 4>(m, a, s);                        \
  }

}  // namespace ee
