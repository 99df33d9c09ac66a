// ee_prompt.cu -- C ABI: attention over packed prompts (causal or full,
// grouped heads, keys that may reach further back than the queries).
#include <atomic>
#include <cfloat>

#include "ee_host.h"
#include "ee_prompt.cuh"
#include "ee_prompt_tc.cuh"

namespace ee {

// ---------------------------------------------------------------------------
// few query rows per key head
// ---------------------------------------------------------------------------
// A row is (token, head of the key head's group), so a key head's whole group
// shares one read of its keys; an item is 16 rows of one sequence and key head
// against the sequence's keys, cut into steps of 16 keys. All items' steps
// form one list, and every warp of the grid takes an equal, contiguous share
// of it whatever the sequences' lengths: each warp is on its own, streaming
// its steps' keys and values through a ring (cp.async, no barrier between
// warps, the next item's loads under the current one's last steps) with a
// running maximum and sum. An item that lies in one share is written at once;
// of an item cut by a border each warp leaves its sums in the workspace, at
// most one at either end of its share, and prompt_join_kernel adds them up.
// HBM-bound on the keys and values, with 128 KB of loads in flight per SM: 64
// sequences of 1 to 1632 keys, 16 / 4 heads of 128: 25 us, 4.4 TB/s, of which
// the arithmetic costs 3 (without it: 22); 8 x 4096 keys, 32 / 8 heads: 26 us,
// 5.2 TB/s; the join takes 5 more. (One CTA per item and part of its keys, joined in a cluster or by a
// second launch, left SMs idle for 27 % of the time on 64 sequences of 1 to
// 1632 keys and waited for each CTA's first loads again: 36 us.)
constexpr int kPrStep = 16, kPrMinSteps = 6;   // keys of a step; steps that are worth a warp
template <int HD> constexpr int pr_warps() { return HD == 128 ? 8 : 16; }
constexpr int kPrStages = 3;
template <int HD> constexpr int pr_stage() { return 2 * kPrStep * HD * 2; }  // K and V of a step
template <int HD> constexpr int pr_smem() { return pr_warps<HD>() * kPrStages * pr_stage<HD>(); }

// steps of sequence b's items (all its row blocks and key heads), and of one item
EE_DEV long long pr_steps(const PromptArgs& a, const PromptSeq& s, int& per_item) {
  per_item = (s.klen + kPrStep - 1) / kPrStep;
  return (long long)((s.qlen * a.group + 15) / 16) * a.n_kv * per_item;
}

// The list of steps: its length, and for every thread the steps before its
// share of the sequences (`per` each, consecutive). All threads of the CTA.
// visit(b, s, before): each of the thread's sequences and the steps of its own
// ones before it.
template <int THREADS>
struct PrList {
  long long before[THREADS];
  long long warp_sum[THREADS / 32];
};
template <int THREADS, typename Visit>
EE_DEV long long pr_list(const PromptArgs& a, PrList<THREADS>* sh, int per, Visit visit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long mine = 0;
  for (int b = tid * per; b < min((tid + 1) * per, a.n_seq); ++b) {
    int n;
    const PromptSeq s = prompt_seq(a, b);
    visit(b, s, mine);
    mine += pr_steps(a, s, n);
  }
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) sh->warp_sum[warp] = inc;
  __syncthreads();
  long long base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) base += sh->warp_sum[w];
    total += sh->warp_sum[w];
  }
  sh->before[tid] = base + inc - mine;
  __syncthreads();
  return total;
}
// Steps in a warp's share of a list of `total`, for `most` warps: warp w takes
// steps w * share .., so step x belongs to warp x / share.
EE_DEV long long pr_div(long long a, long long b) {  // of values >= 0, mostly below 2^32
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
EE_DEV long long pr_share(long long total, int most) {
  const long long q = pr_div(total + most - 1, most);
  return q < kPrMinSteps ? kPrMinSteps : q;
}

EE_DEV void pr_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
EE_DEV void pr_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// A place in the list: a step of an item of a sequence.
struct PrAt {
  int b, step, per_item, item, items;  // sequence; step of the item; steps per item; item of the sequence (row block
  PromptSeq s;                         // x key heads + key head) and their number
  EE_DEV void enter(const PromptArgs& a, int seq) {  // sequence `seq` or the next one that has steps
    for (b = seq; b < a.n_seq; ++b) {
      s = prompt_seq(a, b);
      const long long n = pr_steps(a, s, per_item);
      if (n > 0) {
        items = (s.qlen * a.group + 15) / 16 * a.n_kv;
        break;
      }
    }
    item = step = 0;
  }
  EE_DEV void next(const PromptArgs& a) {
    if (++step < per_item) return;
    step = 0;
    if (++item == items) enter(a, b + 1);
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(32 * pr_warps<HD>(), 1) prompt_rows_kernel(const __grid_constant__ PromptArgs a) {
  constexpr int NW = pr_warps<HD>(), NT = 32 * NW, NS = kPrStages;
  constexpr int RB = HD * 2;             // bytes per key row
  constexpr int CH = HD / 8;             // 16-byte chunks per key row
  constexpr int TILE = kPrStep * RB;
  extern __shared__ __align__(128) char smem[];
  __shared__ PrList<NT> sh;
  pdl_entry();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3, mi = lane >> 3;
  const int per = (a.n_seq + NT - 1) / NT;
  const long long total = pr_list<NT>(a, &sh, per, [](int, const PromptSeq&, long long) {});
  const long long share = pr_share(total, (int)gridDim.x * NW);
  const long long me = (long long)warp * gridDim.x + blockIdx.x;  // neighbours in the list on different SMs
  const long long first = me * share;
  if (first >= total) return;
  int left = (int)(total - first < share ? total - first : share);  // steps to go
  // where the share starts: the last thread whose sequences begin at or before it, then along its sequences
  PrAt ld{};
  {
    int lo = 0;
#pragma unroll
    for (int o = NT / 2; o > 0; o >>= 1)
      if (sh.before[lo + o] <= first) lo += o;
    long long at = first - sh.before[lo];
    ld.enter(a, lo * per);
    while (ld.b < a.n_seq) {
      const long long n = (long long)ld.items * ld.per_item;
      if (at < n) break;
      at -= n;
      ld.enter(a, ld.b + 1);
    }
    if (ld.b >= a.n_seq) return;  // the lengths have changed meanwhile
    ld.item = (int)pr_div(at, ld.per_item);
    ld.step = (int)(at - (long long)ld.item * ld.per_item);
  }
  PrAt at = ld;
  const uint32_t ring = smem_u32(smem) + warp * NS * 2 * TILE;
  auto off = [](int row, int ch) { return row * RB + ((ch ^ (row & 7)) << 4); };
  const int lrow = lane / CH, lch = lane % CH;  // this lane's row and chunk of every 32 / CH rows
  // where this lane reads step `ld` from, and the keys that the sequence has from there on
  const char *kp = nullptr, *vp = nullptr;
  int valid = 0;
  const long long k_row = a.k_tok * 2, v_row = a.v_tok * 2;
  auto aim = [&]() {
    const int kvh = ld.item % a.n_kv;
    const long long k0 = ld.s.k0 + (long long)ld.step * kPrStep + lrow;
    kp = reinterpret_cast<const char*>(a.k) + k0 * k_row + kvh * a.k_head * 2 + lch * 16;
    vp = reinterpret_cast<const char*>(a.v) + k0 * v_row + kvh * a.v_head * 2 + lch * 16;
    valid = ld.s.klen - ld.step * kPrStep - lrow;
  };
  aim();
  // the keys and values of step `ld`, those past the sequence's end zero-filled; then on to the next step
  auto load = [&](int buf) {
    const uint32_t d = ring + buf * 2 * TILE;
    const char *kr = kp, *vr = vp;
#pragma unroll
    for (int i = 0; i < kPrStep * CH / 32; ++i) {
      const int row = lrow + i * (32 / CH);
      const bool ok = i * (32 / CH) < valid;
      // a copy of nothing reads nothing: any address will do
      cp_async16(d + off(row, lch), ok ? kr : reinterpret_cast<const char*>(a.k), ok);
      cp_async16(d + TILE + off(row, lch), ok ? vr : reinterpret_cast<const char*>(a.v), ok);
      kr += 32 / CH * k_row;
      vr += 32 / CH * v_row;
    }
    if (ld.step + 1 < ld.per_item) {
      ++ld.step;
      kp += kPrStep * k_row;
      vp += kPrStep * v_row;
      valid -= kPrStep;
    } else {
      ld.next(a);
      if (ld.b < a.n_seq) aim();
    }
  };
  int ahead = 0;  // steps loaded beyond the current one
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (i < left && ld.b < a.n_seq) {
      load(i);
      ++ahead;
    }
    cp_async_commit();
  }
  uint32_t qf[HD / 16][4];
  float o[HD / 8][4];
  float m0 = 0.f, m1 = 0.f, l0 = 0.f, l1 = 0.f;
  int rows = 0, r0 = 0, kvh = 0, lim0 = 0, lim1 = 0;
  bool fresh = true;      // the item's first step of this share
  int from = 0;           // that step
  bool head = true;       // no item of the share has been finished yet
  int buf = 0;
  for (; left > 0 && ahead > 0; --left, --ahead) {
    if (fresh) {
      fresh = false;
      from = at.step;
      rows = at.s.qlen * a.group;
      r0 = at.item / a.n_kv * 16;
      kvh = at.item % a.n_kv;
      const int ra = min(r0 + g, rows - 1), rb = min(r0 + g + 8, rows - 1);
      auto qrow = [&](int r) {
        const int tok = r / a.group, h = kvh * a.group + r % a.group;
        return reinterpret_cast<const char*>(a.q) + ((long long)(at.s.q0 + tok) * a.q_tok + h * a.q_head) * 2;
      };
      const char *pa = qrow(ra), *pb = qrow(rb);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        qf[ks][0] = *reinterpret_cast<const uint32_t*>(pa + ks * 32 + t * 4);
        qf[ks][1] = *reinterpret_cast<const uint32_t*>(pb + ks * 32 + t * 4);
        qf[ks][2] = *reinterpret_cast<const uint32_t*>(pa + ks * 32 + 16 + t * 4);
        qf[ks][3] = *reinterpret_cast<const uint32_t*>(pb + ks * 32 + 16 + t * 4);
      }
      // keys below lim are seen by rows ra and rb
      lim0 = a.causal ? min(at.s.klen, at.s.klen - at.s.qlen + ra / a.group + 1) : at.s.klen;
      lim1 = a.causal ? min(at.s.klen, at.s.klen - at.s.qlen + rb / a.group + 1) : at.s.klen;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
      m0 = m1 = -INFINITY;
      l0 = l1 = 0.f;
    }
    if (left > NS - 1 && ld.b < a.n_seq) {
      load(buf == 0 ? NS - 1 : buf - 1);
      ++ahead;
    }
    cp_async_commit();
    cp_async_wait<NS - 1>();
    __syncwarp();
    const uint32_t kt = ring + buf * 2 * TILE, vt = kt + TILE;
    const int key = at.step * kPrStep;
    float p[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      uint32_t b[4];
      pr_ldsm(kt + off((mi >> 1) * 8 + (lane & 7), 2 * ks + (mi & 1)), b);
      mma16816<T>(p[0], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[0], b[1]);
      mma16816<T>(p[1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[2], b[3]);
    }
    if (__any_sync(0xffffffffu, key + kPrStep > min(lim0, lim1))) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int kk = key + 8 * j + 2 * t + c;
          if (kk >= lim0) p[j][c] = -INFINITY;
          if (kk >= lim1) p[j][2 + c] = -INFINITY;
        }
      }
    }
    float x0 = fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[1][0], p[1][1]));
    float x1 = fmaxf(fmaxf(p[0][2], p[0][3]), fmaxf(p[1][2], p[1][3]));
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
    }
    // fp16: weights up to 2^15
    const float n0 = fmaxf(m0, prompt_reference<T, 15>(x0 * a.scale_log2));
    const float n1 = fmaxf(m1, prompt_reference<T, 15>(x1 * a.scale_log2));
    // nothing seen yet: any finite reference will do, 2^-inf = 0
    const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
    if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
      const float c0 = ex2(m0 - u0), c1 = ex2(m1 - u1);
      m0 = n0;
      m1 = n1;
      l0 *= c0;
      l1 *= c1;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        o[i][0] *= c0;
        o[i][1] *= c0;
        o[i][2] *= c1;
        o[i][3] *= c1;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        p[j][c] = ex2(fmaf(p[j][c], a.scale_log2, -u0));
        p[j][2 + c] = ex2(fmaf(p[j][2 + c], a.scale_log2, -u1));
        l0 += p[j][c];
        l1 += p[j][2 + c];
      }
    }
    // 16 bits, as the product with v takes them (half a step each, in either direction; their sum above keeps fp32):
    // the whole error is 1.1 times that of a plain fp32 form (64 x 1 token behind 1..1632, bf16: 1.8e-3 to 1.6e-3)
    const uint32_t pa0 = Act<T>::pack2(p[0][0], p[0][1]), pa1 = Act<T>::pack2(p[0][2], p[0][3]);
    const uint32_t pa2 = Act<T>::pack2(p[1][0], p[1][1]), pa3 = Act<T>::pack2(p[1][2], p[1][3]);
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
      uint32_t b[4];
      pr_ldsm_t(vt + off((mi & 1) * 8 + (lane & 7), 2 * d + (mi >> 1)), b);
      mma16816<T>(o[2 * d], pa0, pa1, pa2, pa3, b[0], b[1]);
      mma16816<T>(o[2 * d + 1], pa0, pa1, pa2, pa3, b[2], b[3]);
    }
    __syncwarp();  // every lane has read the stage before it is loaded again
    if (++buf == NS) buf = 0;
    const bool end = at.step + 1 == at.per_item;
    if (end || left == 1) {
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
      }
      const bool whole = end && from == 0;
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        const int rr = g + 8 * hr, r = r0 + rr;
        if (r >= rows) continue;
        const float m = hr ? m1 : m0, l = hr ? l1 : l0;
        if (whole) {
          const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
          T* out = reinterpret_cast<T*>(a.out) + (long long)(at.s.q0 + r / a.group) * a.o_tok +
                   (kvh * a.group + r % a.group) * a.o_head;
#pragma unroll
          for (int i = 0; i < HD / 8; ++i)
            *reinterpret_cast<uint32_t*>(out + 8 * i + 2 * t) = Act<T>::pack2(o[i][2 * hr] * inv, o[i][2 * hr + 1] * inv);
        } else {
          const long long slot = (me * 2 + (head ? 0 : 1)) * 16 + rr;  // at the share's front, or its end
#pragma unroll
          for (int i = 0; i < HD / 8; ++i)
            *reinterpret_cast<float2*>(a.part + slot * HD + 8 * i + 2 * t) = make_float2(o[i][2 * hr], o[i][2 * hr + 1]);
          if (t == 0) *reinterpret_cast<float2*>(a.stat + 2 * slot) = make_float2(m, l);
        }
      }
      fresh = true;
      head = false;
    }
    at.next(a);
  }
  cp_async_wait<0>();
}

// Joins the partial rows of one (token, head) by one CTA: `n` of them at
// slot(i) of part / stat, 1024 at a time with a running maximum. A thread per
// part for the weights, then hd / 4 threads across the values and the rest
// across the parts, so that both passes have their loads in flight together.
constexpr int kPrJoin = 256, kPrChunk = 4 * kPrJoin;
template <int HD>
struct JoinSmem {
  float wt[kPrChunk], red[2][kPrJoin / 32];
  float4 sv[4 * kPrJoin / HD][HD / 4];
};
template <typename T, int HD, typename Slot>
EE_DEV void join_row(const PromptArgs& a, long long n, Slot slot, T* out, JoinSmem<HD>* sh) {
  constexpr int LANES = HD / 4, GROUPS = kPrJoin / LANES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = tid % LANES, grp = tid / LANES;
  const float2* stat = reinterpret_cast<const float2*>(a.stat);
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (long long i0 = 0; i0 < n; i0 += kPrChunk) {
    const int here = (int)(n - i0 < kPrChunk ? n - i0 : kPrChunk);
    float2 st[kPrChunk / kPrJoin];
    float x = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPrChunk / kPrJoin; ++j) {
      const int i = tid + j * kPrJoin;
      st[j] = i < here ? __ldg(stat + slot(i0 + i)) : make_float2(-INFINITY, 0.f);
      x = fmaxf(x, st[j].x);
    }
    x = warp_max(x);
    if (lane == 0) sh->red[0][warp] = x;
    __syncthreads();
    float top = m;
#pragma unroll
    for (int i = 0; i < kPrJoin / 32; ++i) top = fmaxf(top, sh->red[0][i]);
    const float u = top == -INFINITY ? 0.f : top, old = exp2f(m - u);
    m = top;
    l *= old;
    acc = make_float4(acc.x * old, acc.y * old, acc.z * old, acc.w * old);
#pragma unroll
    for (int j = 0; j < kPrChunk / kPrJoin; ++j) {
      // weight 0: the part has seen no key, its sums need not have been written
      const float f = st[j].y == 0.f ? 0.f : exp2f(st[j].x - u);
      l += f * st[j].y;
      sh->wt[tid + j * kPrJoin] = f;
    }
    __syncthreads();
    for (int i = grp; i < here; i += 8 * GROUPS) {  // loads first: none waits for another's weight
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = __ldg(reinterpret_cast<const float4*>(a.part + slot(i0 + min(i + k * GROUPS, here - 1)) * HD) + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = i + k * GROUPS < here ? sh->wt[i + k * GROUPS] : 0.f;
        if (w != 0.f) {
          acc.x += w * v[k].x;
          acc.y += w * v[k].y;
          acc.z += w * v[k].z;
          acc.w += w * v[k].w;
        }
      }
    }
    __syncthreads();
  }
  l = warp_sum(l);
  if (lane == 0) sh->red[1][warp] = l;
  sh->sv[grp][c] = acc;
  __syncthreads();
  if (grp) return;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kPrJoin / 32; ++i) l += sh->red[1][i];
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) {
    const float4 v = sh->sv[g][c];
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
  *reinterpret_cast<uint2*>(out + 4 * c) =
      make_uint2(Act<T>::pack2(acc.x * inv, acc.y * inv), Act<T>::pack2(acc.z * inv, acc.w * inv));
}

// The parts of the tensor-core kernel's keys, by (part, token, head).
template <typename T, int HD>
__global__ void __launch_bounds__(kPrJoin) prompt_combine_kernel(const __grid_constant__ PromptArgs a) {
  __shared__ JoinSmem<HD> sh;
  pdl_entry();
  const int tok = blockIdx.x, h = blockIdx.y;
  // rows outside the sequences have no parts and stay as they were
  if (tok < __ldg(a.cu_q) || tok >= __ldg(a.cu_q + a.n_seq)) return;
  const long long step = (long long)a.tq * a.n_q, at = (long long)tok * a.n_q + h;
  join_row<T, HD>(a, a.splits, [&](long long i) { return at + i * step; },
                  reinterpret_cast<T*>(a.out) + (long long)tok * a.o_tok + h * a.o_head, &sh);
}

// The same by one warp, 32 parts at a time, hd / 32 values a lane: for items of
// few parts, where a CTA's barriers cost more than its width saves.
template <typename T, int HD, typename Slot>
EE_DEV void join_row_warp(const PromptArgs& a, long long n, Slot slot, T* out) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.f, v[V] = {};
  for (long long i0 = 0; i0 < n; i0 += 32) {
    const int here = (int)(n - i0 < 32 ? n - i0 : 32);
    const float2 st = lane < here ? __ldg(reinterpret_cast<const float2*>(a.stat) + slot(i0 + lane))
                                  : make_float2(-INFINITY, 0.f);
    const float top = fmaxf(m, warp_max(st.x));
    const float u = top == -INFINITY ? 0.f : top, old = exp2f(m - u);
    m = top;
    const float f = st.y == 0.f ? 0.f : exp2f(st.x - u);
    l = l * old + f * st.y;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= old;
    for (int i = 0; i < here; i += 8) {  // loads first: none waits for another's weight
      float2 x[8][V / 2];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < V / 2; ++e)
          x[k][e] = __ldg(reinterpret_cast<const float2*>(a.part + slot(i0 + min(i + k, here - 1)) * HD + lane * V) + e);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(0xffffffffu, f, (i + k) & 31);  // 0 past the last part
        if (w != 0.f) {
#pragma unroll
          for (int e = 0; e < V / 2; ++e) {
            v[2 * e] += w * x[k][e].x;
            v[2 * e + 1] += w * x[k][e].y;
          }
        }
      }
    }
  }
  l = warp_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
#pragma unroll
  for (int e = 0; e < V; e += 2)
    *reinterpret_cast<uint32_t*>(out + lane * V + e) = Act<T>::pack2(v[e] * inv, v[e + 1] * inv);
}

// The rows of the kernel for few rows whose item was cut, and rows without
// keys. MANY: a CTA per (token, head); else a warp. The search reads only the
// offsets, which are final -- the kernel before this one has waited for them --
// so it runs under that kernel's end.
template <typename T, int HD, bool MANY>
__global__ void __launch_bounds__(kPrJoin) prompt_join_kernel(const __grid_constant__ PromptArgs a, int most) {
  __shared__ PrList<kPrJoin> list;
  __shared__ JoinSmem<HD> sh;
  __shared__ PromptSeq seq;
  __shared__ long long seq_first;
  __shared__ int found;  // the token's sequence: the first that claims it, should a table that decreases have several
  const int tok = blockIdx.x;
  if (threadIdx.x == 0) found = 0x7fffffff;
  __syncthreads();
  const int per = (a.n_seq + kPrJoin - 1) / kPrJoin;
  PromptSeq hit{};
  int hit_b = -1;
  long long hit_at = 0;  // steps of the thread's own sequences before the token's
  const long long total = pr_list<kPrJoin>(a, &list, per, [&](int b, const PromptSeq& s, long long before) {
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
  pdl_entry();  // by every thread, the ones that return too: this grid must not end before the one it follows
  if (found == 0x7fffffff) return;  // rows outside the sequences stay as they were
  const PromptSeq s = seq;
  int steps;
  pr_steps(a, s, steps);
  const long long share = pr_share(total, most);
  const int h = MANY ? blockIdx.y : blockIdx.y * (kPrJoin / 32) + (threadIdx.x >> 5);
  if (h < a.n_q) {
    const int kvh = h / a.group, r = (tok - s.q0) * a.group + h % a.group;
    long long w0 = 0, n = 0, front = 0;
    if (steps > 0) {
      const long long first = seq_first + (long long)(r / 16 * a.n_kv + kvh) * steps;
      w0 = pr_div(first, share);
      n = pr_div(first + steps - 1, share) - w0 + 1;
      if (n == 1) return;  // in one share: written already
      front = w0 * share == first ? 0 : 16;  // else the first part is at its share's end
    }
    auto slot = [&](long long i) { return (w0 + i) * 32 + (i == 0 ? front : 0) + r % 16; };
    T* out = reinterpret_cast<T*>(a.out) + (long long)tok * a.o_tok + h * a.o_head;
    if (MANY) join_row<T, HD>(a, n, slot, out, &sh);
    else join_row_warp<T, HD>(a, n, slot, out);
  }
}

// How a call runs, by what the host knows of it: rows (queries x group) per
// sequence and key head, and keys per sequence, on average.
//   tc      more than 16 rows: the tensor-core kernel's 128-row tiles (8 x 50
//           new tokens behind 816, 16 heads of 128: 19.6 us, where 64-row warp
//           MMA units took 68), 16 or fewer: the kernel for few rows' single
//           MMA tile. One kernel runs the whole call: a long prompt among many
//           single tokens is walked 16 rows at a time (4096 tokens beside 300 x
//           1 behind 816, 16 heads of 128: 920 us, as two calls 65 + 310)
//   splits  of the tensor-core kernel: where its items would leave SMs idle,
//           parts of 512 keys or more, joined by a second launch
constexpr long long kPrRows = 16, kPtMinKeys = 512;
struct PromptPlan { bool tc; int splits; };
static PromptPlan prompt_plan(long long tq, long long tk, int n_seq, int n_q, int n_kv) {
  PromptPlan pl{false, 1};
  if (n_seq < 1) return pl;
  const int group = n_q / n_kv;
  const long long rows = tq * group;
  pl.tc = rows > kPrRows * n_seq && tk > 0 && group <= 128;
  if (!pl.tc) return pl;
  const long long per = 2 * (128 / group) * group;  // rows of an item: two tiles of whole tokens
  const long long items = (rows / per > n_seq ? rows / per : n_seq) * n_kv;
  const long long want = device_sms() / items, most = tk / n_seq / kPtMinKeys;
  const long long s = want < most ? want : most;
  pl.splits = s < 1 ? 1 : (int)s;
  return pl;
}
static long long prompt_partials(const PromptPlan& pl, long long tq, int n_q, int hd) {  // partial rows
  if (pl.tc) return pl.splits > 1 ? pl.splits * tq * n_q : 0;
  return (long long)device_sms() * (hd == 128 ? pr_warps<128>() : pr_warps<64>()) * 32;
}
static size_t prompt_ws_bytes(const PromptPlan& pl, long long tq, int n_q, int hd) {
  return (size_t)prompt_partials(pl, tq, n_q, hd) * (hd + 2) * 4;
}

template <typename T, int HD>
static int launch_combine(const PromptArgs& a, cudaStream_t s) {
  if (a.splits == 1) return EE_OK;
  return launch_pdl(prompt_combine_kernel<T, HD>, dim3((unsigned)a.tq, a.n_q), dim3(kPrJoin), 0, s, a) == cudaSuccess
             ? EE_OK
             : EE_ERR_LAUNCH;
}

template <typename T, int HD>
static int launch_rows(const PromptArgs& a, cudaStream_t s) {
  auto fn = prompt_rows_kernel<T, HD>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  const int sms = device_sms();
  if (launch_pdl(fn, dim3(sms), dim3(32 * pr_warps<HD>()), pr_smem<HD>(), s, a) != cudaSuccess) return EE_ERR_LAUNCH;
  // parts of an item, on average: a CTA per row from 16 on
  const long long items = (((long long)a.tq * a.group / 16 > a.n_seq ? (long long)a.tq * a.group / 16 : a.n_seq)) * a.n_kv;
  const int most = sms * pr_warps<HD>();
  const cudaError_t e =
      most > 16 * items
          ? launch_pdl(prompt_join_kernel<T, HD, true>, dim3((unsigned)a.tq, a.n_q), dim3(kPrJoin), 0, s, a, most)
          : launch_pdl(prompt_join_kernel<T, HD, false>, dim3((unsigned)a.tq, (a.n_q + kPrJoin / 32 - 1) / (kPrJoin / 32)),
                       dim3(kPrJoin), 0, s, a, most);
  return e == cudaSuccess ? EE_OK : EE_ERR_LAUNCH;
}

int* gemm_status_ptr();  // ee_ops.cu: the status word of the tensor-core kernels on the current device

// [tokens][heads][hd] by strides, read in boxes of 64 columns of bh heads and bt tokens
static bool make_head_map(CUtensorMap* map, const void* base, int hd, int heads, long long tokens, long long head,
                          long long tok, int bh, int bt) {
  auto enc = tmap_encoder();
  if (!enc) return false;
  if (heads == 1) head = hd;   // strides of dimensions of one entry mean nothing
  if (tokens == 1) tok = (long long)hd * heads;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)tok * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)bh, (cuuint32_t)bt}, estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr unsigned long long kPtWaitNs = 1000000000ull;
static std::atomic<unsigned long long> g_wait_limit{kPtWaitNs};

template <typename T, int HD>
static int launch_tc(const PromptArgs& p, cudaStream_t s) {
  auto fn = prompt_tc_kernel<T, HD>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  const DevProps* dp = device_props();
  if (!dp) return EE_ERR_DEVICE;
  PromptTcArgs a{};
  a.p = p;
  a.tpt = 128 / p.group;
  a.status = gemm_status_ptr();
  a.timeout_ns = g_wait_limit.load(std::memory_order_relaxed);
  if (!a.status) return EE_ERR_DEVICE;
  CUtensorMap mq, mk, mv;
  if (!make_head_map(&mq, p.q, HD, p.n_q, p.tq, p.q_head, p.q_tok, p.group, a.tpt) ||
      !make_head_map(&mk, p.k, HD, p.n_kv, p.tk, p.k_head, p.k_tok, 1, 128) ||
      !make_head_map(&mv, p.v, HD, p.n_kv, p.tk, p.v_head, p.v_tok, 1, 128))
    return EE_ERR_SHAPE;  // a stride the loads cannot address
  // at most one partial unit per sequence beyond the rows' whole units
  const long long items = ((long long)p.tq / (2 * a.tpt) + p.n_seq) * p.n_kv * p.splits;
  if (items > 0x7fffffff) return EE_ERR_SHAPE;
  const unsigned grid = (unsigned)(items < dp->sms ? items : dp->sms);
  if (launch_pdl(fn, dim3(grid), dim3(kPtThreads), pt_smem<HD>(), s, mq, mk, mv, a) != cudaSuccess) return EE_ERR_LAUNCH;
  return launch_combine<T, HD>(p, s);
}

template <typename T>
static int launch_prompt(const PromptArgs& a, const PromptPlan& pl, int hd, cudaStream_t s) {
  if (pl.tc) return hd == 64 ? launch_tc<T, 64>(a, s) : launch_tc<T, 128>(a, s);
  return hd == 64 ? launch_rows<T, 64>(a, s) : launch_rows<T, 128>(a, s);
}

}  // namespace ee

using namespace ee;

extern "C" {

size_t ee_prompt_attention_workspace_bytes(int64_t tq, int64_t tk, int32_t n_seq, int32_t n_q, int32_t n_kv,
                                           int32_t head_dim) {
  if (tq < 0 || tk < 0 || n_seq < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv || tq > 0x7fffff00 || tk > 0x7fffff00) return 0;
  return prompt_ws_bytes(prompt_plan(tq, tk, n_seq, n_q, n_kv), tq, n_q, head_dim);
}

int ee_prompt_attention_wait_limit(uint64_t ns) {
  g_wait_limit.store(ns ? ns : kPtWaitNs, std::memory_order_relaxed);
  return EE_OK;
}

int ee_prompt_attention(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok, int64_t k_head,
                        const void* v, int64_t v_tok, int64_t v_head, void* out, int64_t o_tok, int64_t o_head,
                        const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_lens, int64_t tq, int64_t tk,
                        int32_t n_seq, int32_t n_q, int32_t n_kv, int32_t head_dim, int32_t causal, float scale,
                        int32_t act_dtype, void* workspace, size_t workspace_bytes, ee_stream_t stream) {
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return EE_ERR_UNSUPPORTED;
  if (tq < 0 || tk < 0 || n_seq < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0) return EE_ERR_SHAPE;
  if (tq > 0x7fffff00 || tk > 0x7fffff00 || n_kv > 65535 || n_q > 65535) return EE_ERR_SHAPE;
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale > 0.f) || !(scale_log2 <= FLT_MAX)) return EE_ERR_ARG;
  if (tq == 0 || n_seq == 0) return EE_OK;
  if (!q || !out || !cu_q || (tk && (!k || !v)) || (!cu_k && tk != tq)) return EE_ERR_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return EE_ERR_ALIGN;
  if (((uintptr_t)cu_q | (uintptr_t)cu_k | (uintptr_t)k_lens) & 3) return EE_ERR_ALIGN;
  if ((q_tok | q_head | k_tok | k_head | v_tok | v_head | o_tok | o_head) % 8 != 0) return EE_ERR_ALIGN;
  const int rc = check_device();
  if (rc) return rc;
  const PromptPlan pl = prompt_plan(tq, tk, n_seq, n_q, n_kv);
  const size_t need = prompt_ws_bytes(pl, tq, n_q, head_dim);
  if (need && (!workspace || workspace_bytes < need)) return EE_ERR_WORKSPACE;
  if (need && !aligned16(workspace)) return EE_ERR_ALIGN;
  PromptArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out;
  a.cu_q = cu_q;
  a.cu_k = cu_k ? cu_k : cu_q;
  a.k_lens = k_lens;
  a.q_tok = q_tok; a.q_head = q_head; a.k_tok = k_tok; a.k_head = k_head;
  a.v_tok = v_tok; a.v_head = v_head; a.o_tok = o_tok; a.o_head = o_head;
  a.tq = (int)tq; a.tk = (int)tk; a.n_seq = n_seq;
  a.n_q = n_q; a.n_kv = n_kv; a.group = n_q / n_kv;
  a.causal = causal != 0;
  a.scale_log2 = scale_log2;
  a.splits = pl.splits;
  a.part = reinterpret_cast<float*>(workspace);
  a.stat = a.part + (size_t)prompt_partials(pl, tq, n_q, head_dim) * head_dim;
  cudaStream_t s = (cudaStream_t)stream;
  return act_dtype == EE_BF16 ? launch_prompt<__nv_bfloat16>(a, pl, head_dim, s)
                               : launch_prompt<__half>(a, pl, head_dim, s);
}

}  // extern "C"
