// ee_prompt_list.cuh -- attention for few query rows, over packed or cached
// keys: all items' steps over their keys as one list of which every worker of
// the grid takes an equal share, and the join of items that a share's border
// cuts.
#pragma once

#include "ee_common.cuh"

namespace ee {

// The list of steps: its length, and for every thread the steps before its
// share of the sequences (`per` each, consecutive). All threads of the CTA.
// list_seq(a, b) is a sequence, list_steps(a, s, n) its steps (n: of an item).
// visit(b, s, before): each of the thread's sequences and the steps of its own
// ones before it.
template <int THREADS>
struct PrList {
  long long before[THREADS];
  long long warp_sum[THREADS / 32];
};
template <int THREADS, typename Args, typename Visit>
EE_DEV long long pr_list(const Args& a, PrList<THREADS>* sh, int per, int n_seq, Visit visit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long mine = 0;
  for (int b = tid * per; b < min((tid + 1) * per, n_seq); ++b) {
    int n;
    const auto s = list_seq(a, b);
    visit(b, s, mine);
    mine += list_steps(a, s, n);
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
// Steps in a worker's share of a list of `total`, for `most` workers: worker w
// takes steps w * share .., so step x belongs to worker x / share.
EE_DEV long long pr_div(long long a, long long b) {  // of values >= 0, mostly below 2^32
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
EE_DEV long long pr_share(long long total, int most, int least) {  // `least` steps are worth a worker
  const long long q = pr_div(total + most - 1, most);
  return q < least ? least : q;
}

EE_DEV void pr_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
EE_DEV void pr_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// Joins the partial rows of one (token, head) by one CTA: `n` of them at
// slot(i) of part / stat, 1024 at a time with a running maximum. A thread per
// part for the weights, then hd / 4 threads across the values and the rest
// across the parts, so that both passes have their loads in flight together.
// (Places of parts are 31-bit numbers: 2^31 rows would be 550 GB.)
constexpr int kPrJoin = 256, kPrChunk = 4 * kPrJoin;
template <int HD>
struct JoinSmem {
  float wt[kPrChunk], red[2][kPrJoin / 32];
  int at[kPrChunk];
  float4 sv[4 * kPrJoin / HD][HD / 4];
};
template <typename T, int HD, typename Slot>
EE_DEV void join_row(const float* part, const float* stats, long long n, Slot slot, T* out, JoinSmem<HD>* sh) {
  constexpr int LANES = HD / 4, GROUPS = kPrJoin / LANES;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = tid % LANES, grp = tid / LANES;
  const float2* stat = reinterpret_cast<const float2*>(stats);
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (long long i0 = 0; i0 < n; i0 += kPrChunk) {
    const int here = (int)(n - i0 < kPrChunk ? n - i0 : kPrChunk);
    float2 st[kPrChunk / kPrJoin];
    float x = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPrChunk / kPrJoin; ++j) {
      const int i = tid + j * kPrJoin;
      const int at = (int)slot(i0 + min(i, here - 1));
      sh->at[i] = at;
      st[j] = i < here ? __ldg(stat + at) : make_float2(-INFINITY, 0.f);
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
      // a part that has seen no key: its sums need not have been written. (A weight that underflows still counts, should
      // its part hold a NaN.)
      const bool seen = st[j].y != 0.f;
      const float f = seen ? exp2f(st[j].x - u) : 0.f;
      l += f * st[j].y;
      sh->wt[tid + j * kPrJoin] = seen ? f : -1.f;
    }
    __syncthreads();
    for (int i = grp; i < here; i += 8 * GROUPS) {  // loads first: none waits for another's weight
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = __ldg(reinterpret_cast<const float4*>(part + (long long)sh->at[min(i + k * GROUPS, here - 1)] * HD) + c);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = i + k * GROUPS < here ? sh->wt[i + k * GROUPS] : -1.f;
        if (w >= 0.f) {
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

// The same by one warp, 32 parts at a time, hd / 32 values a lane: for items of
// few parts, where a CTA's barriers cost more than its width saves. A part's
// place is found by one lane and passed on: found by all for each of them it is
// most of the time (64 x 16 rows of 5 parts: 5.2 us, 1.8 so).
template <typename T, int HD, typename Slot>
EE_DEV void join_row_warp(const float* part, const float* stat, long long n, Slot slot, T* out) {
  constexpr int V = HD / 32, UN = 8;
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.f, v[V] = {};
  for (long long i0 = 0; i0 < n; i0 += 32) {
    const int here = (int)(n - i0 < 32 ? n - i0 : 32);
    const int at = (int)slot(i0 + min(lane, here - 1));
    float x[UN][V];
    auto values = [&](int i) {
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const float* src = part + (long long)__shfl_sync(0xffffffffu, at, min(i + k, 31)) * HD + lane * V;  // past `here`: the last
        if (V == 4) {
          const float4 y = __ldg(reinterpret_cast<const float4*>(src));
          x[k][0] = y.x, x[k][1] = y.y, x[k][V - 2] = y.z, x[k][V - 1] = y.w;
        } else {
          const float2 y = __ldg(reinterpret_cast<const float2*>(src));
          x[k][0] = y.x, x[k][1] = y.y;
        }
      }
    };
    const float2 st = lane < here ? __ldg(reinterpret_cast<const float2*>(stat) + at) : make_float2(-INFINITY, 0.f);
    values(0);  // loads first: none waits for another's weight
    const float top = fmaxf(m, warp_max(st.x));
    const float u = top == -INFINITY ? 0.f : top, old = exp2f(m - u);
    m = top;
    const bool seen = st.y != 0.f;
    const float f = seen ? exp2f(st.x - u) : 0.f, wt = seen ? f : -1.f;
    l = l * old + f * st.y;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= old;
    for (int i = 0; i < here; i += UN) {
      if (i > 0) values(i);
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        const float w = __shfl_sync(0xffffffffu, wt, (i + k) & 31);  // below 0 past the last part
        if (w >= 0.f) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] += w * x[k][e];
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

}  // namespace ee
