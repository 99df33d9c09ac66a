// ee_prompt.cu -- C ABI: attention over packed prompts (causal or full,
// grouped heads, keys that may reach further back than the queries).
#include <atomic>

#include "ee_host.h"
#include "ee_prompt.cuh"
#include "ee_prompt_tc.cuh"

namespace ee {

// ---------------------------------------------------------------------------
// few query rows per key head
// ---------------------------------------------------------------------------
// A row is (token, head of the key head's group), so a key head's whole group
// shares one read of its keys. A CTA takes 16 rows of one sequence and key
// head and, where the units alone would not fill the GPU, one of `splits`
// parts of their keys. Its four warps each stream 16 keys of every 64 through
// a ring of their own (cp.async, no barrier between warps) with their own
// running maximum and sum; they are merged through shared memory at the end,
// and the parts through distributed shared memory when they are a cluster (up
// to 8), else by prompt_combine_kernel. HBM-bound on the keys and values: two
// or three CTAs share an SM, 128 KB of loads in flight.
constexpr int kPrWarps = 4, kPrKeys = 64;   // keys per step of the CTA
template <int HD> constexpr int pr_stages() { return HD == 128 ? 3 : 4; }
template <int HD> constexpr int pr_smem() { return pr_stages<HD>() * 2 * kPrKeys * HD * 2; }

EE_DEV void pr_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
EE_DEV void pr_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

template <typename T, int HD>
__global__ void __launch_bounds__(32 * kPrWarps) prompt_rows_kernel(const __grid_constant__ PromptArgs a) {
  constexpr int NW = kPrWarps, NT = 32 * NW, NS = pr_stages<HD>();
  constexpr int RB = HD * 2;             // bytes per key row
  constexpr int CH = HD / 8;             // 16-byte chunks per key row
  constexpr int TILE = 16 * RB;          // a warp's 16 keys
  extern __shared__ __align__(128) char smem[];
  __shared__ PromptFind<NT> sh;
  pdl_entry();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, part = blockIdx.x % a.splits;
  PromptSeq s;
  if (!prompt_find<NT>(a, blockIdx.x / a.splits, a.group, 16, &sh, s)) return;  // the same for a whole cluster
  const int rows = s.qlen * a.group, r0 = s.blk * 16;
  // keys this CTA's rows see at most, and its part of them in steps of 64
  const int last_tok = (min(r0 + 16, rows) - 1) / a.group;
  const int kend = a.causal ? max(min(s.klen, s.klen - s.qlen + last_tok + 1), 0) : s.klen;
  const int nst = (kend + kPrKeys - 1) / kPrKeys;
  const int st0 = (int)((long long)nst * part / a.splits), st1 = (int)((long long)nst * (part + 1) / a.splits);
  const uint32_t ring = smem_u32(smem) + warp * NS * 2 * TILE;
  auto off = [](int row, int ch) { return row * RB + ((ch ^ (row & 7)) << 4); };
  // keys 64 st + 16 warp ..: K, then V; those past the last seen one are zero-filled
  const char* kp = reinterpret_cast<const char*>(a.k) + ((long long)(s.k0 + 16 * warp) * a.k_tok + kvh * a.k_head) * 2;
  const char* vp = reinterpret_cast<const char*>(a.v) + ((long long)(s.k0 + 16 * warp) * a.v_tok + kvh * a.v_head) * 2;
  const int lrow = lane / CH, lch = lane % CH;  // this lane's row and chunk of every 32 / CH rows
  auto load = [&](int st, int buf) {
    const long long k0 = (long long)st * kPrKeys;
    const int valid = kend - (int)k0 - 16 * warp;
    const uint32_t d = ring + buf * 2 * TILE;
#pragma unroll
    for (int i = 0; i < 16 * CH / 32; ++i) {
      const int row = lrow + i * (32 / CH);
      const bool ok = row < valid;
      cp_async16(d + off(row, lch), kp + (ok ? (k0 + row) * a.k_tok * 2 + lch * 16 : 0), ok);
      cp_async16(d + TILE + off(row, lch), vp + (ok ? (k0 + row) * a.v_tok * 2 + lch * 16 : 0), ok);
    }
  };
  // an address to hand to a load that reads nothing
  if (s.k0 + 16 * warp >= a.tk) kp = reinterpret_cast<const char*>(a.k), vp = reinterpret_cast<const char*>(a.v);
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    if (st0 + i < st1) load(st0 + i, i);
    cp_async_commit();
  }
  // the query fragments
  const int ra = r0 + g, rb = ra + 8;
  uint32_t qf[HD / 16][4];
  {
    auto qrow = [&](int r) {
      const int tok = r / a.group, h = kvh * a.group + r % a.group;
      return reinterpret_cast<const char*>(a.q) + ((long long)(s.q0 + tok) * a.q_tok + h * a.q_head) * 2;
    };
    const char *pa = qrow(min(ra, rows - 1)), *pb = qrow(min(rb, rows - 1));
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      qf[ks][0] = *reinterpret_cast<const uint32_t*>(pa + ks * 32 + t * 4);
      qf[ks][1] = *reinterpret_cast<const uint32_t*>(pb + ks * 32 + t * 4);
      qf[ks][2] = *reinterpret_cast<const uint32_t*>(pa + ks * 32 + 16 + t * 4);
      qf[ks][3] = *reinterpret_cast<const uint32_t*>(pb + ks * 32 + 16 + t * 4);
    }
  }
  // keys below lim are seen by rows ra and rb
  const int lim0 = a.causal ? min(s.klen, s.klen - s.qlen + ra / a.group + 1) : s.klen;
  const int lim1 = a.causal ? min(s.klen, s.klen - s.qlen + rb / a.group + 1) : s.klen;
  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const int mi = lane >> 3;
  int buf = 0;
  for (int st = st0; st < st1; ++st) {
    if (st + NS - 1 < st1) load(st + NS - 1, buf == 0 ? NS - 1 : buf - 1);
    cp_async_commit();
    cp_async_wait<NS - 1>();
    __syncwarp();
    const uint32_t kt = ring + buf * 2 * TILE, vt = kt + TILE;
    const int key = st * kPrKeys + 16 * warp;  // first of the warp's 16 keys
    if (key < kend) {
      float p[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t b[4];
        pr_ldsm(kt + off((mi >> 1) * 8 + (lane & 7), 2 * ks + (mi & 1)), b);
        mma16816<T>(p[0], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[0], b[1]);
        mma16816<T>(p[1], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], b[2], b[3]);
      }
      float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int kk = key + 8 * j + 2 * t + c;
          p[j][c] = kk < lim0 ? p[j][c] * a.scale_log2 : -INFINITY;
          p[j][2 + c] = kk < lim1 ? p[j][2 + c] * a.scale_log2 : -INFINITY;
          x0 = fmaxf(x0, p[j][c]);
          x1 = fmaxf(x1, p[j][2 + c]);
        }
      }
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
      }
      const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
      // nothing seen yet: any finite reference will do, exp2(-inf) = 0
      const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
      if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
        const float c0 = exp2f(m0 - u0), c1 = exp2f(m1 - u1);
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
          p[j][c] = exp2f(p[j][c] - u0);
          p[j][2 + c] = exp2f(p[j][2 + c] - u1);
          l0 += p[j][c];
          l1 += p[j][2 + c];
        }
      }
      const uint32_t pa0 = Act<T>::pack2(p[0][0], p[0][1]), pa1 = Act<T>::pack2(p[0][2], p[0][3]);
      const uint32_t pa2 = Act<T>::pack2(p[1][0], p[1][1]), pa3 = Act<T>::pack2(p[1][2], p[1][3]);
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) {
        uint32_t b[4];
        pr_ldsm_t(vt + off((mi & 1) * 8 + (lane & 7), 2 * d + (mi >> 1)), b);
        mma16816<T>(o[2 * d], pa0, pa1, pa2, pa3, b[0], b[1]);
        mma16816<T>(o[2 * d + 1], pa0, pa1, pa2, pa3, b[2], b[3]);
      }
    }
    __syncwarp();  // every lane has read the stage before it is loaded again
    if (++buf == NS) buf = 0;
  }
  cp_async_wait<0>();
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }
  // merge the warps: [warp][16 rows][HD + 4] fp32 over the rings; this CTA's sums behind them
  constexpr int ML = HD + 4;
  static_assert((NW + 1) * 16 * ML * 4 <= pr_smem<HD>(), "the merge fits the rings");
  float* mg = reinterpret_cast<float*>(smem) + warp * 16 * ML;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) {
    *reinterpret_cast<float2*>(mg + g * ML + 8 * i + 2 * t) = make_float2(o[i][0], o[i][1]);
    *reinterpret_cast<float2*>(mg + (g + 8) * ML + 8 * i + 2 * t) = make_float2(o[i][2], o[i][3]);
  }
  if (t == 0) {
    *reinterpret_cast<float2*>(mg + g * ML + HD) = make_float2(m0, l0);
    *reinterpret_cast<float2*>(mg + (g + 8) * ML + HD) = make_float2(m1, l1);
  }
  __syncthreads();
  // n partial sums of row r's values c .. c + 3, `at(i)` giving (maximum, weight) and the values
  auto merge = [&](int n, auto stat, auto vals, float& m, float& l) {
    m = -INFINITY;
    for (int w = 0; w < n; ++w) m = fmaxf(m, stat(w).x);
    const float u = m == -INFINITY ? 0.f : m;
    l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < n; ++w) {
      const float2 st = stat(w);
      const float f = exp2f(st.x - u);
      const float4 v = vals(w);
      l += f * st.y;
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    return acc;
  };
  auto write = [&](int r, int c, float4 acc, float l) {
    const int tok = s.q0 + (r0 + r) / a.group, h = kvh * a.group + (r0 + r) % a.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key is zero
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (long long)tok * a.o_tok + h * a.o_head + c) =
        make_uint2(Act<T>::pack2(acc.x * inv, acc.y * inv), Act<T>::pack2(acc.z * inv, acc.w * inv));
  };
  const int live = min(16, rows - r0) * (HD / 4);
  float* own = reinterpret_cast<float*>(smem) + NW * 16 * ML;
  for (int i = tid; i < live; i += NT) {  // 4 values of a row over the warps
    const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
    const float* base = reinterpret_cast<const float*>(smem) + r * ML;
    float m, l;
    const float4 acc = merge(
        NW, [&](int w) { return *reinterpret_cast<const float2*>(base + w * 16 * ML + HD); },
        [&](int w) { return *reinterpret_cast<const float4*>(base + w * 16 * ML + c); }, m, l);
    if (a.splits == 1) {
      write(r, c, acc, l);
    } else if (a.clustered) {
      *reinterpret_cast<float4*>(own + r * ML + c) = acc;
      if (c == 0) *reinterpret_cast<float2*>(own + r * ML + HD) = make_float2(m, l);
    } else {  // this part's sums, relative to its maximum
      const int tok = s.q0 + (r0 + r) / a.group, h = kvh * a.group + (r0 + r) % a.group;
      const long long at = ((long long)part * a.tq + tok) * a.n_q + h;
      if (c == 0) *reinterpret_cast<float2*>(a.stat + 2 * at) = make_float2(m, l);
      if (l != 0.f) *reinterpret_cast<float4*>(a.part + at * HD + c) = acc;
    }
  }
  if (a.splits > 1 && a.clustered) {
    cluster_sync();
    const uint32_t base = smem_u32(own);
    for (int i = tid + part * NT; i < live; i += NT * a.splits) {
      const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
      float m, l;
      const float4 acc = merge(
          a.splits,
          [&](int w) {
            const uint32_t at = mapa(base + (r * ML + HD) * 4, w);
            return make_float2(ld_dsmem_f32(at), ld_dsmem_f32(at + 4));
          },
          [&](int w) { return ld_dsmem_f4(mapa(base + (r * ML + c) * 4, w)); }, m, l);
      write(r, c, acc, l);
    }
    cluster_sync();  // the sums stay until the whole cluster has read them
  }
}

// Joins the parts of every (token, head), one CTA each: first a thread per
// part for the common maximum and the parts' weights, then hd / 4 threads
// across the values and the rest across the parts, so that both passes have
// their loads in flight together.
constexpr int kPrCombine = 256, kPrMaxSplits = 512;
template <typename T, int HD>
__global__ void __launch_bounds__(kPrCombine) prompt_combine_kernel(const __grid_constant__ PromptArgs a) {
  constexpr int LANES = HD / 4, GROUPS = kPrCombine / LANES;
  __shared__ float wt[kPrMaxSplits];
  __shared__ float4 sv[GROUPS][LANES];
  __shared__ float red[2][kPrCombine / 32];
  pdl_entry();
  const int tok = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // rows outside the sequences have no parts and stay as they were
  if (tok < __ldg(a.cu_q) || tok >= __ldg(a.cu_q + a.n_seq)) return;
  const long long step = (long long)a.tq * a.n_q, at = (long long)tok * a.n_q + h;
  float2 st[kPrMaxSplits / kPrCombine];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPrMaxSplits / kPrCombine; ++i) {
    const int sp = threadIdx.x + i * kPrCombine;
    st[i] = sp < a.splits ? __ldg(reinterpret_cast<const float2*>(a.stat) + at + sp * step) : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, st[i].x);
  }
  m = warp_max(m);
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPrCombine / 32; ++i) m = fmaxf(m, red[0][i]);
  const float u = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < kPrMaxSplits / kPrCombine; ++i) {
    const float f = st[i].y == 0.f ? 0.f : exp2f(st[i].x - u);  // weight 0: no key seen, its sums were not written
    wt[threadIdx.x + i * kPrCombine] = f;
    l += f * st[i].y;
  }
  l = warp_sum(l);
  if (lane == 0) red[1][warp] = l;
  __syncthreads();
  const int c = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = grp; i < a.splits; i += GROUPS) {
    const float f = wt[i];
    if (f != 0.f) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(a.part + (at + i * step) * HD) + c);
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
  }
  sv[grp][c] = acc;
  __syncthreads();
  if (grp) return;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kPrCombine / 32; ++i) l += red[1][i];
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) {
    const float4 v = sv[g][c];
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (long long)tok * a.o_tok + h * a.o_head + 4 * c) =
      make_uint2(Act<T>::pack2(acc.x * inv, acc.y * inv), Act<T>::pack2(acc.z * inv, acc.w * inv));
}

// How a call runs, by what the host knows of it: rows (queries x group) per
// sequence and key head, and keys per sequence, on average.
//   tc      more than 16 rows: the tensor-core kernel's 128-row tiles (8 x 50
//           new tokens behind 816, 16 heads of 128: 27 us, 68 with 64-row warp
//           MMA units), 16 or fewer: the rows kernel's single MMA row tile
//   splits  parts of the keys, joined by a second launch. Rows kernel: enough
//           CTAs for four an SM, of 128 keys or more each (two or eight an SM
//           measured within 10 % or slower: 8 x 4096 keys, 32 / 8 heads of 128:
//           53 / 47 / 49 us for 2 / 4 / 8). Tensor-core kernel: where the items
//           would leave SMs idle, parts of 512 keys or more.
#ifndef EE_PR_PER_SM
#define EE_PR_PER_SM 4
#endif
#ifndef EE_PR_CLUSTER
#define EE_PR_CLUSTER 8
#endif
constexpr long long kPrRows = 16, kPrCtasPerSm = EE_PR_PER_SM, kPrMinKeys = 128, kPtMinKeys = 512;
struct PromptPlan { bool tc; int splits; bool clustered; };
static PromptPlan prompt_plan(long long tq, long long tk, int n_seq, int n_q, int n_kv) {
  PromptPlan pl{false, 1, false};
  if (n_seq < 1) return pl;
  const int group = n_q / n_kv;
  const long long rows = tq * group;
  pl.tc = rows > kPrRows * n_seq && tk > 0 && group <= 128;
  // rows of a unit: two tiles of whole tokens, or one MMA tile
  const long long per = pl.tc ? 2 * (128 / group) * group : kPrRows;
  const long long units = (rows / per > n_seq ? rows / per : n_seq) * n_kv;
  const long long want = pl.tc ? device_sms() / units : (kPrCtasPerSm * device_sms() + units - 1) / units;
  const long long most = pl.tc ? tk / n_seq / kPtMinKeys : (tk / n_seq + kPrMinKeys - 1) / kPrMinKeys;
  const long long s = want < most ? want : most;
  pl.splits = s < 1 ? 1 : (int)(s < kPrMaxSplits ? s : kPrMaxSplits);
  pl.clustered = !pl.tc && pl.splits > 1 && pl.splits <= EE_PR_CLUSTER;
  return pl;
}
static size_t prompt_ws_bytes(const PromptPlan& pl, long long tq, int n_q, int hd) {
  return pl.splits > 1 && !pl.clustered ? (size_t)pl.splits * tq * n_q * (hd + 2) * 4 : 0;
}

template <typename T, int HD>
static int launch_combine(const PromptArgs& a, cudaStream_t s) {
  if (a.splits == 1 || a.clustered) return EE_OK;
  return launch_pdl(prompt_combine_kernel<T, HD>, dim3((unsigned)a.tq, a.n_q), dim3(kPrCombine), 0, s, a) == cudaSuccess
             ? EE_OK
             : EE_ERR_LAUNCH;
}

template <typename T, int HD>
static int launch_rows(const PromptArgs& a, cudaStream_t s) {
  auto fn = prompt_rows_kernel<T, HD>;
  static std::atomic<int> set[64];
  allow_max_smem(fn, set);
  // at most one partial block per sequence beyond the rows' whole blocks
  const long long units = (long long)a.tq * a.group / 16 + a.n_seq;
  if (units * a.splits > 0x7fffffff) return EE_ERR_SHAPE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * a.splits), a.n_kv);
  cfg.blockDim = dim3(32 * kPrWarps);
  cfg.dynamicSmemBytes = pr_smem<HD>();
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  unsigned int n = 0;
  add_pdl_attr(attr, n);
  if (a.clustered) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, fn, a) != cudaSuccess) return EE_ERR_LAUNCH;
  return launch_combine<T, HD>(a, s);
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
  a.timeout_ns = 1000000000ull;
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

int ee_prompt_attention(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok, int64_t k_head,
                        const void* v, int64_t v_tok, int64_t v_head, void* out, int64_t o_tok, int64_t o_head,
                        const int32_t* cu_q, const int32_t* cu_k, const int32_t* k_lens, int64_t tq, int64_t tk,
                        int32_t n_seq, int32_t n_q, int32_t n_kv, int32_t head_dim, int32_t causal, float scale,
                        int32_t act_dtype, void* workspace, size_t workspace_bytes, ee_stream_t stream) {
  if (act_dtype != EE_BF16 && act_dtype != EE_F16) return EE_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return EE_ERR_UNSUPPORTED;
  if (tq < 0 || tk < 0 || n_seq < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0) return EE_ERR_SHAPE;
  if (tq > 0x7fffff00 || tk > 0x7fffff00 || n_kv > 65535 || n_q > 65535) return EE_ERR_SHAPE;
  if (!(scale > 0.f) || scale > 3.0e38f) return EE_ERR_ARG;
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
  a.scale_log2 = scale * 1.4426950408889634f;
  a.splits = pl.splits;
  a.clustered = pl.clustered;
  a.part = reinterpret_cast<float*>(workspace);
  a.stat = a.part + (size_t)pl.splits * tq * n_q * head_dim;
  cudaStream_t s = (cudaStream_t)stream;
  return act_dtype == EE_BF16 ? launch_prompt<__nv_bfloat16>(a, pl, head_dim, s)
                               : launch_prompt<__half>(a, pl, head_dim, s);
}

}  // extern "C"
