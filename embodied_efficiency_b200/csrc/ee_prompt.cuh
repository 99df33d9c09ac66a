// ee_prompt.cuh -- what the kernels of packed-prompt attention share: the
// call's arguments and the search for the sequence of a unit of query rows.
//
// Sequence b's queries are rows cu_q[b] .. cu_q[b + 1] of q, its keys
// klen(b) rows of k / v from cu_k[b] on; its last query sees its last key, so
// with the causal mask query i sees keys 0 .. klen - qlen + i. Lengths live
// on the device, so a grid is sized by what the host knows (total rows and
// the number of sequences) and every CTA finds its own sequence. Offsets that
// the call's totals do not cover are cut to them: no table can make a kernel
// read or write outside the tensors.
#pragma once

#include "ee_common.cuh"

namespace ee {

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  const int *cu_q, *cu_k, *k_lens;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // strides, elements
  int tq, tk, n_seq, n_q, n_kv, group, causal;
  float scale_log2;  // scale * log2(e)
  int splits;        // parts of the keys
  int clustered;     // the parts are a cluster's CTAs, joined there; else through part and stat
  float* part;       // [splits][tq][n_q][hd] sums of a part and [splits][tq][n_q][2] their maximum and weight
  float* stat;
};

struct PromptSeq {
  int q0, qlen, k0, klen, blk;  // first row and length in q and in k / v; block of the sequence
};

EE_DEV PromptSeq prompt_seq(const PromptArgs& a, int b) {
  PromptSeq s;
  s.q0 = min(max(__ldg(a.cu_q + b), 0), a.tq);
  s.qlen = min(max(__ldg(a.cu_q + b + 1), s.q0), a.tq) - s.q0;
  s.k0 = min(max(__ldg(a.cu_k + b), 0), a.tk);
  int end = __ldg(a.cu_k + b + 1);
  if (a.k_lens) end = min(end, s.k0 + min(max(__ldg(a.k_lens + b), 0), a.tk - s.k0));
  s.klen = min(max(end, s.k0), a.tk) - s.k0;
  s.blk = 0;
  return s;
}

// The sequence and block of unit `u`, the sequences' query rows (times `mul`)
// being cut into blocks of `rows`; false when there is no such unit. All
// THREADS threads of the CTA call it, each with a sequence of its own whose
// whole record it reads at once, so a call of up to THREADS sequences waits
// for global memory once.
template <int THREADS>
struct PromptFind {
  int sums[THREADS / 32], hit;
  PromptSeq seq;
};
template <int THREADS>
EE_DEV bool prompt_find(const PromptArgs& a, int u, int mul, int rows, PromptFind<THREADS>* sh, PromptSeq& out) {
  constexpr int NW = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int before = 0;
  for (int b0 = 0; b0 < a.n_seq; b0 += THREADS) {
    PromptSeq s{};
    if (b0 + tid < a.n_seq) s = prompt_seq(a, b0 + tid);
    const int nb = (int)(((long long)s.qlen * mul + rows - 1) / rows);
    int inc = nb;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (tid == 0) sh->hit = 0;
    if (lane == 31) sh->sums[warp] = inc;
    __syncthreads();
    int base = before, total = before;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) base += sh->sums[w];
      total += sh->sums[w];
    }
    if (u >= base + inc - nb && u < base + inc) {
      s.blk = u - (base + inc - nb);
      sh->seq = s;
      sh->hit = 1;
    }
    __syncthreads();
    if (sh->hit) {
      out = sh->seq;
      return true;
    }
    before = total;
  }
  return false;
}

}  // namespace ee
