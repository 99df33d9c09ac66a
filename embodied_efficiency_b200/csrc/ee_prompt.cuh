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

#include <type_traits>

#include "ee_common.cuh"

namespace ee {

// What a row's weights 2^(x - reference) are taken relative to, given its
// largest scaled score x. Weights are rounded to 16 bits for their product with
// v, and fp16 ends at 2^-24: beside a largest weight of 1, keys 17 nats below
// it would be lost however many they are. So for fp16 the reference lies BITS
// below x and the weights are that much larger; their sum is too, and the
// division drops the factor. (Not from 2^20 on, where fp32 no longer takes
// BITS off exactly enough; bf16 has fp32's range.)
template <typename T, int BITS>
EE_DEV float prompt_reference(float x) {
  if (!std::is_same<T, __half>::value) return x;
  return fabsf(x) < 1048576.f ? x - (float)BITS : x;
}

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  const int *cu_q, *cu_k, *k_lens;
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // strides, elements
  int tq, tk, n_seq, n_q, n_kv, group, causal;
  float scale_log2;  // scale * log2(e)
  int splits;        // tensor-core kernel: parts of the keys
  float* part;       // sums of partial rows and, in stat, their maximum and weight: [splits][tq][n_q][hd], or by
  float* stat;       // worker ([workers][2][16][hd]) in the kernel for few rows
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

}  // namespace ee
