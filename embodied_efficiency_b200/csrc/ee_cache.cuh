// ee_cache.cuh -- the paged cache of quantised keys and values: where a token
// of a sequence lies.
//
// A page holds `page` consecutive tokens of one sequence: for every key head
// page rows of head_dim codes (8 bits, or two 4-bit codes a byte, the even one
// in the low half), and beside them an fp32 step per row. Key i of sequence b
// is row i % page of page table[b][i / page]. Lengths, offsets and the table
// live on the device: whatever they say, nothing outside the cache and the
// packed tensors is read or written. A place that the table does not have, or
// whose page number the cache does not have, holds no key.
#pragma once

#include <type_traits>

#include "ee_common.cuh"

namespace ee {

struct CacheView {
  const int* table;
  const int* k_lens;
  long long table_row;  // entries between the rows of the table
  int n_seq, width;     // sequences; pages a row of the table names
  int pages, n_kv, shift;  // of the cache; a page is 2^shift tokens
};

// Row of the flattened cache [pages][n_kv][page] for head 0 of a place (head h: h << shift further), -1 for none.
EE_DEV long long cache_row(const CacheView& c, int page, int at) {
  if ((unsigned)page >= (unsigned)c.pages) return -1;
  return ((long long)page * c.n_kv << c.shift) + at;
}

// The sequence of packed row `t`, by a whole warp: the last b with cu[b] <= t, 32 offsets looked at in each round.
EE_DEV int cache_seq(const int* cu, int n_seq, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seq;  // cu[lo] <= t (or lo = 0), the answer is among lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, i < lo + n && (lane == 0 || __ldg(cu + i) <= t));
    const int hit = 31 - __clz(below), end = lo + n;
    lo += hit * step;
    n = min(step, end - lo);
  }
  return lo;
}

// Where packed row t of sequence b lies: it is one of the last tokens before k_lens[b].
EE_DEV long long cache_place(const CacheView& c, const int* cu, int b, int t) {
  const int first = __ldg(cu + b), end = __ldg(cu + b + 1);
  if (t < first || t >= end) return -1;
  const long long key = (long long)__ldg(c.k_lens + b) - ((long long)end - t);
  if (key < 0 || (key >> c.shift) >= c.width) return -1;
  return cache_row(c, __ldg(c.table + b * c.table_row + (key >> c.shift)), (int)(key & ((1 << c.shift) - 1)));
}

// Two signed 4-bit codes of a word, byte `p`, or two 8-bit ones of bytes 2p and
// 2p + 1, as 16-bit values: exact, for 8 bits in bf16 a 64th of it (bf16's
// numbers below 2^-126 take a byte as it is, times 2^-133; one multiplication by
// 2^127 and the sum take it to where it belongs, where an exponent OR-ed above
// it has seven bits only and takes three instructions).
template <typename T> EE_DEV uint32_t code_pair8(uint32_t flipped, int p);  // of a word with its sign bits flipped
template <> EE_DEV uint32_t code_pair8<__half>(uint32_t w, int p) {
  return fma2<__half>(prmt(w, 0x64u, p ? 0x4342u : 0x4140u), 0x3C003C00u, 0xE480E480u);
}
template <> EE_DEV uint32_t code_pair8<__nv_bfloat16>(uint32_t w, int p) {
  return fma2<__nv_bfloat16>(prmt(w, 0u, p ? 0x4342u : 0x4140u), 0x7F007F00u, 0xC000C000u);
}
template <typename T> EE_DEV uint32_t code_pair4(uint32_t w, uint32_t w_shr4, int p) {
  return fma2<T>(nib_pair<T>(w, w_shr4, p, 0x00080008u), Act<T>::kOne2, std::is_same<T, __half>::value ? 0xE408E408u : 0xC308C308u);
}
// what code_pair8 leaves out
template <typename T, int BITS> EE_DEV constexpr float code_unit() { return BITS == 8 && !std::is_same<T, __half>::value ? 64.f : 1.f; }

}  // namespace ee
