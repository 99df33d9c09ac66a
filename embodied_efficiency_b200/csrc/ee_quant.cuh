// ee_quant.cuh -- rounding to integer codes, shared by the quantisers of tokens
// and of cached keys and values.
#pragma once

#include "ee_common.cuh"

namespace ee {

// nearest integers (ties to even) of the fp32 quotients v / s of four values,
// one byte each: t = v * (1 / s) is within 1.5 ulp of the quotient, so only a t
// that close to a tie is divided for. In packed pairs, as the instructions per
// value, not the bytes, bound a long row otherwise.
EE_DEV uint32_t quant_word(uint64_t v01, uint64_t v23, float s, uint64_t inv2) {
  const uint64_t magic = both(12582912.f), back = both(-12582912.f);  // 1.5 * 2^23: the sum's rounding is rint(t)
  const uint64_t t01 = mul2f(v01, inv2), t23 = mul2f(v23, inv2);
  uint64_t r01 = add2f(t01, magic), r23 = add2f(t23, magic);
  // rint(t) - t, exact and at most 1/2
  const uint64_t d01 = fma2f(t01, both(-1.f), add2f(r01, back)), d23 = fma2f(t23, both(-1.f), add2f(r23, back));
  uint32_t d[4], b[4];
  unpack64(d01, d[0], d[1]);
  unpack64(d23, d[2], d[3]);
  const float far = fmaxf(fmaxf(fabsf(__uint_as_float(d[0])), fabsf(__uint_as_float(d[1]))),
                          fmaxf(fabsf(__uint_as_float(d[2])), fabsf(__uint_as_float(d[3]))));
  unpack64(r01, b[0], b[1]);
  unpack64(r23, b[2], b[3]);
  if (far > 0.49993896484375f) {  // 1/2 - 2^-14
    uint32_t v[4];
    unpack64(v01, v[0], v[1]);
    unpack64(v23, v[2], v[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(__fdiv_rn(__uint_as_float(v[e]), s) + 12582912.f);
  }
  return prmt(prmt(b[0], b[1], 0x0040u), prmt(b[2], b[3], 0x0040u), 0x5410u);
}

}  // namespace ee
