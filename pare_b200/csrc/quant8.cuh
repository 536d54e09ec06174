// 16-bit floats -> int8 codes on a symmetric grid, shared by the paged cache's append and the W8A8 linear.
#pragma once

#include "common.cuh"

namespace pare {
namespace q8 {

// Largest magnitude of eight 16-bit floats as their bits, in both halves of a word: magnitudes order like their bits, infinities and NaN
// above all numbers.
__device__ __forceinline__ uint32_t magnitudes(const uint4& x) {
  return __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
}

struct Grid {
  float step, inv;
  bool finite, tiny;
  // step = amax / 127, the quotient
  __device__ __forceinline__ explicit Grid(float amax) {
    step = __fdiv_rn(amax, 127.f);
    finite = step < INFINITY;
    tiny = step < 1e-25f;               // 1 / step may overflow, x - q step underflow
    inv = finite && !tiny ? __fdiv_rn(1.f, step) : 0.f;
  }
  // round_half_even(x / step) in [-127, 127]; 0 on a grid that has no step or is not finite
  __device__ __forceinline__ int code(float x) const {
    if (!finite || step == 0.f) return 0;
    return (int)fminf(fmaxf(rintf(__fdiv_rn(x, step)), -127.f), 127.f);
  }
  // Eight of them.  The quotient by Markstein's theorem (IBM J. Res. Dev. 34, 1990): with inv the reciprocal rounded to nearest and q
  // within one unit in the last place of x / step, q + (x - q step) inv is the quotient rounded to nearest; the first correction
  // brings x * inv there.  Plus 1.5 * 2^23 it has the code in its low byte, rounded half to even.  No branch: x = amax / 2 and its kind
  // lie next to a border in most rows, and a division for the warps that see one took two thirds of the time (2048 rows of 4096, kernel
  // 11.4 us; two reciprocals that decide which).
  template <typename T>
  __device__ __forceinline__ uint2 codes(const uint4& w) const {
    constexpr float kMagic = 12582912.f;
    const T* v = reinterpret_cast<const T*>(&w);
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = to_float<T>(v[j]);
      float q = x * inv;
      q = fmaf(fmaf(-q, step, x), inv, q);
      q = fmaf(fmaf(-q, step, x), inv, q);
      r[j] = q + kMagic;
    }
    if (tiny || !finite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = (float)code(to_float<T>(v[j])) + kMagic;
    }
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __byte_perm(__float_as_uint(r[4 * j]), __float_as_uint(r[4 * j + 1]), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(r[4 * j + 2]), __float_as_uint(r[4 * j + 3]), 0x0040);
      o[j] = __byte_perm(lo, hi, 0x5410);
    }
    return make_uint2(o[0], o[1]);
  }
};

}  // namespace q8
}  // namespace pare
