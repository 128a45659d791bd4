// The 8-bit convention that the norm, the row quantiser, the int8 products and the packed
// activations share: a run of values (a row, or a group of columns of a row) is held as
//   q = round(v * 127 / a) in -127..127,  scale = a / 127,  a = max(largest |v|, 2^-100)
// rounded to the nearest, ties to even, as if the quotient were exact. A run that holds NaN or
// infinity has scale NaN and q = 0, so that everything computed from it reads NaN instead of a
// finite wrong value. The floor 2^-100 keeps 127 / a finite for runs that are (almost) zero.
#pragma once

#include "common.cuh"

namespace fmoe {

#ifdef __CUDACC__

constexpr uint32_t kInfBits = 0x7f800000u;

// Largest magnitude of a run as the bit pattern of |v|: unsigned order is the order of the
// magnitudes, with infinity and NaN above every finite value, so a maximum never loses a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Quantiser {
  float top;    // a
  float inv;    // 127 / a
  float scale;  // a / 127, or NaN
  bool fine;
  __device__ explicit Quantiser(uint32_t top_bits) {
    fine = top_bits < kInfBits;
    top = fine ? fmaxf(__uint_as_float(top_bits), 0x1p-100f) : 1.f;
    inv = __fdiv_rn(127.f, top);
    scale = fine ? __fdiv_rn(top, 127.f) : __uint_as_float(0x7fc00000u);
  }
  // v * (127 / a) in fp32 is off by at most 127 * 2 * 2^-24 = 1.6e-5: only a quotient that close
  // to the border between two whole numbers is taken again in 64 bits (6 in 100000 values).
  __device__ __forceinline__ int operator()(float v) const {
    const float t = v * inv;
    float r = rintf(t);
    if (fabsf(t - r) > 0.5f - 3e-5f) r = static_cast<float>(rint(static_cast<double>(v) * 127.0 / static_cast<double>(top)));
    return fine ? static_cast<int>(r) : 0;
  }
};

__device__ __forceinline__ uint32_t pack_int8(int a, int b, int c, int d) {
  return (a & 255) | ((b & 255) << 8) | ((c & 255) << 16) | (static_cast<uint32_t>(d) << 24);
}

// Four int8 in a word as floats.
__device__ __forceinline__ void unpack_int8(uint32_t w, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
}

#endif  // __CUDACC__

}  // namespace fmoe
