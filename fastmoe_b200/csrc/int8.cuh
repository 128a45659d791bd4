// The 8-bit convention that the norm, the row quantiser, the int8 products and the packed
// activations share: a run of values (a row, or a group of columns of a row) is held as
//   q = round(v * 127 / a) in -127..127,  scale = a / 127,  a = max(largest |v|, 2^-100)
// rounded to the nearest, ties to even, as if the quotient were exact. A run that holds NaN or
// infinity has scale NaN and q = 0, so that everything computed from it reads NaN instead of a
// finite wrong value. The floor 2^-100 keeps 127 / a finite for runs that are (almost) zero.
#pragma once

#include "common.cuh"

namespace fmoe {

// Quotients by a run-time constant, as a multiplication: n / d = n * (2^s / d + 1) / 2^s for n < 2^31,
// with s = 31 + ceil(log2 d) (the excess of the factor, below 2^-s each, adds less than 1 / d).
struct FastDiv {
  uint32_t mul = 0, shift = 0;
  int d = 1;
  explicit FastDiv(int64_t divisor) : d(static_cast<int>(divisor)) {
    uint32_t log = 0;
    while ((1ll << log) < divisor) ++log;
    shift = 31 + log;
    mul = static_cast<uint32_t>((1ull << shift) / static_cast<uint64_t>(divisor) + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
};

#ifdef __CUDACC__

constexpr uint32_t kInfBits = 0x7f800000u;

// Largest magnitude of a run as the bit pattern of |v|: unsigned order is the order of the
// magnitudes, with infinity and NaN above every finite value, so a maximum never loses a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Larger of `top` and |v|, NaN if either is.
__device__ __forceinline__ float max_abs(float top, float v) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(top), "f"(fabsf(v)));
  return m;
}

// Adding this to |t| < 2^22 rounds t to a whole number (nearest, ties to even) and leaves that number's
// two's complement in the low bits of the sum. Conversion instructions run at an eighth of the rate of
// an addition, too few for the values that HBM delivers.
constexpr float kRounder = 12582912.f;  // 1.5 * 2^23
constexpr float kNear = 0.5f - 5e-5f;

// The fast exponential and quotient are off by (2 + |x|) and 2 steps of 2^-23 (below x = -87.3, where the
// result is less than 2^-126, it is zero). The exact quotient's
// slow path is a branch per value, which keeps a lane's values from overlapping: with it the SwiGLU
// epilogue of one 128 x 256 tile took 24 us.
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// The normal distribution's cdf, 0.5 (1 + erf(x / sqrt 2)), by Abramowitz and Stegun 7.1.26 (absolute
// error of erf 1.5e-7 and of its complement alike), without branches, for the same reason. x times it is off
// by 2e-7 or less for negative x (the erff form, 0.5 x (1 + erf(x / sqrt 2)): 8e-8) and by 4e-7 for positive x (4e-7);
// relative to itself by 7e-7 for x > -1 (2e-7), 5e-5 at -3 (1e-5), 1.6e-3 at -5 (5e-2) and 4e-3 at -6, where
// the erff form has no bit left. `bell` receives exp(-x^2 / 2), which the density needs too.
__device__ __forceinline__ float normal_cdf(float x, float* bell) {
  const float z = fabsf(x) * 0.70710678f;
  const float t = __fdividef(1.f, fmaf(0.3275911f, z, 1.f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  *bell = __expf(-z * z);
  const float tail = 0.5f * p * *bell;
  return x < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gelu(float x) {
  float bell;
  return x * normal_cdf(x, &bell);
}

// Two fp32 operations in one instruction (sm_100's packed fp32 forms; the rounding is that of each).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

struct Quantiser {
  float top;    // a
  float inv;    // 127 / a, off by two steps of 2^-23 or less
  bool fine;
  __device__ explicit Quantiser(uint32_t top_bits) {
    fine = top_bits < kInfBits;
    top = fine ? fmaxf(__uint_as_float(top_bits), 0x1p-100f) : 1.f;
    inv = __fdividef(127.f * 0x1p-8f, top * 0x1p-8f);  // scaled: the fast quotient gives up above 2^126
  }
  // a / 127, or NaN: rounded as a quotient, for the one thread that stores it
  __device__ __forceinline__ float scale() const { return fine ? __fdiv_rn(top, 127.f) : __uint_as_float(0x7fc00000u); }
  // v * inv is off by at most 127 * 2 * 2^-23 = 3.1e-5. A quotient that lies that close to the border
  // between two whole numbers is compared with the border exactly. (One in 10000 of arbitrary values
  // does; among 16-bit values one that is exactly a / 2, at 63.5, is common.)
  __device__ __forceinline__ void settle(float v, float& s) const {
    const float r = s - kRounder, d = fmaf(v, inv, -r);
    if (fabsf(d) > kNear) {
      // The border next to r on d's side is m / 2 with m = 2 r +- 1; the side of v is the sign of
      // 254 v - m a, both taken times 2^-8 against overflow. m a = h + low exactly; 254 v - h and the
      // difference that is left have 18 bits or fewer in units of v's last one: exact too.
      const float sign = copysignf(1.f, d);
      const float m = fmaf(2.f, r, sign) * 0x1p-8f;
      const float h = m * top, low = fmaf(m, top, -h);
      const float side = (fmaf(v, 254.f / 256.f, -h) - low) * sign;
      if (side > 0.f || (side == 0.f && (__float_as_uint(s) & 1u))) s += sign;
    }
  }
  // Values that come straight from a 16-bit type. With significands of 11 bits or fewer, a = b 2^x and
  // v = c 2^y, a quotient that is not on a border is |254 c - odd b 2^s| / (2 b 2^s) >= |t| / (254 * 2047)
  // = 1.9e-6 |t| away from it: more than a factor that is too large by 2.4e-7 to 7.2e-7 moves it. That leaves the
  // exact ties, 254 c = odd b 2^s: either v = a / 2, where 63.5 belongs to 64 and the excess takes it
  // there, or b is a multiple of 127, which one largest magnitude in 128 is: only then each value is
  // looked at as any fp32 value is.
  template <int N>
  __device__ __forceinline__ void from16(const float* v, uint32_t* words) const {
    const uint32_t significand = (__float_as_uint(top) & 0x7fffffu) | 0x800000u;
    if (!fine || significand % 127u == 0u) return this->template operator()<N>(v, words);
    const float more = inv * (1.f + 0x1p-21f);
    float s[N];
    if constexpr (N == 1) {
      s[0] = fmaf(v[0], more, kRounder);
      words[0] = __float_as_uint(s[0]) & 255u;
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const float2 t = fma2(make_float2(v[j], v[j + 1]), make_float2(more, more), make_float2(kRounder, kRounder));
        s[j] = t.x;
        s[j + 1] = t.y;
      }
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const uint32_t lo = __byte_perm(__float_as_uint(s[j]), __float_as_uint(s[j + 1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(s[j + 2]), __float_as_uint(s[j + 3]), 0x0040);
        words[j / 4] = __byte_perm(lo, hi, 0x5410);
      }
    }
  }
  // N values: words[i] holds q of v[4 i .. 4 i + 3] (N = 1: of v[0], in the low byte). The budget is
  // tight: three bytes of DRAM traffic per 16-bit value leave eight instructions for it, so the
  // arithmetic goes in pairs.
  template <int N>
  __device__ __forceinline__ void operator()(const float* v, uint32_t* words) const {
    float s[N];
    if constexpr (N == 1) {
      s[0] = fmaf(v[0], inv, kRounder);
      settle(v[0], s[0]);
    } else {
      const float2 inv2 = make_float2(inv, inv), up = make_float2(kRounder, kRounder), minus = make_float2(-1.f, -1.f);
      constexpr int kPart = N > 8 ? 4 : N;  // values that are looked at together
      float off[N / kPart];                 // their largest distance between a quotient and the whole number it went to
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const float2 x = make_float2(v[j], v[j + 1]);
        const float2 t = fma2(x, inv2, up);
        const float2 d = fma2(x, inv2, fma2(t, minus, up));
        s[j] = t.x;
        s[j + 1] = t.y;
        const float most = fmaxf(fabsf(d.x), fabsf(d.y));
        off[j / kPart] = j % kPart == 0 ? most : fmaxf(off[j / kPart], most);
      }
      float most = off[0];
#pragma unroll
      for (int j = kPart; j < N; j += kPart) most = fmaxf(most, off[j / kPart]);
      if (most > kNear) {
#pragma unroll
        for (int j = 0; j < N; j += kPart) {
          if (kPart == N || off[j / kPart] > kNear) {
#pragma unroll
            for (int i = 0; i < kPart; ++i) settle(v[j + i], s[j + i]);
          }
        }
      }
    }
    if constexpr (N == 1) {
      words[0] = fine ? __float_as_uint(s[0]) & 255u : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const uint32_t lo = __byte_perm(__float_as_uint(s[j]), __float_as_uint(s[j + 1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(s[j + 2]), __float_as_uint(s[j + 3]), 0x0040);
        words[j / 4] = fine ? __byte_perm(lo, hi, 0x5410) : 0u;
      }
    }
  }
};

// Largest |v| over 16-byte vectors of DT as they lie in memory: a run keeps a word (for 16-bit types one
// maximum in each half; unsigned order again) and ends with top_bits.
template <int DT>
__device__ __forceinline__ uint32_t vec_top(const uint4& v, uint32_t top) {
  if constexpr (DT == FMOE_F32)
    return max(max(top, max(v.x & 0x7fffffffu, v.y & 0x7fffffffu)), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
  else
    return __vimax3_u16x2(__vimax3_u16x2(top, v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), v.z & 0x7fff7fffu, v.w & 0x7fff7fffu);
}
template <int DT>
__device__ __forceinline__ uint32_t top_bits(uint32_t top) {
  if constexpr (DT == FMOE_F32) {
    return top;
  } else {
    const uint32_t b = max(top & 0xffffu, top >> 16);
    return DT == FMOE_BF16 ? b << 16 : abs_bits(__half2float(__ushort_as_half(static_cast<uint16_t>(b))));
  }
}

// Four int8 in a word as floats: v + 128 goes into the last bits of 2^23, no conversion either.
__device__ __forceinline__ void unpack_int8(uint32_t w, float* f) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 + i)) - 8388736.f;
}

#endif  // __CUDACC__

}  // namespace fmoe
