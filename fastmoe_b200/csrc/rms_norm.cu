// Root-mean-square norm of the residual stream, forward and backward, with an optional 8-bit
// output, and the row quantiser of the int8 products.
//
//   s    = x + residual, rounded to the rows' type (that is what the stream holds)
//   rstd = 1 / sqrt(mean(s^2) + eps)            y = s * rstd * w
//   dx   = rstd * (g - xh * mean(g * xh)) + ds  with g = dy * w, xh = s * rstd
//   dw   = sum over rows of dy * xh
//
// Every kernel is bound by HBM: a row is read once, held in registers across its reductions, and
// every output is written once. The sum of squares runs in 64 bits: the 8-bit output rounds next
// to borders. How a row is split over threads then moves rstd in fp32 only where it lies within some 2^-50 of
// a border between two fp32 values, so a row quantises the same in a batch of one and in a batch of
// thousands, but for about one row in 2^25. It costs one conversion and one fused multiply-add per
// element, far below what a row's bytes take.
#include "int8.cuh"

namespace fmoe {

struct RowArgs {
  const void* x;
  const void* residual;  // optional
  const void* w;         // NORM only
  void* y;               // optional
  void* sum;             // with residual: s
  float* rstd;           // optional [T]
  int8_t* q;             // optional
  float* q_scale;
  int64_t T, D;
  int64_t x_stride, r_stride, q_stride;
  double eps, inv_d;  // inv_d: 1 / D
  int w_f32;
  int shift0, shift_step;  // see row_shift
};

// ---- a row as 16-byte vectors, wherever it starts ------------------------------------------------
// A row of odd width starts anywhere on the 2- or 4-byte grid. What matters for wide accesses is that
// all tensors of a call are off the 16-byte grid by the same number of elements in a given row,
// which contiguous tensors of one shape are: the row is then cut at the grid, vector c holds the
// elements c * VE - shift + (0 .. VE - 1), and only the first and the last one may be partial. Those are
// loaded whole too, as far as the tensor goes, and masked: a row then waits for HBM once, not once more
// for each of its ends (8631 x 4669 bf16: 76 us with the ends read element by element).
__device__ __forceinline__ int row_shift(int shift0, int shift_step, int64_t row, int VE) {
  return (shift0 + static_cast<int>(row & (VE - 1)) * shift_step) & (VE - 1);
}

// What a shifted row's partial vectors need, one at each end of a row, on words as they lie in memory: for
// rows of a few hundred columns they are much of the work (36036 x 333 bf16 with residual 49 -> 34 us against
// conversions to floats and back, 14742 x 814 30 -> 24.5). The load is out of line: it is for the first and
// the last row of a tensor alone.
template <int DT>
__device__ __noinline__ uint4 load_partial(const typename Elem<DT>::type* row, int e, int D) {
  float f[Elem<DT>::kVec];
#pragma unroll
  for (int j = 0; j < Elem<DT>::kVec; ++j) f[j] = e + j >= 0 && e + j < D ? to_float<DT>(row[e + j]) : 0.f;
  return pack16<DT>(f);
}
// v with zeros for the elements outside the row.
template <int DT>
__device__ __forceinline__ uint4 mask_partial(uint4 v, int e, int D) {
  uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == FMOE_F32) {
      if (static_cast<uint32_t>(e + i) >= static_cast<uint32_t>(D)) x[i] = 0;
    } else {
      if (static_cast<uint32_t>(e + 2 * i) >= static_cast<uint32_t>(D)) x[i] &= 0xffff0000u;
      if (static_cast<uint32_t>(e + 2 * i + 1) >= static_cast<uint32_t>(D)) x[i] &= 0xffffu;
    }
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}
template <int DT>
__device__ __forceinline__ void store_partial(typename Elem<DT>::type* row, int e, int D, uint4 v) {
  const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == FMOE_F32) {
      if (static_cast<uint32_t>(e + i) < static_cast<uint32_t>(D)) reinterpret_cast<uint32_t*>(row + e)[i] = x[i];
    } else {
      uint16_t* to = reinterpret_cast<uint16_t*>(row + e) + 2 * i;
      if (static_cast<uint32_t>(e + 2 * i) < static_cast<uint32_t>(D)) to[0] = static_cast<uint16_t>(x[i]);
      if (static_cast<uint32_t>(e + 2 * i + 1) < static_cast<uint32_t>(D)) to[1] = static_cast<uint16_t>(x[i] >> 16);
    }
  }
}

// A row and how far its tensors are known to reach around it: elements [lo, hi) may be read.
struct Span {
  int D, lo, hi;
  __device__ Span(int64_t row, int64_t T, int64_t width) : D(static_cast<int>(width)) {
    // rows are at least `width` apart; no vector reaches further than 8 elements over an end
    lo = row > 0 ? -static_cast<int>(width < 8 && row * width < 8 ? row * width : 8) : 0;
    const int64_t behind = (T - 1 - row) * width;
    hi = D + static_cast<int>(behind < 8 ? behind : 8);
  }
};

// How the kernels cut rows: rows that start on the grid and end on it, shifted rows, or (tensors that
// are off the grid by different amounts) one element at a time.
enum Cut { kAligned, kShifted, kSingle };

// Elements e .. e + kElems - 1 of a row of D, in registers as they lie in memory; those outside the row are zeros.
template <int DT, int CUT>
struct Vec {
  using E = typename Elem<DT>::type;
  static constexpr int kElems = Elem<DT>::kVec;
  uint4 v;
  __device__ __forceinline__ static bool whole(int e, int D) { return CUT == kAligned || (e >= 0 && e + kElems <= D); }
  __device__ __forceinline__ static bool readable(int e, const Span& s) {
    return CUT == kAligned || (e >= s.lo && e + kElems <= s.hi);
  }
  __device__ __forceinline__ void load(const E* row, int e, const Span& s) {
    if (readable(e, s)) v = ld_stream16(reinterpret_cast<const uint4*>(row + e));
    else v = load_partial<DT>(row, e, s.D);
  }
  __device__ __forceinline__ void mask(int e, const Span& s) {
    if (!whole(e, s.D)) v = mask_partial<DT>(v, e, s.D);
  }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  // load() on its way to 16 bytes of shared memory, asynchronously.
  __device__ __forceinline__ static void fetch(uint4* slot, const E* row, int e, const Span& s) {
    if (readable(e, s))
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(slot))),
                   "l"(row + e)
                   : "memory");
    else
      *slot = load_partial<DT>(row, e, s.D);
  }
  __device__ __forceinline__ void get(float* f) const { unpack16<DT>(v, f); }
  __device__ __forceinline__ void set(const float* f) { v = pack16<DT>(f); }
  __device__ __forceinline__ void store(E* row, int e, int D) const {
    if (whole(e, D)) *reinterpret_cast<uint4*>(row + e) = v;
    else store_partial<DT>(row, e, D, v);
  }
  __device__ __forceinline__ uint32_t top(uint32_t t) const { return vec_top<DT>(v, t); }
  __device__ __forceinline__ static uint32_t bits(uint32_t t) { return top_bits<DT>(t); }
};
template <int DT>
struct Vec<DT, kSingle> {
  using E = typename Elem<DT>::type;
  static constexpr int kElems = 1;
  E v;
  __device__ __forceinline__ void load(const E* row, int e, const Span&) { v = row[e]; }
  __device__ __forceinline__ void mask(int, const Span&) {}
  __device__ __forceinline__ void zero() { v = from_float<DT>(0.f); }
  __device__ __forceinline__ void get(float* f) const { f[0] = to_float<DT>(v); }
  __device__ __forceinline__ void set(const float* f) { v = from_float<DT>(f[0]); }
  __device__ __forceinline__ void store(E* row, int e, int) const { row[e] = v; }
  __device__ __forceinline__ uint32_t top(uint32_t t) const { return max(t, abs_bits(to_float<DT>(v))); }
  __device__ __forceinline__ static uint32_t bits(uint32_t t) { return t; }
};

// Words that 16-bit weights e .. e + 7 lie in, from the word of e on: an odd e needs half of a fifth. The
// vectors that are read so end before the last weight (e + 8 < D); no word of theirs reaches past it.
__host__ __device__ constexpr int weight_words(int e) { return 4 + (e & 1); }
constexpr bool weight_words_inside() {
  for (int D = 9; D < 64; ++D)
    for (int e = 1; e + 8 < D; ++e)
      if ((e & ~1) + 2 * weight_words(e) > D) return false;
  return true;
}
static_assert(weight_words_inside(), "a shifted row's weights are read inside the weight");

// Weights e .. e + VE - 1, fp32 or of the rows' type, as floats; zeros outside the row. The weight
// starts on the grid whatever the row does, so in a shifted row a vector of 16-bit weights comes in four or five words,
// fp32 ones one by one, out of L1 (1714 x 7001 bf16: 17.2 us with single 16-bit ones, 15.5).
template <int DT, int CUT>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int e, int D, float* f) {
  using E = typename Elem<DT>::type;
  constexpr int VE = Vec<DT, CUT>::kElems;
  if (CUT == kAligned || (CUT == kShifted && (e & (VE - 1)) == 0 && e + VE <= D)) {
    if constexpr (CUT != kSingle) {
      if (w_f32) {
#pragma unroll
        for (int j = 0; j < VE; j += 4)
          unpack16<FMOE_F32>(ld_cached16(reinterpret_cast<const uint4*>(static_cast<const float*>(w) + e + j)), f + j);
      } else {
        unpack16<DT>(ld_cached16(reinterpret_cast<const uint4*>(static_cast<const E*>(w) + e)), f);
      }
    }
  } else if (CUT == kShifted && DT != FMOE_F32 && !w_f32 && e > 0 && e + VE < D) {
    const uint32_t* from = reinterpret_cast<const uint32_t*>(static_cast<const E*>(w) + (e & ~1));
    uint32_t x[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) x[i] = i < weight_words(e) ? __ldg(from + i) : 0u;
    if (e & 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __funnelshift_r(x[i], x[i + 1], 16);
    unpack16<DT>(make_uint4(x[0], x[1], x[2], x[3]), f);
  } else if (e >= 0 && e + VE <= D) {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      f[j] = w_f32 ? static_cast<const float*>(w)[e + j] : to_float<DT>(static_cast<const E*>(w)[e + j]);
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      f[j] = 0.f;
      if (e + j >= 0 && e + j < D)
        f[j] = w_f32 ? static_cast<const float*>(w)[e + j] : to_float<DT>(static_cast<const E*>(w)[e + j]);
    }
  }
}

// q of elements e .. to a row of 8-bit values, which starts on the grid: in the widest pieces that the
// shift leaves aligned.
template <int VE, int CUT>
__device__ __forceinline__ void store_int8(int8_t* row, int e, int D, const uint32_t* words) {
  if constexpr (VE == 1) {
    row[e] = static_cast<int8_t>(words[0]);
  } else if (CUT == kAligned || (e >= 0 && e + VE <= D && (e & (VE - 1)) == 0)) {
    if constexpr (VE == 8) *reinterpret_cast<uint2*>(row + e) = make_uint2(words[0], words[1]);
    else *reinterpret_cast<uint32_t*>(row + e) = words[0];
  } else if (e >= 0 && e + VE <= D && (e & 1) == 0) {
#pragma unroll
    for (int j = 0; j < VE / 2; ++j)
      *reinterpret_cast<uint16_t*>(row + e + 2 * j) = static_cast<uint16_t>(words[j / 2] >> (16 * (j & 1)));
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (e + j >= 0 && e + j < D) row[e + j] = static_cast<int8_t>(words[j / 4] >> (8 * (j & 3)));
  }
}

// ---- reductions over the threads of a row: a warp, or the whole CTA ----------------------------
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
template <bool WARP, typename T>
__device__ __forceinline__ T row_sum(T v, T* part) {
  v = warp_sum(v);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = warp_sum(lane < (blockDim.x >> 5) ? part[lane] : T(0));
  }
  return v;
}
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lane < (blockDim.x >> 5) ? part[lane] : 0u);
  }
  return v;
}

// 1 / sqrt(mean + eps) to the last bit of 64: the fp32 instruction's 22 good bits, doubled once by
// Householder's iteration of third order. Quotient and root in 64 bits cost 150 instructions, which
// every warp of a row would issue.
__device__ __forceinline__ float inv_rms(double sum_sq, double inv_d, double eps) {
  const double v = fma(sum_sq, inv_d, eps);
  if (!(v > 1e-30 && v < 1e30)) return static_cast<float>(1.0 / sqrt(v));
  const double y = static_cast<double>(rsqrtf(static_cast<float>(v)));
  const double e = fma(-(v * y), y, 1.0);
  return static_cast<float>(fma(y * e, fma(e, 0.375, 0.5), y));
}

// Threads that a CTA of these kernels may have: 16 elements a thread and more need over 64 registers.
constexpr int row_threads(int elements) { return elements > 8 ? 512 : 1024; }

// One row per CTA, or per warp (WARP: narrow rows, threadIdx.y picks the row), each thread holding
// VPT vectors of it in registers, as they lie in memory: what is unpacked twice costs fewer cycles
// than the CTAs that 32 fp32 registers a thread would keep off the SM.
template <int DT, int CUT, int VPT, bool WARP, bool NORM>
__global__ void __launch_bounds__(WARP ? 256 : row_threads(VPT * Vec<DT, CUT>::kElems),
                                  !WARP && NORM && DT != FMOE_F32 && VPT == 4 ? 2 : 0) row_kernel(const RowArgs a) {
  __shared__ double part_sum[32];
  __shared__ uint32_t part_max[32];
  constexpr int VE = Vec<DT, CUT>::kElems;
  const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y : blockIdx.x;
  // the product that reads these rows may set itself up meanwhile; it waits for this grid to end
  if (a.q != nullptr) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (row >= a.T) return;  // WARP only: no barrier follows
  const int tid = threadIdx.x, nthr = WARP ? 32 : blockDim.x;
  const int D = static_cast<int>(a.D);
  using E = typename Elem<DT>::type;
  const int first = tid * VE - (CUT == kShifted ? row_shift(a.shift0, a.shift_step, row, VE) : 0);  // this thread's first element
  const int step = nthr * VE;
  const Span span(row, a.T, a.D);

  Vec<DT, CUT> sv[VPT];
  {
    const E* x = static_cast<const E*>(a.x) + row * a.x_stride;
    const E* r = static_cast<const E*>(a.residual) + row * a.r_stride;
    Vec<DT, CUT> rv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = first + i * step;
      if (e < D) {
        sv[i].load(x, e, span);
        if (NORM && a.residual != nullptr) rv[i].load(r, e, span);
      } else {
        sv[i].zero();
      }
    }
    if constexpr (CUT == kShifted) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = first + i * step;
        if (e < D) {
          sv[i].mask(e, span);
          if (NORM && a.residual != nullptr) rv[i].mask(e, span);
        }
      }
    }
    if (NORM && a.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = first + i * step;
        if (e < D) {
          float f[VE], g[VE];
          sv[i].get(f);
          rv[i].get(g);
#pragma unroll
          for (int j = 0; j < VE; ++j) f[j] += g[j];
          sv[i].set(f);  // the one rounding of the sum
          sv[i].store(static_cast<E*>(a.sum) + row * a.D, e, D);
        }
      }
    }
  }
  uint32_t top = 0;
  float rstd = 1.f;
  if constexpr (NORM) {
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[VE];
      sv[i].get(f);
#pragma unroll
      for (int j = 0; j < VE; ++j) sq = fma(static_cast<double>(f[j]), static_cast<double>(f[j]), sq);
    }
    rstd = inv_rms(row_sum<WARP>(sq, part_sum), a.inv_d, a.eps);
    if (a.rstd != nullptr && tid == 0) a.rstd[row] = rstd;
  }
  auto value = [&](int i, float* f) {
    sv[i].get(f);
    if constexpr (NORM) {
      float w[VE];
      load_weight<DT, CUT>(a.w, a.w_f32, first + i * step, D, w);
      if constexpr (VE > 1) {  // two to an instruction
#pragma unroll
        for (int j = 0; j < VE; j += 2) {
          const float2 y = mul2(mul2(make_float2(f[j], f[j + 1]), make_float2(rstd, rstd)), make_float2(w[j], w[j + 1]));
          f[j] = y.x;
          f[j + 1] = y.y;
        }
      } else {
        f[0] = f[0] * rstd * w[0];
      }
    }
  };
  float top_y = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = first + i * step;
    if (e < D) {
      if constexpr (NORM) {
        float f[VE];
        value(i, f);
        if (a.y != nullptr) {
          Vec<DT, CUT> out;
          out.set(f);
          out.store(static_cast<E*>(a.y) + row * a.D, e, D);
        }
        // elements outside the row are zeros, or NaN where the row is not finite
#pragma unroll
        for (int j = 0; j < VE; ++j) top_y = max_abs(top_y, f[j]);
      } else {
        top = sv[i].top(top);
      }
    }
  }
  if (a.q == nullptr) return;
  if constexpr (NORM) top = abs_bits(top_y);
  else top = Vec<DT, CUT>::bits(top);
  const Quantiser quant(row_max<WARP>(top, part_max));
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = first + i * step;
    if (e < D) {
      float f[VE];
      uint32_t words[(VE + 3) / 4];
      value(i, f);
      if constexpr (NORM || DT == FMOE_F32) quant.template operator()<VE>(f, words);
      else quant.template from16<VE>(f, words);
      store_int8<VE, CUT>(q, e, D, words);
    }
  }
  const int pad = static_cast<int>((16 - (a.D & 15)) & 15);  // up to the next 16 bytes: zeros
  if (tid < pad) q[a.D + tid] = 0;
  if (tid == 0) a.q_scale[row] = quant.scale();
}

// Rows too wide for registers: three passes over the row, the later ones out of L2.
template <int DT, bool NORM>
__global__ void __launch_bounds__(1024) row_loop_kernel(const RowArgs a) {
  __shared__ double part_sum[32];
  __shared__ uint32_t part_max[32];
  using E = typename Elem<DT>::type;
  const int64_t row = blockIdx.x;
  const int D = static_cast<int>(a.D);
  const E* x = static_cast<const E*>(a.x) + row * a.x_stride;
  E* sum = static_cast<E*>(a.sum) + row * a.D;
  double sq = 0.0;
  for (int c = threadIdx.x; c < D; c += blockDim.x) {
    float f = to_float<DT>(x[c]);
    if (a.residual != nullptr) {
      const E s = from_float<DT>(f + to_float<DT>(static_cast<const E*>(a.residual)[row * a.r_stride + c]));
      sum[c] = s;  // read again below by this same thread
      f = to_float<DT>(s);
    }
    sq = fma(static_cast<double>(f), static_cast<double>(f), sq);
  }
  float rstd = 1.f;
  if constexpr (NORM) {
    rstd = inv_rms(row_sum<false>(sq, part_sum), a.inv_d, a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
  }
  auto value = [&](int c) {
    float f = to_float<DT>(a.residual != nullptr ? sum[c] : x[c]);
    if constexpr (NORM) {
      float w;
      load_weight<DT, kSingle>(a.w, a.w_f32, c, D, &w);
      f = f * rstd * w;
    }
    return f;
  };
  uint32_t top = 0;
  for (int c = threadIdx.x; c < D; c += blockDim.x) {
    const float f = value(c);
    if (a.y != nullptr) static_cast<E*>(a.y)[row * a.D + c] = from_float<DT>(f);
    top = max(top, abs_bits(f));
  }
  if (a.q == nullptr) return;
  const Quantiser quant(row_max<false>(top, part_max));
  int8_t* q = a.q + row * a.q_stride;
  for (int c = threadIdx.x; c < D; c += blockDim.x) {
    const float f = value(c);
    uint32_t word;
    if constexpr (NORM || DT == FMOE_F32) quant.operator()<1>(&f, &word);
    else quant.from16<1>(&f, &word);
    q[c] = static_cast<int8_t>(word);
  }
  const int pad = static_cast<int>((16 - (a.D & 15)) & 15);
  if (threadIdx.x < pad) q[a.D + threadIdx.x] = 0;
  if (threadIdx.x == 0) a.q_scale[row] = quant.scale();
}

// ---- backward -------------------------------------------------------------------------------
struct RowBwdArgs {
  const void* dy;
  const void* ds;  // optional: gradient of the stream
  const void* s;   // the stream as stored
  const float* rstd;
  const void* w;
  void* dx;
  float* part;  // optional [gridDim.x, D]: this CTA's share of dw
  int64_t T, D;
  int64_t dy_stride, ds_stride, s_stride;
  float inv_d;  // 1 / D
  int w_f32;
  int shift0, shift_step;
};

// A CTA (or each of its warps) walks rows t, t + grid, ... and keeps its columns' share of dw in
// registers; the shares are added by rms_dw_kernel in a fixed order, so dw has the same bits from
// run to run. Rows of one thread are a multiple of VE apart, so that their shift is the same and a
// thread's columns stay its own. The weight lies in shared memory as fp32, in the CTA's shifted
// order and in planes of four columns (16-byte reads without bank conflicts). Each thread fetches its
// vectors of the next row into shared memory slots of its own while it works on this one: with the
// loads issued row by row into registers two CTAs an SM left HBM idle half of the time between
// them (16384 x 7168 bf16: 169 us, 5.5 TB/s).
// CTAs of eight one-warp rows that an SM holds at a time, for the columns of a thread: the grid is this many
// to an SM, all of them at once (60000 x 200 bf16 34 -> 24 us, 23437 x 512 29 -> 22 us, against four to an SM).
constexpr int warp_ctas(int columns) { return columns <= 8 ? 3 : 2; }

template <int DT, int CUT, int VPT, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : row_threads(VPT * Vec<DT, CUT>::kElems),
                                  WARP ? warp_ctas(VPT * Vec<DT, CUT>::kElems) : 0) rms_bwd_kernel(const RowBwdArgs a) {
  __shared__ float part_sum[2][32];
  extern __shared__ __align__(16) float w_smem[];
  constexpr int VE = Vec<DT, CUT>::kElems;
  using E = typename Elem<DT>::type;
  const int tid = threadIdx.x, nthr = WARP ? 32 : blockDim.x;
  const int D = static_cast<int>(a.D);
  const int rows_per_cta = WARP ? blockDim.y : 1;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_per_cta + (WARP ? threadIdx.y : 0);
  const int first = tid * VE - (CUT == kShifted ? row_shift(a.shift0, a.shift_step, row0, VE) : 0);
  const int step = nthr * VE;
  constexpr int kPlanes = VE >= 4 ? VE / 4 : 1, kWide = VE >= 4 ? 4 : 1;
  const int plane = nthr * VPT * kWide;  // floats per plane
  if constexpr (!WARP) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float w[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) w[j] = 0.f;
      if (first + i * step < D) load_weight<DT, CUT>(a.w, a.w_f32, first + i * step, D, w);
#pragma unroll
      for (int p = 0; p < kPlanes; ++p)
#pragma unroll
        for (int j = 0; j < kWide; ++j) w_smem[p * plane + (i * nthr + tid) * kWide + j] = w[p * kWide + j];
    }
  }  // each thread reads back what it wrote itself: no barrier
  float w_own[WARP ? VPT : 1][VE];  // a warp's row is short enough for registers
  if constexpr (WARP) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (first + i * step < D) load_weight<DT, CUT>(a.w, a.w_f32, first + i * step, D, w_own[i]);
  }
  auto weight = [&](int i, float* w) {
    if constexpr (WARP) {
#pragma unroll
      for (int j = 0; j < VE; ++j) w[j] = w_own[i][j];
    } else if constexpr (VE >= 4) {
#pragma unroll
      for (int p = 0; p < kPlanes; ++p) {
        const float4 q = *reinterpret_cast<const float4*>(w_smem + p * plane + (i * nthr + tid) * 4);
        w[4 * p] = q.x, w[4 * p + 1] = q.y, w[4 * p + 2] = q.z, w[4 * p + 3] = q.w;
      }
    } else {
      w[0] = w_smem[i * nthr + tid];
    }
  };
  float dw[VPT][VE];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[i][j] = 0.f;
  constexpr bool kAhead = CUT != kSingle;
  uint4* slots = reinterpret_cast<uint4*>(w_smem + (WARP ? (D + 3) / 4 * 4 : kPlanes * plane)) +
                 (WARP ? threadIdx.y * (3 * VPT * 32) : 0) + tid;  // [3][VPT][nthr], kAhead only
  const int64_t row_step = static_cast<int64_t>(gridDim.x) * rows_per_cta;
  auto fetch = [&](int64_t row) {
    if constexpr (kAhead) {
      const Span span(row, a.T, a.D);
      const E* s = static_cast<const E*>(a.s) + row * a.s_stride;
      const E* dy = static_cast<const E*>(a.dy) + row * a.dy_stride;
      const E* ds = static_cast<const E*>(a.ds) + row * a.ds_stride;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = first + i * step;
        if (e < D) {
          Vec<DT, CUT>::fetch(slots + i * nthr, s, e, span);
          Vec<DT, CUT>::fetch(slots + (VPT + i) * nthr, dy, e, span);
          if (a.ds != nullptr) Vec<DT, CUT>::fetch(slots + (2 * VPT + i) * nthr, ds, e, span);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  if (row0 < a.T) fetch(row0);
  int flip = 0;  // two sets of partial sums: a row's first write never meets the last row's reads
  for (int64_t row = row0; row < a.T; row += row_step, flip ^= 1) {
    Vec<DT, CUT> sv[VPT], gv[VPT], dv[VPT];
    const float rstd = a.rstd[row];
    const Span span(row, a.T, a.D);
    if constexpr (kAhead) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        sv[i].v = slots[i * nthr];
        gv[i].v = slots[(VPT + i) * nthr];
        dv[i].v = slots[(2 * VPT + i) * nthr];
      }
      if (row + row_step < a.T) fetch(row + row_step);  // this thread has read its slots
    } else {
      const E* s = static_cast<const E*>(a.s) + row * a.s_stride;
      const E* dy = static_cast<const E*>(a.dy) + row * a.dy_stride;
      const E* ds = static_cast<const E*>(a.ds) + row * a.ds_stride;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = first + i * step;
        if (e < D) {
          sv[i].load(s, e, span);
          gv[i].load(dy, e, span);
          if (a.ds != nullptr) dv[i].load(ds, e, span);
        }
      }
    }
    if constexpr (CUT == kShifted) {  // what lies outside the row counts as zero; ds only meets the store
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e = first + i * step;
        if (e < D) {
          sv[i].mask(e, span);
          gv[i].mask(e, span);
        }
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (first + i * step < D) {
        float xh[VE], g[VE], w[VE];
        sv[i].get(xh);
        gv[i].get(g);
        weight(i, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float t = g[j] * (xh[j] * rstd);
          dw[i][j] += t;
          dot = fmaf(t, w[j], dot);
        }
      }
    }
    const float mean = row_sum<WARP>(dot, part_sum[flip]) * a.inv_d;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = first + i * step;
      if (e < D) {
        float xh[VE], g[VE], w[VE], d[VE];
        sv[i].get(xh);
        gv[i].get(g);
        weight(i, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) d[j] = 0.f;
        if (a.ds != nullptr) dv[i].get(d);
#pragma unroll
        for (int j = 0; j < VE; ++j) d[j] = fmaf(rstd, fmaf(-(xh[j] * rstd), mean, g[j] * w[j]), d[j]);
        Vec<DT, CUT> out;
        out.set(d);
        out.store(static_cast<E*>(a.dx) + row * a.D, e, D);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * a.D;
  if constexpr (WARP) {  // the CTA's warps, one after the other
    for (int y = 0; y < blockDim.y; ++y) {
      if (threadIdx.y == y) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const int e = first + i * step + j;
            if (e >= 0 && e < D) w_smem[e] = y == 0 ? dw[i][j] : w_smem[e] + dw[i][j];
          }
      }
      __syncthreads();
    }
    for (int e = threadIdx.y * 32 + tid; e < D; e += blockDim.y * 32) part[e] = w_smem[e];
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const int e = first + i * step + j;
        if (e >= 0 && e < D) part[e] = dw[i][j];
      }
  }
}

// Rows too wide for registers: two passes over a row, dw gathered in this CTA's row of `part`.
template <int DT>
__global__ void __launch_bounds__(1024) rms_bwd_loop_kernel(const RowBwdArgs a) {
  __shared__ float part_sum[2][32];
  using E = typename Elem<DT>::type;
  const int D = static_cast<int>(a.D);
  float* part = a.part == nullptr ? nullptr : a.part + static_cast<int64_t>(blockIdx.x) * a.D;
  int flip = 0;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1) {
    const E* s = static_cast<const E*>(a.s) + row * a.s_stride;
    const E* dy = static_cast<const E*>(a.dy) + row * a.dy_stride;
    const float rstd = a.rstd[row];
    float dot = 0.f;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      float w;
      load_weight<DT, kSingle>(a.w, a.w_f32, c, D, &w);
      const float t = to_float<DT>(dy[c]) * (to_float<DT>(s[c]) * rstd);
      if (part != nullptr) part[c] = first ? t : part[c] + t;  // this thread alone has this column
      dot = fmaf(t, w, dot);
    }
    first = false;
    const float mean = row_sum<false>(dot, part_sum[flip]) * a.inv_d;
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      float w;
      load_weight<DT, kSingle>(a.w, a.w_f32, c, D, &w);
      const float d = a.ds == nullptr ? 0.f : to_float<DT>(static_cast<const E*>(a.ds)[row * a.ds_stride + c]);
      const float v = fmaf(rstd, fmaf(-(to_float<DT>(s[c]) * rstd), mean, to_float<DT>(dy[c]) * w), d);
      static_cast<E*>(a.dx)[row * a.D + c] = from_float<DT>(v);
    }
  }
}

// dw[c] = sum over the CTAs' shares: 32 warps take every 32nd share of 32 columns each, then the 32 sums
// are added in order.
constexpr int kDwWarps = 32;
__global__ void __launch_bounds__(32 * kDwWarps) rms_dw_kernel(const float* part, int shares, int64_t D, void* dw, int dt) {
  __shared__ float acc[kDwWarps][32];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
  float sum = 0.f;
  if (c < D)
#pragma unroll 8
    for (int i = threadIdx.y; i < shares; i += kDwWarps) sum += part[static_cast<int64_t>(i) * D + c];
  acc[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < D) {
#pragma unroll
    for (int y = 1; y < kDwWarps; ++y) sum += acc[y][threadIdx.x];
    store_scalar_from_float(dw, c, dt, sum);
  }
}

// ---- 8-bit rows back to floating point --------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out,
                                                         int total, int D, FastDiv per_row, int vec) {
  using E = typename Elem<DT>::type;
  constexpr int VE = Elem<DT>::kVec;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * VE;
    const int64_t row = row_of;
    const float s = scale[row];
    const int8_t* p = q + row * q_stride + c;
    E* o = static_cast<E*>(out) + row * D + c;
    if (vec) {
      float f[VE];
      if constexpr (VE == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        unpack_int8(w.x, f);
        unpack_int8(w.y, f + 4);
      } else {
        unpack_int8(*reinterpret_cast<const uint32_t*>(p), f);
      }
#pragma unroll
      for (int j = 0; j < VE; j += 2) {
        const float2 y = mul2(make_float2(f[j], f[j + 1]), make_float2(s, s));
        f[j] = y.x;
        f[j + 1] = y.y;
      }
      st_stream16(reinterpret_cast<uint4*>(o), pack16<DT>(f));
    } else {
      for (int j = 0; j < VE && c + j < D; ++j) o[j] = from_float<DT>(static_cast<float>(p[j]) * s);
    }
  }
}

// ---- host side ------------------------------------------------------------------------------
// The shift of row r is (shift0 + r * shift_step) mod VE (row_shift) if all tensors of the call agree on
// it; `vec` says whether they do.
struct RowGrid {
  int ve, shift0 = -1, shift_step = 0;
  bool vec = true;
  RowGrid(int dtype) : ve(16 / dtype_size(dtype)), es(dtype_size(dtype)) {}
  void add(const void* p, int64_t stride, int64_t T) {
    if (p == nullptr) return;
    const int s0 = static_cast<int>(reinterpret_cast<uintptr_t>(p) / es % ve);
    const int st = T > 1 ? static_cast<int>(stride % ve) : 0;
    if (reinterpret_cast<uintptr_t>(p) % es != 0 || (shift0 >= 0 && (s0 != shift0 || st != shift_step))) vec = false;
    shift0 = s0;
    shift_step = st;
  }
  void weight(const void* w) { vec = vec && aligned_to(w, 16); }
  bool shifted() const { return vec && (shift0 != 0 || shift_step != 0); }

 private:
  int es;
};

// How a row is split: a warp per row while a row fits 32 threads, else a CTA. A CTA takes four vectors a
// thread when there are rows enough to fill the GPU (more loads in flight per thread), one or two
// when there are not (the latency of a single row falls with the vectors per thread). The backward pass
// of 16-bit rows of up to 256 vectors takes two: it holds three inputs and the dw of eight columns to a
// vector, and is short of warps at four (14742 x 814 bf16 43 -> 29 us, 11718 x 1024 23 -> 19; fp32 rows,
// half the columns to a vector, are slower with two, 33 -> 38 us).
struct RowShape {
  Cut cut;
  bool warp, loop;
  int vpt, threads;
};
static RowShape row_shape(const RowGrid& g, int64_t D, int64_t T, int dtype, bool backward) {
  const bool vec = g.vec;
  RowShape s{!vec ? kSingle : g.shifted() || D % g.ve != 0 ? kShifted : kAligned, false, false, 0, 0};
  const int ve = vec ? g.ve : 1;
  const int most = vec ? (dtype == FMOE_F32 ? 8 : 4) : 16;  // vectors a thread can hold: 32 elements, or 16 single ones
  const int64_t nvec = (D + (g.shifted() ? ve - 1 : 0) + ve - 1) / ve;  // of the row with the largest shift
  if (nvec <= 32 * (vec ? 2 : 16)) {
    s.warp = true;
    s.threads = 32;
    s.vpt = vec ? (nvec <= 32 ? 1 : 2) : 16;
    return s;
  }
  s.vpt = T <= 2 * kNumSMs ? (vec ? 1 : 4) : (vec ? (backward && dtype != FMOE_F32 && nvec <= 256 ? 2 : 4) : 16);
  while (s.vpt <= most && (nvec + s.vpt - 1) / s.vpt > row_threads(s.vpt * ve)) s.vpt *= vec ? 2 : 4;
  s.loop = s.vpt > most;
  s.threads = static_cast<int>(((nvec + s.vpt - 1) / s.vpt + 31) / 32 * 32);
  return s;
}

// The instantiation for RowShape s, through FMOE_ROWS(CUT, VPT, WARP).
#define FMOE_PICK_ROWS                                                   \
  do {                                                                   \
    if (s.cut == kSingle) {                                              \
      if (s.warp) FMOE_ROWS(kSingle, 16, true);                          \
      else if (s.vpt == 4) FMOE_ROWS(kSingle, 4, false);                 \
      else FMOE_ROWS(kSingle, 16, false);                                \
    } else if (s.cut == kAligned) {                                      \
      FMOE_PICK_VPT(kAligned);                                           \
    } else {                                                             \
      FMOE_PICK_VPT(kShifted);                                           \
    }                                                                    \
  } while (0)
#define FMOE_PICK_VPT(CUT)                                               \
  do {                                                                   \
    if (s.warp && s.vpt == 1) FMOE_ROWS(CUT, 1, true);                   \
    else if (s.warp) FMOE_ROWS(CUT, 2, true);                            \
    else if (s.vpt == 1) FMOE_ROWS(CUT, 1, false);                       \
    else if (s.vpt == 2) FMOE_ROWS(CUT, 2, false);                       \
    else if (s.vpt == 4) FMOE_ROWS(CUT, 4, false);                       \
    else if constexpr (Elem<DT>::kVec == 4) FMOE_ROWS(CUT, 8, false);    \
  } while (0)

template <int DT, bool NORM>
static int launch_rows(const RowArgs& a, const RowShape& s, cudaStream_t st) {
  const dim3 block = s.warp ? dim3(32, a.T >= 8 * kNumSMs ? 8 : 1) : dim3(s.threads);
  const unsigned grid = static_cast<unsigned>(s.warp ? (a.T + block.y - 1) / block.y : a.T);
#define FMOE_ROWS(CUT, VPT, WARP) row_kernel<DT, CUT, VPT, WARP, NORM><<<grid, block, 0, st>>>(a)
  if (s.loop) row_loop_kernel<DT, NORM><<<grid, 1024, 0, st>>>(a);
  else FMOE_PICK_ROWS;
#undef FMOE_ROWS
  return check_launch(NORM ? "row_kernel (norm)" : "row_kernel (quantize)");
}

constexpr int kBwdWarps = 8;  // rows per CTA where a warp takes a row
// Wider rows go through rms_bwd_loop_kernel, three to four times as slow: fp32 3584 x 16384 385 us, floor 108 (bf16
// 7168 x 16384, the same bytes, 145).
constexpr int kBwdSmemMost = 220 * 1024;

// Shared memory of rms_bwd_kernel: the weight (where a warp takes a row the sum of the warps' dw) and the next row's slots.
static int bwd_smem(const RowShape& s, int64_t D, int ve) {
  if (s.warp) return 4 * static_cast<int>((D + 3) / 4 * 4) + (s.cut == kSingle ? 0 : kBwdWarps * 3 * s.vpt * 32 * 16);
  return s.threads * s.vpt * (s.cut == kSingle ? 4 : 4 * ve + 3 * 16);
}

template <int DT>
static int launch_bwd(const RowBwdArgs& a, const RowShape& s, int grid, cudaStream_t st) {
  constexpr int V = Elem<DT>::kVec;
  const dim3 block = s.warp ? dim3(32, kBwdWarps) : dim3(s.threads);
  const int smem = bwd_smem(s, a.D, V);
  cudaError_t err = cudaSuccess;
  // The attribute is one of the kernel, whoever launches it: every caller sets the same value, so that none lowers
  // the limit between another thread's call here and its launch.
#define FMOE_ROWS(CUT, VPT, WARP)                                                                                \
  do {                                                                                                           \
    if (smem > 40 * 1024) /* 48 KB is the limit for this and the static part together */                         \
      err = cudaFuncSetAttribute(rms_bwd_kernel<DT, CUT, VPT, WARP>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                 kBwdSmemMost);                                                                  \
    if (err == cudaSuccess) rms_bwd_kernel<DT, CUT, VPT, WARP><<<grid, block, smem, st>>>(a);                     \
  } while (0)
  if (s.loop) rms_bwd_loop_kernel<DT><<<grid, 1024, 0, st>>>(a);
  else FMOE_PICK_ROWS;
#undef FMOE_ROWS
  FMOE_CUDA(err);
  return check_launch("rms_bwd_kernel");
}

// CTAs of the backward pass, and so shares of dw: as many as the SMs hold at a time (128 registers a
// thread where a CTA takes a row), in a multiple of eight (see rms_bwd_kernel).
static int bwd_grid(int64_t T, int threads, bool warp, int columns) {
  const int per_sm = warp ? warp_ctas(columns) : threads >= 512 ? 1 : threads <= 64 ? 8 : 512 / threads;
  const int64_t rows = warp ? (T + kBwdWarps - 1) / kBwdWarps : T, most = per_sm * kNumSMs / 8 * 8;
  return static_cast<int>(rows < most ? rows : most);
}
// The size query knows neither the type nor the alignment: it answers for the fewest threads a row may get.
static int bwd_grid_most(int64_t T, int64_t D) { return bwd_grid(T, static_cast<int>(D / 32 < 512 ? D / 32 : 512), false, 0); }

}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t r_stride, const void* w,
                             int w_dtype, void* y, void* sum, float* rstd, int8_t* q, int64_t q_stride, float* q_scale,
                             int64_t T, int64_t D, double eps, int dtype, void* stream) {
  FMOE_RANGE("fmoe_rms_norm");
  FMOE_REQUIRE(valid_dtype(dtype) && (w_dtype == dtype || w_dtype == FMOE_F32), FMOE_ERR_ARG,
               "fmoe_rms_norm: bad dtype (the weight is fp32 or of the rows' type)");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 30), FMOE_ERR_ARG, "fmoe_rms_norm: bad sizes");
  FMOE_REQUIRE(eps >= 0.0, FMOE_ERR_ARG, "fmoe_rms_norm: eps must not be negative");
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(x && w && (y || q), FMOE_ERR_ARG, "fmoe_rms_norm: null pointer argument");
  FMOE_REQUIRE((residual == nullptr) == (sum == nullptr), FMOE_ERR_ARG,
               "fmoe_rms_norm: residual and sum come together");
  FMOE_REQUIRE(T == 1 || (x_stride >= D && (!residual || r_stride >= D)), FMOE_ERR_ARG,
               "fmoe_rms_norm: row strides must be at least D");
  FMOE_REQUIRE((q == nullptr) == (q_scale == nullptr), FMOE_ERR_ARG, "fmoe_rms_norm: q and q_scale come together");
  FMOE_REQUIRE(!q || (q_stride % 16 == 0 && q_stride >= D && aligned_to(q, 16)), FMOE_ERR_ARG,
               "fmoe_rms_norm: 8-bit rows must lie at 16-byte steps");
  RowGrid g(dtype);
  g.add(x, x_stride, T);
  g.add(residual, r_stride, T);
  g.add(sum, D, T);
  g.add(y, D, T);
  g.weight(w);
  const RowArgs a{x, residual, w, y, sum, rstd, q, q_scale, T, D, x_stride, r_stride, q_stride, eps, 1.0 / static_cast<double>(D), w_dtype == FMOE_F32,
                  g.shift0, g.shift_step};
  const RowShape s = row_shape(g, D, T, dtype, false);
  int rc = FMOE_OK;
  FMOE_DISPATCH_DTYPE(dtype, DT, rc = (launch_rows<DT, true>(a, s, static_cast<cudaStream_t>(stream))));
  return rc;
}

extern "C" int fmoe_quantize_rows(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* q_scale, int64_t T,
                                  int64_t D, int dtype, void* stream) {
  FMOE_RANGE("fmoe_quantize_rows");
  FMOE_REQUIRE(valid_dtype(dtype), FMOE_ERR_ARG, "fmoe_quantize_rows: bad dtype");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 30), FMOE_ERR_ARG, "fmoe_quantize_rows: bad sizes");
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(x && q && q_scale, FMOE_ERR_ARG, "fmoe_quantize_rows: null pointer argument");
  FMOE_REQUIRE(T == 1 || x_stride >= D, FMOE_ERR_ARG, "fmoe_quantize_rows: the row stride must be at least D");
  FMOE_REQUIRE(q_stride % 16 == 0 && q_stride >= D && aligned_to(q, 16), FMOE_ERR_ARG,
               "fmoe_quantize_rows: 8-bit rows must lie at 16-byte steps");
  RowGrid g(dtype);
  g.add(x, x_stride, T);
  const RowArgs a{x, nullptr, nullptr, nullptr, nullptr, nullptr, q, q_scale, T, D, x_stride, 0, q_stride, 0.0, 0.0, 0,
                  g.shift0, g.shift_step};
  const RowShape s = row_shape(g, D, T, dtype, false);
  int rc = FMOE_OK;
  FMOE_DISPATCH_DTYPE(dtype, DT, rc = (launch_rows<DT, false>(a, s, static_cast<cudaStream_t>(stream))));
  return rc;
}

extern "C" int fmoe_dequantize_rows(const int8_t* q, int64_t q_stride, const float* q_scale, void* out, int64_t T, int64_t D,
                                    int dtype, void* stream) {
  FMOE_RANGE("fmoe_dequantize_rows");
  FMOE_REQUIRE(valid_dtype(dtype), FMOE_ERR_ARG, "fmoe_dequantize_rows: bad dtype");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 30), FMOE_ERR_ARG, "fmoe_dequantize_rows: bad sizes");
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(q && q_scale && out, FMOE_ERR_ARG, "fmoe_dequantize_rows: null pointer argument");
  FMOE_REQUIRE(T == 1 || q_stride >= D, FMOE_ERR_ARG, "fmoe_dequantize_rows: the row stride must be at least D");
  const int ve = 16 / dtype_size(dtype);
  const int vec = D % ve == 0 && q_stride % ve == 0 && aligned_to(q, ve) && aligned_to(out, 16);
  const int64_t per_row = (D + ve - 1) / ve, total = T * per_row;
  FMOE_REQUIRE(total < (1ll << 31) - 1024, FMOE_ERR_UNSUPPORTED, "fmoe_dequantize_rows: too many values");
  const int64_t want = (total + 255) / 256, most = 16 * kNumSMs;
  const unsigned grid = static_cast<unsigned>(want < most ? want : most);
  FMOE_DISPATCH_DTYPE(dtype, DT, dequantize_kernel<DT><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
                                     q, q_stride, q_scale, out, static_cast<int>(total), static_cast<int>(D),
                                     FastDiv(per_row), vec));
  return check_launch("dequantize_kernel");
}

extern "C" size_t fmoe_rms_norm_bwd_bytes(int64_t T, int64_t D) {
  if (T <= 0 || D <= 0) return 0;
  return static_cast<size_t>(bwd_grid_most(T, D)) * static_cast<size_t>(D) * sizeof(float);
}

extern "C" int fmoe_rms_norm_bwd(const void* dy, int64_t dy_stride, const void* dsum, int64_t ds_stride, const void* sum,
                                 int64_t s_stride, const float* rstd, const void* w, int w_dtype, void* dx, void* dw,
                                 void* scratch, size_t scratch_bytes, int64_t T, int64_t D, int dtype, void* stream) {
  FMOE_RANGE("fmoe_rms_norm_bwd");
  FMOE_REQUIRE(valid_dtype(dtype) && (w_dtype == dtype || w_dtype == FMOE_F32), FMOE_ERR_ARG,
               "fmoe_rms_norm_bwd: bad dtype (the weight is fp32 or of the rows' type)");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 30), FMOE_ERR_ARG, "fmoe_rms_norm_bwd: bad sizes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // no rows: the weight's gradient is zero
    if (dw != nullptr) FMOE_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(D) * dtype_size(w_dtype), st));
    return FMOE_OK;
  }
  FMOE_REQUIRE(dy && sum && rstd && w && dx, FMOE_ERR_ARG, "fmoe_rms_norm_bwd: null pointer argument");
  FMOE_REQUIRE(T == 1 || (dy_stride >= D && s_stride >= D && (!dsum || ds_stride >= D)), FMOE_ERR_ARG,
               "fmoe_rms_norm_bwd: row strides must be at least D");
  FMOE_REQUIRE(!dw || (scratch && aligned_to(scratch, 4) && scratch_bytes >= fmoe_rms_norm_bwd_bytes(T, D)),
               FMOE_ERR_WORKSPACE, "fmoe_rms_norm_bwd: scratch of %zu bytes needed", fmoe_rms_norm_bwd_bytes(T, D));
  RowGrid g(dtype);
  g.add(dy, dy_stride, T);
  g.add(sum, s_stride, T);
  g.add(dsum, ds_stride, T);
  g.add(dx, D, T);
  g.weight(w);
  RowShape s = row_shape(g, D, T, dtype, true);
  if (bwd_smem(s, D, g.ve) > kBwdSmemMost) s.loop = true;  // fp32 rows of more than 13312 columns
  const int grid = s.loop ? bwd_grid_most(T, D) : bwd_grid(T, s.threads, s.warp, s.vpt * (g.vec ? g.ve : 1));
  const RowBwdArgs a{dy, dsum, sum, rstd, w, dx, dw ? static_cast<float*>(scratch) : nullptr, T, D,
                     dy_stride, ds_stride, s_stride, 1.f / static_cast<float>(D), w_dtype == FMOE_F32, g.shift0, g.shift_step};
  int rc = FMOE_OK;
  FMOE_DISPATCH_DTYPE(dtype, DT, rc = (launch_bwd<DT>(a, s, grid, st)));
  if (rc != 0 || dw == nullptr) return rc;
  rms_dw_kernel<<<static_cast<unsigned>((D + 31) / 32), dim3(32, kDwWarps), 0, st>>>(static_cast<const float*>(scratch), grid, D, dw,
                                                                            w_dtype);
  return check_launch("rms_dw_kernel");
}
