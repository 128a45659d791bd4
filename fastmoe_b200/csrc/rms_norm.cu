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
// to borders, and with a 64-bit sum the fp32 result does not depend on how the row is split over
// threads, so a row quantises the same in a batch of one and in a batch of thousands. It costs
// one conversion and one fused multiply-add per element, far below what a row's bytes take.
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
  double eps;
  int w_f32;
};

// ---- loads and stores of VE elements -----------------------------------------------------------
template <int DT, int VE>
struct Vec {  // VE elements of 16 bytes in all
  uint4 v;
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    v = ld_stream16(reinterpret_cast<const uint4*>(static_cast<const typename Elem<DT>::type*>(p) + i));
  }
  __device__ __forceinline__ void get(float* f) const { unpack16<DT>(v, f); }
  __device__ __forceinline__ void set(const float* f) { v = pack16<DT>(f); }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    *reinterpret_cast<uint4*>(static_cast<typename Elem<DT>::type*>(p) + i) = v;
  }
};
template <int DT>
struct Vec<DT, 1> {  // one element
  typename Elem<DT>::type v;
  __device__ __forceinline__ void load(const void* p, int64_t i) { v = static_cast<const typename Elem<DT>::type*>(p)[i]; }
  __device__ __forceinline__ void get(float* f) const { f[0] = to_float<DT>(v); }
  __device__ __forceinline__ void set(const float* f) { v = from_float<DT>(f[0]); }
  __device__ __forceinline__ void store(void* p, int64_t i) const { static_cast<typename Elem<DT>::type*>(p)[i] = v; }
};

// VE weights, fp32 or of the rows' type, as floats.
template <int DT, int VE>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int64_t i, float* f) {
  if constexpr (VE == 1) {
    f[0] = w_f32 ? static_cast<const float*>(w)[i] : to_float<DT>(static_cast<const typename Elem<DT>::type*>(w)[i]);
  } else if (w_f32) {
#pragma unroll
    for (int j = 0; j < VE; j += 4)
      unpack16<FMOE_F32>(ld_cached16(reinterpret_cast<const uint4*>(static_cast<const float*>(w) + i + j)), f + j);
  } else {
    unpack16<DT>(ld_cached16(reinterpret_cast<const uint4*>(static_cast<const typename Elem<DT>::type*>(w) + i)), f);
  }
}

template <int VE>
__device__ __forceinline__ void store_int8(int8_t* p, const int* r) {
  if constexpr (VE == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_int8(r[0], r[1], r[2], r[3]), pack_int8(r[4], r[5], r[6], r[7]));
  else if constexpr (VE == 4)
    *reinterpret_cast<uint32_t*>(p) = pack_int8(r[0], r[1], r[2], r[3]);
  else
    *p = static_cast<int8_t>(r[0]);
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

__device__ __forceinline__ float inv_rms(double sum_sq, int64_t D, double eps) {
  return static_cast<float>(1.0 / sqrt(sum_sq / static_cast<double>(D) + eps));
}

// Threads that a CTA of these kernels may have: 16 elements a thread and more need over 64 registers.
constexpr int row_threads(int elements) { return elements > 8 ? 512 : 1024; }

// One row per CTA, or per warp (WARP: narrow rows, threadIdx.y picks the row), each thread holding
// VPT vectors of VE elements of it in registers.
template <int DT, int VE, int VPT, bool WARP, bool NORM>
__global__ void __launch_bounds__(WARP ? 256 : row_threads(VPT * VE)) row_kernel(const RowArgs a) {
  __shared__ double part_sum[32];
  __shared__ uint32_t part_max[32];
  const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y : blockIdx.x;
  if (row >= a.T) return;  // WARP only: no barrier follows
  const int tid = threadIdx.x, nthr = WARP ? 32 : blockDim.x;
  const int nvec = static_cast<int>(a.D / VE);
  using E = typename Elem<DT>::type;
  const E* x = static_cast<const E*>(a.x) + row * a.x_stride;

  float v[VPT][VE];
  {
    Vec<DT, VE> xv[VPT], rv[VPT];
    const E* r = static_cast<const E*>(a.residual) + row * a.r_stride;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
        xv[i].load(x, static_cast<int64_t>(c) * VE);
        if (a.residual != nullptr) rv[i].load(r, static_cast<int64_t>(c) * VE);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
        xv[i].get(v[i]);
        if (a.residual != nullptr) {
          float f[VE];
          rv[i].get(f);
#pragma unroll
          for (int j = 0; j < VE; ++j) f[j] += v[i][j];
          rv[i].set(f);  // the one rounding of the sum
          rv[i].store(static_cast<E*>(a.sum) + row * a.D, static_cast<int64_t>(c) * VE);
          rv[i].get(v[i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) v[i][j] = 0.f;
      }
    }
  }
  if constexpr (NORM) {
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) sq = fma(static_cast<double>(v[i][j]), static_cast<double>(v[i][j]), sq);
    const float rstd = inv_rms(row_sum<WARP>(sq, part_sum), a.D, a.eps);
    if (a.rstd != nullptr && tid == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
        float w[VE];
        load_weight<DT, VE>(a.w, a.w_f32, static_cast<int64_t>(c) * VE, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) v[i][j] = v[i][j] * rstd * w[j];
        if (a.y != nullptr) {
          Vec<DT, VE> out;
          out.set(v[i]);
          out.store(static_cast<E*>(a.y) + row * a.D, static_cast<int64_t>(c) * VE);
        }
      }
    }
  }
  if (a.q == nullptr) return;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) top = max(top, i * nthr + tid < nvec ? abs_bits(v[i][j]) : 0u);
  const Quantiser quant(row_max<WARP>(top, part_max));
  int8_t* q = a.q + row * a.q_stride;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = i * nthr + tid;
    if (c < nvec) {
      int r[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) r[j] = quant(v[i][j]);
      store_int8<VE>(q + static_cast<int64_t>(c) * VE, r);
    }
  }
  const int pad = static_cast<int>((16 - (a.D & 15)) & 15);  // up to the next 16 bytes: zeros
  if (tid < pad) q[a.D + tid] = 0;
  if (tid == 0) a.q_scale[row] = quant.scale;
}

// Rows too wide for registers: three passes over the row, the later ones out of L2.
template <int DT, bool NORM>
__global__ void __launch_bounds__(1024) row_loop_kernel(const RowArgs a) {
  __shared__ double part_sum[32];
  __shared__ uint32_t part_max[32];
  using E = typename Elem<DT>::type;
  const int64_t row = blockIdx.x;
  const E* x = static_cast<const E*>(a.x) + row * a.x_stride;
  E* sum = static_cast<E*>(a.sum) + row * a.D;
  double sq = 0.0;
  for (int64_t c = threadIdx.x; c < a.D; c += blockDim.x) {
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
    rstd = inv_rms(row_sum<false>(sq, part_sum), a.D, a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
  }
  auto value = [&](int64_t c) {
    float f = to_float<DT>(a.residual != nullptr ? sum[c] : x[c]);
    if constexpr (NORM) {
      float w;
      load_weight<DT, 1>(a.w, a.w_f32, c, &w);
      f = f * rstd * w;
    }
    return f;
  };
  uint32_t top = 0;
  for (int64_t c = threadIdx.x; c < a.D; c += blockDim.x) {
    const float f = value(c);
    if (a.y != nullptr) static_cast<E*>(a.y)[row * a.D + c] = from_float<DT>(f);
    top = max(top, abs_bits(f));
  }
  if (a.q == nullptr) return;
  const Quantiser quant(row_max<false>(top, part_max));
  int8_t* q = a.q + row * a.q_stride;
  for (int64_t c = threadIdx.x; c < a.D; c += blockDim.x) q[c] = static_cast<int8_t>(quant(value(c)));
  const int pad = static_cast<int>((16 - (a.D & 15)) & 15);
  if (threadIdx.x < pad) q[a.D + threadIdx.x] = 0;
  if (threadIdx.x == 0) a.q_scale[row] = quant.scale;
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
  int w_f32;
};

// A CTA (or each of its warps) walks rows t, t + grid, ... and keeps its columns' share of dw in
// registers; the shares are added by rms_dw_kernel in a fixed order, so dw has the same bits from
// run to run.
template <int DT, int VE, int VPT, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : row_threads(VPT * VE)) rms_bwd_kernel(const RowBwdArgs a) {
  __shared__ float part_sum[2][32];
  using E = typename Elem<DT>::type;
  const int tid = threadIdx.x, nthr = WARP ? 32 : blockDim.x;
  const int nvec = static_cast<int>(a.D / VE);
  const int rows_per_cta = WARP ? blockDim.y : 1;
  float dw[VPT][VE];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[i][j] = 0.f;
  int flip = 0;  // two sets of partial sums: a row's first write never meets the last row's reads
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_cta + (WARP ? threadIdx.y : 0); row < a.T;
       row += static_cast<int64_t>(gridDim.x) * rows_per_cta, flip ^= 1) {
    const E* s = static_cast<const E*>(a.s) + row * a.s_stride;
    const E* dy = static_cast<const E*>(a.dy) + row * a.dy_stride;
    const E* ds = static_cast<const E*>(a.ds) + row * a.ds_stride;
    Vec<DT, VE> sv[VPT], gv[VPT], dv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
        sv[i].load(s, static_cast<int64_t>(c) * VE);
        gv[i].load(dy, static_cast<int64_t>(c) * VE);
        if (a.ds != nullptr) dv[i].load(ds, static_cast<int64_t>(c) * VE);
      }
    }
    const float rstd = a.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
        float xh[VE], g[VE], w[VE];
        sv[i].get(xh);
        gv[i].get(g);
        load_weight<DT, VE>(a.w, a.w_f32, static_cast<int64_t>(c) * VE, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float t = g[j] * (xh[j] * rstd);
          dw[i][j] += t;
          dot = fmaf(t, w[j], dot);
        }
      }
    }
    const float mean = row_sum<WARP>(dot, part_sum[flip]) / static_cast<float>(a.D);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
        float xh[VE], g[VE], w[VE], d[VE];
        sv[i].get(xh);
        gv[i].get(g);
        load_weight<DT, VE>(a.w, a.w_f32, static_cast<int64_t>(c) * VE, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) d[j] = 0.f;
        if (a.ds != nullptr) dv[i].get(d);
#pragma unroll
        for (int j = 0; j < VE; ++j) d[j] = fmaf(rstd, fmaf(-(xh[j] * rstd), mean, g[j] * w[j]), d[j]);
        Vec<DT, VE> out;
        out.set(d);
        out.store(static_cast<E*>(a.dx) + row * a.D, static_cast<int64_t>(c) * VE);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * a.D;
  if constexpr (WARP) {  // the CTA's warps, one after the other
    __shared__ float acc[32 * VPT * VE];
    for (int y = 0; y < blockDim.y; ++y) {
      if (threadIdx.y == y) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const int k = (i * 32 + tid) * VE + j;
            acc[k] = y == 0 ? dw[i][j] : acc[k] + dw[i][j];
          }
      }
      __syncthreads();
    }
    for (int k = threadIdx.y * 32 + tid; k < a.D; k += blockDim.y * 32) part[k] = acc[k];
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = i * nthr + tid;
      if (c < nvec) {
#pragma unroll
        for (int j = 0; j < VE; ++j) part[static_cast<int64_t>(c) * VE + j] = dw[i][j];
      }
    }
  }
}

// Rows too wide for registers: two passes over a row, dw gathered in this CTA's row of `part`.
template <int DT>
__global__ void __launch_bounds__(1024) rms_bwd_loop_kernel(const RowBwdArgs a) {
  __shared__ float part_sum[2][32];
  using E = typename Elem<DT>::type;
  float* part = a.part == nullptr ? nullptr : a.part + static_cast<int64_t>(blockIdx.x) * a.D;
  int flip = 0;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.T; row += gridDim.x, flip ^= 1) {
    const E* s = static_cast<const E*>(a.s) + row * a.s_stride;
    const E* dy = static_cast<const E*>(a.dy) + row * a.dy_stride;
    const float rstd = a.rstd[row];
    float dot = 0.f;
    for (int64_t c = threadIdx.x; c < a.D; c += blockDim.x) {
      float w;
      load_weight<DT, 1>(a.w, a.w_f32, c, &w);
      const float t = to_float<DT>(dy[c]) * (to_float<DT>(s[c]) * rstd);
      if (part != nullptr) part[c] = first ? t : part[c] + t;  // this thread alone has this column
      dot = fmaf(t, w, dot);
    }
    first = false;
    const float mean = row_sum<false>(dot, part_sum[flip]) / static_cast<float>(a.D);
    for (int64_t c = threadIdx.x; c < a.D; c += blockDim.x) {
      float w;
      load_weight<DT, 1>(a.w, a.w_f32, c, &w);
      const float d = a.ds == nullptr ? 0.f : to_float<DT>(static_cast<const E*>(a.ds)[row * a.ds_stride + c]);
      const float v = fmaf(rstd, fmaf(-(to_float<DT>(s[c]) * rstd), mean, to_float<DT>(dy[c]) * w), d);
      static_cast<E*>(a.dx)[row * a.D + c] = from_float<DT>(v);
    }
  }
}

// dw[c] = sum over the CTAs' shares: 8 warps take every 8th share of 32 columns each, then the
// eight sums are added in order.
__global__ void __launch_bounds__(256) rms_dw_kernel(const float* part, int shares, int64_t D, void* dw, int dt) {
  __shared__ float acc[8][32];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
  float sum = 0.f;
  if (c < D)
#pragma unroll 8
    for (int i = threadIdx.y; i < shares; i += 8) sum += part[static_cast<int64_t>(i) * D + c];
  acc[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y == 0 && c < D) {
#pragma unroll
    for (int y = 1; y < 8; ++y) sum += acc[y][threadIdx.x];
    store_scalar_from_float(dw, c, dt, sum);
  }
}

// ---- 8-bit rows back to floating point --------------------------------------------------------
template <int DT>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out,
                                                         int64_t T, int64_t D, int vec) {
  using E = typename Elem<DT>::type;
  constexpr int VE = Elem<DT>::kVec;
  const int64_t per_row = (D + VE - 1) / VE;
  const int64_t total = T * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row, c = (i - row * per_row) * VE;
    const float s = scale[row];
    const int8_t* p = q + row * q_stride + c;
    E* o = static_cast<E*>(out) + row * D + c;
    float f[VE];
    if (vec) {
#pragma unroll
      for (int j = 0; j < VE; j += 4) unpack_int8(*reinterpret_cast<const uint32_t*>(p + j), f + j);
#pragma unroll
      for (int j = 0; j < VE; ++j) f[j] *= s;
      *reinterpret_cast<uint4*>(o) = pack16<DT>(f);
    } else {
      for (int j = 0; j < VE && c + j < D; ++j) o[j] = from_float<DT>(static_cast<float>(p[j]) * s);
    }
  }
}

// ---- host side ------------------------------------------------------------------------------
// How a row is split: 16-byte vectors where widths, strides and addresses allow, else single
// elements; a warp per row while a row fits 32 threads, else a CTA. A CTA takes four vectors a
// thread when there are rows enough to fill the GPU (more loads in flight per thread), one or two
// when there are not (the latency of a single row falls with the vectors per thread).
struct RowShape {
  bool vec, warp, loop;
  int vpt, threads;
};
static RowShape row_shape(bool vec, int64_t D, int64_t T, int dtype) {
  RowShape s{vec, false, false, 0, 0};
  const int ve = vec ? 16 / dtype_size(dtype) : 1;
  const int most = vec ? (dtype == FMOE_F32 ? 8 : 4) : 16;  // vectors a thread can hold: 32 elements, or 16 single ones
  const int64_t nvec = D / ve;
  if (nvec <= 32 * (vec ? 4 : 16)) {
    s.warp = true;
    s.threads = 32;
    s.vpt = vec ? (nvec <= 32 ? 1 : nvec <= 64 ? 2 : 4) : 16;
    return s;
  }
  s.vpt = T <= 2 * kNumSMs ? (vec ? 1 : 4) : (vec ? 4 : 16);
  while (s.vpt <= most && (nvec + s.vpt - 1) / s.vpt > row_threads(s.vpt * ve)) s.vpt *= vec ? 2 : 4;
  s.loop = s.vpt > most;
  s.threads = static_cast<int>(((nvec + s.vpt - 1) / s.vpt + 31) / 32 * 32);
  return s;
}

template <int DT, bool NORM>
static int launch_rows(const RowArgs& a, const RowShape& s, cudaStream_t st) {
  constexpr int V = Elem<DT>::kVec;
  const dim3 block = s.warp ? dim3(32, a.T >= 8 * kNumSMs ? 8 : 1) : dim3(s.threads);
  const unsigned grid = static_cast<unsigned>(s.warp ? (a.T + block.y - 1) / block.y : a.T);
#define FMOE_ROWS(VE, VPT, WARP) row_kernel<DT, VE, VPT, WARP, NORM><<<grid, block, 0, st>>>(a)
  if (s.loop) row_loop_kernel<DT, NORM><<<grid, 1024, 0, st>>>(a);
  else if (!s.vec && s.warp) FMOE_ROWS(1, 16, true);
  else if (!s.vec && s.vpt == 4) FMOE_ROWS(1, 4, false);
  else if (!s.vec) FMOE_ROWS(1, 16, false);
  else if (s.warp && s.vpt == 1) FMOE_ROWS(V, 1, true);
  else if (s.warp && s.vpt == 2) FMOE_ROWS(V, 2, true);
  else if (s.warp) FMOE_ROWS(V, 4, true);
  else if (s.vpt == 1) FMOE_ROWS(V, 1, false);
  else if (s.vpt == 2) FMOE_ROWS(V, 2, false);
  else if (s.vpt == 4) FMOE_ROWS(V, 4, false);
  else if constexpr (V == 4) FMOE_ROWS(V, 8, false);
#undef FMOE_ROWS
  return check_launch(NORM ? "row_kernel (norm)" : "row_kernel (quantize)");
}

template <int DT>
static int launch_bwd(const RowBwdArgs& a, const RowShape& s, int grid, cudaStream_t st) {
  constexpr int V = Elem<DT>::kVec;
  const dim3 block = s.warp ? dim3(32, 8) : dim3(s.threads);
#define FMOE_ROWS(VE, VPT, WARP) rms_bwd_kernel<DT, VE, VPT, WARP><<<grid, block, 0, st>>>(a)
  if (s.loop) rms_bwd_loop_kernel<DT><<<grid, 1024, 0, st>>>(a);
  else if (!s.vec && s.warp) FMOE_ROWS(1, 16, true);
  else if (!s.vec && s.vpt == 4) FMOE_ROWS(1, 4, false);
  else if (!s.vec) FMOE_ROWS(1, 16, false);
  else if (s.warp && s.vpt == 1) FMOE_ROWS(V, 1, true);
  else if (s.warp && s.vpt == 2) FMOE_ROWS(V, 2, true);
  else if (s.warp) FMOE_ROWS(V, 4, true);
  else if (s.vpt == 1) FMOE_ROWS(V, 1, false);
  else if (s.vpt == 2) FMOE_ROWS(V, 2, false);
  else if (s.vpt == 4) FMOE_ROWS(V, 4, false);
  else if constexpr (V == 4) FMOE_ROWS(V, 8, false);
#undef FMOE_ROWS
  return check_launch("rms_bwd_kernel");
}

// CTAs of the backward pass, and so shares of dw: enough to fill the GPU, each with a few rows.
static int bwd_grid(int64_t T, int64_t D) {
  const int64_t per_sm = D <= 1024 ? 4 : D <= 2048 ? 8 : D <= 4096 ? 4 : 2;
  const int64_t rows = D <= 1024 ? (T + 7) / 8 : T;  // the narrowest rows run eight to a CTA
  const int64_t most = per_sm * kNumSMs;
  return static_cast<int>(rows < most ? (rows > 0 ? rows : 1) : most);
}

static bool rows16(const void* p, int64_t stride, int dtype) {
  return aligned_to(p, 16) && stride * dtype_size(dtype) % 16 == 0;
}

}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t r_stride, const void* w,
                             int w_dtype, void* y, void* sum, float* rstd, int8_t* q, int64_t q_stride, float* q_scale,
                             int64_t T, int64_t D, double eps, int dtype, void* stream) {
  FMOE_RANGE("fmoe_rms_norm");
  FMOE_REQUIRE(valid_dtype(dtype) && (w_dtype == dtype || w_dtype == FMOE_F32), FMOE_ERR_ARG,
               "fmoe_rms_norm: bad dtype (the weight is fp32 or of the rows' type)");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 31), FMOE_ERR_ARG, "fmoe_rms_norm: bad sizes");
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
  const bool vec = D % (16 / dtype_size(dtype)) == 0 && rows16(x, x_stride, dtype) && aligned_to(w, 16) &&
                   (!residual || (rows16(residual, r_stride, dtype) && aligned_to(sum, 16))) && (!y || aligned_to(y, 16));
  const RowArgs a{x, residual, w, y, sum, rstd, q, q_scale, T, D, x_stride, r_stride, q_stride, eps, w_dtype == FMOE_F32};
  const RowShape s = row_shape(vec, D, T, dtype);
  int rc = FMOE_OK;
  FMOE_DISPATCH_DTYPE(dtype, DT, rc = (launch_rows<DT, true>(a, s, static_cast<cudaStream_t>(stream))));
  return rc;
}

extern "C" int fmoe_quantize_rows(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* q_scale, int64_t T,
                                  int64_t D, int dtype, void* stream) {
  FMOE_RANGE("fmoe_quantize_rows");
  FMOE_REQUIRE(valid_dtype(dtype), FMOE_ERR_ARG, "fmoe_quantize_rows: bad dtype");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 31), FMOE_ERR_ARG, "fmoe_quantize_rows: bad sizes");
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(x && q && q_scale, FMOE_ERR_ARG, "fmoe_quantize_rows: null pointer argument");
  FMOE_REQUIRE(T == 1 || x_stride >= D, FMOE_ERR_ARG, "fmoe_quantize_rows: the row stride must be at least D");
  FMOE_REQUIRE(q_stride % 16 == 0 && q_stride >= D && aligned_to(q, 16), FMOE_ERR_ARG,
               "fmoe_quantize_rows: 8-bit rows must lie at 16-byte steps");
  const bool vec = D % (16 / dtype_size(dtype)) == 0 && rows16(x, x_stride, dtype);
  const RowArgs a{x, nullptr, nullptr, nullptr, nullptr, nullptr, q, q_scale, T, D, x_stride, 0, q_stride, 0.0, 0};
  const RowShape s = row_shape(vec, D, T, dtype);
  int rc = FMOE_OK;
  FMOE_DISPATCH_DTYPE(dtype, DT, rc = (launch_rows<DT, false>(a, s, static_cast<cudaStream_t>(stream))));
  return rc;
}

extern "C" int fmoe_dequantize_rows(const int8_t* q, int64_t q_stride, const float* q_scale, void* out, int64_t T, int64_t D,
                                    int dtype, void* stream) {
  FMOE_RANGE("fmoe_dequantize_rows");
  FMOE_REQUIRE(valid_dtype(dtype), FMOE_ERR_ARG, "fmoe_dequantize_rows: bad dtype");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 31), FMOE_ERR_ARG, "fmoe_dequantize_rows: bad sizes");
  if (T == 0) return FMOE_OK;
  FMOE_REQUIRE(q && q_scale && out, FMOE_ERR_ARG, "fmoe_dequantize_rows: null pointer argument");
  FMOE_REQUIRE(T == 1 || q_stride >= D, FMOE_ERR_ARG, "fmoe_dequantize_rows: the row stride must be at least D");
  const int ve = 16 / dtype_size(dtype);
  const int vec = D % ve == 0 && q_stride % 4 == 0 && aligned_to(q, 4) && aligned_to(out, 16);
  const int64_t total = T * ((D + ve - 1) / ve);
  const int64_t want = (total + 255) / 256, most = 16 * kNumSMs;
  const unsigned grid = static_cast<unsigned>(want < most ? want : most);
  FMOE_DISPATCH_DTYPE(dtype, DT, dequantize_kernel<DT><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
                                     q, q_stride, q_scale, out, T, D, vec));
  return check_launch("dequantize_kernel");
}

extern "C" size_t fmoe_rms_norm_bwd_bytes(int64_t T, int64_t D) {
  if (T <= 0 || D <= 0) return 0;
  return static_cast<size_t>(bwd_grid(T, D)) * static_cast<size_t>(D) * sizeof(float);
}

extern "C" int fmoe_rms_norm_bwd(const void* dy, int64_t dy_stride, const void* dsum, int64_t ds_stride, const void* sum,
                                 int64_t s_stride, const float* rstd, const void* w, int w_dtype, void* dx, void* dw,
                                 void* scratch, size_t scratch_bytes, int64_t T, int64_t D, int dtype, void* stream) {
  FMOE_RANGE("fmoe_rms_norm_bwd");
  FMOE_REQUIRE(valid_dtype(dtype) && (w_dtype == dtype || w_dtype == FMOE_F32), FMOE_ERR_ARG,
               "fmoe_rms_norm_bwd: bad dtype (the weight is fp32 or of the rows' type)");
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 31), FMOE_ERR_ARG, "fmoe_rms_norm_bwd: bad sizes");
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
  const bool vec = D % (16 / dtype_size(dtype)) == 0 && rows16(dy, dy_stride, dtype) && rows16(sum, s_stride, dtype) &&
                   (!dsum || rows16(dsum, ds_stride, dtype)) && aligned_to(w, 16) && aligned_to(dx, 16);
  const RowShape s = row_shape(vec, D, T, dtype);
  const int grid = bwd_grid(T, D);
  const RowBwdArgs a{dy, dsum, sum, rstd, w, dx, dw ? static_cast<float*>(scratch) : nullptr, T, D,
                     dy_stride, ds_stride, s_stride, w_dtype == FMOE_F32};
  int rc = FMOE_OK;
  FMOE_DISPATCH_DTYPE(dtype, DT, rc = (launch_bwd<DT>(a, s, grid, st)));
  if (rc != 0 || dw == nullptr) return rc;
  rms_dw_kernel<<<static_cast<unsigned>((D + 31) / 32), dim3(32, 8), 0, st>>>(static_cast<const float*>(scratch), grid, D, dw,
                                                                            w_dtype);
  return check_launch("rms_dw_kernel");
}
