// Activations kept in 8 bits for the backward pass, and the activation derivatives that read them.
// A row's columns are split into groups of 128 (the last one may be short); a group is held as
// int8 values with one fp32 scale (int8.cuh): 1.03 bytes per value instead of 2 or 4.
//   pack     h -> q, scale
//   unpack   h~ = q * scale
//   SwiGLU   from h~ = [gate | up] and grad: d_gate, d_up, and hidden = silu(gate) * up again,
//            which the down projection's weight gradient needs and the forward need not keep
//   GELU     the same for hidden = gelu(h~)
// All are single streaming passes bound by HBM.
#include "int8.cuh"
#include "tcgen05.cuh"

namespace fmoe {

constexpr int kGroup = 128;

// f[0..8) of a row from column c on (zeros past D).
template <int DT>
__device__ __forceinline__ void load8(const void* row, int64_t c, int64_t D, int vec, float* f) {
  using E = typename Elem<DT>::type;
  const E* p = static_cast<const E*>(row) + c;
  if (vec) {
#pragma unroll
    for (int j = 0; j < 8; j += Elem<DT>::kVec) unpack16<DT>(ld_stream16(reinterpret_cast<const uint4*>(p + j)), f + j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = c + j < D ? to_float<DT>(p[j]) : 0.f;
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* row, int64_t c, int64_t D, int vec, const float* f) {
  using E = typename Elem<DT>::type;
  E* p = static_cast<E*>(row) + c;
  if (vec) {
#pragma unroll
    for (int j = 0; j < 8; j += Elem<DT>::kVec) st_stream16(reinterpret_cast<uint4*>(p + j), pack16<DT>(f + j));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < D) p[j] = from_float<DT>(f[j]);
  }
}
// Eight packed values from column c on, as floats; rows of q lie at 16-byte steps with zeros up to
// the next step, so eight bytes from a multiple of eight are always there.
__device__ __forceinline__ void load8_packed(const int8_t* row, int64_t c, float s, float* f) {
  const uint2 w = *reinterpret_cast<const uint2*>(row + c);
  unpack_int8(w.x, f);
  unpack_int8(w.y, f + 4);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= s;
}

// Eight lanes share a group, sixteen columns each.
template <int DT>
__global__ void __launch_bounds__(256) pack_kernel(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride,
                                                   float* scale, int64_t T, int64_t D, int groups, int vec) {
  using E = typename Elem<DT>::type;
  constexpr int VE = Elem<DT>::kVec;
  const int64_t total = T * groups;
  const int sub = threadIdx.x & 7;
  // the four groups of a warp stay in the loop together: the shuffles below need all 32 lanes
  for (int64_t g0 = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 5) * 4; g0 < total;
       g0 += static_cast<int64_t>(gridDim.x) * 32) {
    const int64_t g = g0 + ((threadIdx.x >> 3) & 3);
    const bool live = g < total;
    const int64_t row = live ? g / groups : 0;
    const int k = static_cast<int>(g - row * groups);
    const int64_t c = static_cast<int64_t>(k) * kGroup + sub * 16;
    const E* p = static_cast<const E*>(x) + row * x_stride + c;
    uint4 v[16 / VE];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16 / VE; ++i) {
      v[i] = make_uint4(0, 0, 0, 0);
      if (live && c + i * VE < D) {
        if (vec) {
          v[i] = ld_stream16(reinterpret_cast<const uint4*>(p + i * VE));
        } else {
          float f[VE];
#pragma unroll
          for (int j = 0; j < VE; ++j) f[j] = c + i * VE + j < D ? to_float<DT>(p[i * VE + j]) : 0.f;
          v[i] = pack16<DT>(f);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 16 / VE; ++i) top = vec_top<DT>(v[i], top);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const Quantiser quant(top);
    if (live && c < q_stride) {  // past D: zeros up to the 16-byte step
      float f[16];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 16 / VE; ++i) unpack16<DT>(v[i], f + i * VE);
      quant.operator()<16>(f, w);
      st_stream16(reinterpret_cast<uint4*>(q + row * q_stride + c), make_uint4(w[0], w[1], w[2], w[3]));
    }
    if (live && sub == 0) scale[row * groups + k] = quant.scale;
  }
}

template <int DT>
__global__ void __launch_bounds__(256) unpack_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out,
                                                     int64_t T, int64_t D, int groups, int vec) {
  using E = typename Elem<DT>::type;
  const int64_t per_row = (D + 7) / 8, total = T * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row, c = (i - row * per_row) * 8;
    float f[8];
    load8_packed(q + row * q_stride, c, scale[row * groups + c / kGroup], f);
    store8<DT>(static_cast<E*>(out) + row * D, c, D, vec, f);
  }
}

// The fast exponential and quotient are off by (2 + |x|) and 2 steps of 2^-23: the result goes into
// products that are rounded to 16 bits, or held to a 32-bit bound that counts them.
__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// One thread: eight columns of the gate half and the same columns of the up half. A width that is
// not a multiple of eight leaves the up half's bytes off the 8-byte grid: they are read one by one.
template <int DT>
__global__ void __launch_bounds__(256) packed_swiglu_bwd_kernel(const int8_t* q, int64_t q_stride, const float* scale,
                                                                const void* grad, int64_t g_stride, void* grad_h,
                                                                void* hidden, int64_t T, int64_t ff, int groups, int vec) {
  using E = typename Elem<DT>::type;
  const int64_t per_row = (ff + 7) / 8, total = T * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row, c = (i - row * per_row) * 8;
    const int8_t* qr = q + row * q_stride;
    const float* sr = scale + row * groups;
    float gate[8], up[8], g[8], d[8], h[8];
    load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, ff, vec, g);
    load8_packed(qr, c, sr[c / kGroup], gate);
    if (vec) {
      load8_packed(qr, ff + c, sr[(ff + c) / kGroup], up);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        up[j] = c + j < ff ? static_cast<float>(qr[ff + c + j]) * sr[(ff + c + j) / kGroup] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float s = sigmoid(gate[j]), act = gate[j] * s;
      h[j] = act * up[j];
      d[j] = g[j] * up[j] * s * (1.f + gate[j] * (1.f - s));
      up[j] = g[j] * act;
    }
    E* out = static_cast<E*>(grad_h) + row * 2 * ff;
    store8<DT>(out, c, ff, vec, d);
    store8<DT>(out + ff, c, ff, vec, up);
    store8<DT>(static_cast<E*>(hidden) + row * ff, c, ff, vec, h);
  }
}

template <int DT>
__global__ void __launch_bounds__(256) packed_gelu_bwd_kernel(const int8_t* q, int64_t q_stride, const float* scale,
                                                              const void* grad, int64_t g_stride, void* grad_h,
                                                              void* hidden, int64_t T, int64_t D, int groups, int vec) {
  using E = typename Elem<DT>::type;
  const int64_t per_row = (D + 7) / 8, total = T * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / per_row, c = (i - row * per_row) * 8;
    float x[8], g[8], h[8];
    load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, D, vec, g);
    load8_packed(q + row * q_stride, c, scale[row * groups + c / kGroup], x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float cdf = 0.5f * (1.f + erff(x[j] * 0.70710678118654752f));
      h[j] = x[j] * cdf;
      g[j] *= cdf + x[j] * 0.39894228040143268f * __expf(-0.5f * x[j] * x[j]);  // 1 / sqrt(2 pi)
    }
    store8<DT>(static_cast<E*>(grad_h) + row * D, c, D, vec, g);
    store8<DT>(static_cast<E*>(hidden) + row * D, c, D, vec, h);
  }
}

static unsigned stream_grid(int64_t blocks) {
  const int64_t most = 16 * kNumSMs;
  return static_cast<unsigned>(blocks < most ? blocks : most);
}
static int packed_groups(int64_t D) { return static_cast<int>((D + kGroup - 1) / kGroup); }

}  // namespace fmoe

using namespace fmoe;

#define FMOE_PACKED_SIZES(name)                                                                             \
  FMOE_REQUIRE(valid_dtype(dtype), FMOE_ERR_ARG, name ": bad dtype");                                       \
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 31), FMOE_ERR_ARG, name ": bad sizes");     \
  if (T == 0) return FMOE_OK;                                                                               \
  FMOE_REQUIRE(q && scale, FMOE_ERR_ARG, name ": null pointer argument");                                   \
  FMOE_REQUIRE(q_stride % 16 == 0 && q_stride >= D && q_stride < D + 16 && aligned_to(q, 16), FMOE_ERR_ARG, \
               name ": packed rows lie at 16-byte steps, the next one after D bytes")

extern "C" int fmoe_pack_activation(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride, float* scale, int64_t T,
                                    int64_t D, int dtype, void* stream) {
  FMOE_RANGE("fmoe_pack_activation");
  FMOE_PACKED_SIZES("fmoe_pack_activation");
  FMOE_REQUIRE(x != nullptr, FMOE_ERR_ARG, "fmoe_pack_activation: null pointer argument");
  FMOE_REQUIRE(T == 1 || x_stride >= D, FMOE_ERR_ARG, "fmoe_pack_activation: the row stride must be at least D");
  const int groups = packed_groups(D);
  const int vec = D % 8 == 0 && aligned_to(x, 16) && x_stride * dtype_size(dtype) % 16 == 0;
  FMOE_DISPATCH_DTYPE(dtype, DT, pack_kernel<DT><<<stream_grid((T * groups + 31) / 32), 256, 0,
                                                   static_cast<cudaStream_t>(stream)>>>(x, x_stride, q, q_stride, scale, T,
                                                                                        D, groups, vec));
  return check_launch("pack_kernel");
}

extern "C" int fmoe_unpack_activation(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t T, int64_t D,
                                      int dtype, void* stream) {
  FMOE_RANGE("fmoe_unpack_activation");
  FMOE_PACKED_SIZES("fmoe_unpack_activation");
  FMOE_REQUIRE(out != nullptr, FMOE_ERR_ARG, "fmoe_unpack_activation: null pointer argument");
  const int vec = D % 8 == 0 && aligned_to(out, 16);
  FMOE_DISPATCH_DTYPE(dtype, DT, unpack_kernel<DT><<<stream_grid((T * ((D + 7) / 8) + 255) / 256), 256, 0,
                                                     static_cast<cudaStream_t>(stream)>>>(q, q_stride, scale, out, T, D,
                                                                                          packed_groups(D), vec));
  return check_launch("unpack_kernel");
}

extern "C" int fmoe_packed_act_bwd(const int8_t* q, int64_t q_stride, const float* scale, const void* grad, int64_t g_stride,
                                   void* grad_h, void* hidden, int64_t T, int64_t D, int activation, int dtype,
                                   void* stream) {
  FMOE_RANGE("fmoe_packed_act_bwd");
  FMOE_PACKED_SIZES("fmoe_packed_act_bwd");
  FMOE_REQUIRE(activation == FMOE_ACT_SWIGLU || activation == FMOE_ACT_GELU, FMOE_ERR_ARG,
               "fmoe_packed_act_bwd: activation must be FMOE_ACT_SWIGLU or FMOE_ACT_GELU");
  FMOE_REQUIRE(grad && grad_h && hidden, FMOE_ERR_ARG, "fmoe_packed_act_bwd: null pointer argument");
  const bool swiglu = activation == FMOE_ACT_SWIGLU;
  FMOE_REQUIRE(!swiglu || D % 2 == 0, FMOE_ERR_ARG, "fmoe_packed_act_bwd: SwiGLU needs D = 2*ff");
  const int64_t cols = swiglu ? D / 2 : D;
  FMOE_REQUIRE(T == 1 || g_stride >= cols, FMOE_ERR_ARG, "fmoe_packed_act_bwd: grad's row stride is too small");
  const int vec = cols % 8 == 0 && aligned_to(grad, 16) && g_stride * dtype_size(dtype) % 16 == 0 && aligned_to(grad_h, 16) &&
                  aligned_to(hidden, 16);
  const unsigned grid = stream_grid((T * ((cols + 7) / 8) + 255) / 256);
  const int groups = packed_groups(D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (swiglu) {
    FMOE_DISPATCH_DTYPE(dtype, DT, packed_swiglu_bwd_kernel<DT><<<grid, 256, 0, st>>>(q, q_stride, scale, grad, g_stride,
                                                                                    grad_h, hidden, T, cols, groups, vec));
  } else {
    FMOE_DISPATCH_DTYPE(dtype, DT, packed_gelu_bwd_kernel<DT><<<grid, 256, 0, st>>>(q, q_stride, scale, grad, g_stride,
                                                                                  grad_h, hidden, T, cols, groups, vec));
  }
  return check_launch("packed_act_bwd_kernel");
}
