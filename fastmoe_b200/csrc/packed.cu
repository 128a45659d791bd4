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
__device__ __forceinline__ void load8(const void* row, int c, int D, int vec, float* f) {
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
__device__ __forceinline__ void store8(void* row, int c, int D, int vec, const float* f) {
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
__device__ __forceinline__ void dequantise8(uint2 w, float s, float2* f) {
  const float2 s2 = make_float2(s, s);
  float t[8];
  unpack_int8(w.x, t);
  unpack_int8(w.y, t + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = mul2(make_float2(t[2 * j], t[2 * j + 1]), s2);
}

// Eight lanes share a group, sixteen columns each. FULL: whole groups in 16-byte vectors, four to a warp,
// without the questions that ragged rows ask per vector (the kernel is bound by its instructions).
template <int DT, bool FULL>
__global__ void __launch_bounds__(256) pack_kernel(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride,
                                                   float* scale, int total, int D, FastDiv groups, int vec) {
  using E = typename Elem<DT>::type;
  constexpr int VE = Elem<DT>::kVec;
  const int sub = threadIdx.x & 7;
  // the four groups of a warp stay in the loop together: the shuffles below need all 32 lanes
  for (int64_t g0 = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 5) * 4; g0 < total;
       g0 += static_cast<int64_t>(gridDim.x) * 32) {
    const int g = static_cast<int>(g0) + ((threadIdx.x >> 3) & 3);
    const bool live = FULL || g < total;
    const int row_of = live ? groups.div(g) : 0;
    const int64_t row = row_of;
    const int k = g - row_of * groups.d;
    const int c = k * kGroup + sub * 16;
    const E* p = static_cast<const E*>(x) + row * x_stride + c;
    uint4 v[16 / VE];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16 / VE; ++i) {
      if (FULL) {
        v[i] = ld_stream16(reinterpret_cast<const uint4*>(p + i * VE));
        continue;
      }
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
    top = top_bits<DT>(top);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const Quantiser quant(top);
    if (FULL || (live && c < q_stride)) {  // past D: zeros up to the 16-byte step
      float f[16];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 16 / VE; ++i) unpack16<DT>(v[i], f + i * VE);
      if constexpr (DT == FMOE_F32) quant.template operator()<16>(f, w);
      else quant.template from16<16>(f, w);
      st_stream16(reinterpret_cast<uint4*>(q + row * q_stride + c), make_uint4(w[0], w[1], w[2], w[3]));
    }
    if (live && sub == 0) scale[g] = quant.scale();
  }
}

template <int DT>
__global__ void __launch_bounds__(256) unpack_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out,
                                                     int total, int D, int groups, FastDiv per_row, int vec) {
  using E = typename Elem<DT>::type;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * 8;
    const int64_t row = row_of;
    float2 f[4];
    dequantise8(*reinterpret_cast<const uint2*>(q + row * q_stride + c), scale[row * groups + c / kGroup], f);
    store8<DT>(static_cast<E*>(out) + row * D, c, D, vec, reinterpret_cast<const float*>(f));
  }
}

// One thread: eight columns of the gate half and the same columns of the up half. A width that is not a multiple of eight leaves the up half's bytes off the 8-byte grid: they are read
// one by one.
template <int DT>
__global__ void __launch_bounds__(256) packed_swiglu_bwd_kernel(const int8_t* q, int64_t q_stride, const float* scale,
                                                                const void* grad, int64_t g_stride, void* grad_h,
                                                                void* hidden, int total, int ff, int groups,
                                                                FastDiv per_row, int vec) {
  using E = typename Elem<DT>::type;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * 8;
    const int64_t row = row_of;
    const int8_t* qr = q + row * q_stride;
    const float* sr = scale + row * groups;
    float2 gate[4], up[4], g[4], d[4], h[4];
    const uint2 qg = *reinterpret_cast<const uint2*>(qr + c);
    if (vec) {
      const uint2 qu = *reinterpret_cast<const uint2*>(qr + ff + c);
      load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, ff, 1, reinterpret_cast<float*>(g));
      dequantise8(qu, sr[(ff + c) / kGroup], up);
    } else {
      load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, ff, 0, reinterpret_cast<float*>(g));
      float* u = reinterpret_cast<float*>(up);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        u[j] = c + j < ff ? static_cast<float>(qr[ff + c + j]) * sr[(ff + c + j) / kGroup] : 0.f;
    }
    dequantise8(qg, sr[c / kGroup], gate);
    const float2 one = make_float2(1.f, 1.f), minus = make_float2(-1.f, -1.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 s = make_float2(sigmoid(gate[j].x), sigmoid(gate[j].y));
      const float2 act = mul2(gate[j], s);
      h[j] = mul2(act, up[j]);
      // d gate = grad up s (1 + gate (1 - s)),  d up = grad gate s
      d[j] = mul2(mul2(mul2(g[j], up[j]), s), fma2(gate[j], fma2(s, minus, one), one));
      up[j] = mul2(g[j], act);
    }
    E* out = static_cast<E*>(grad_h) + row * 2 * ff;
    store8<DT>(out, c, ff, vec, reinterpret_cast<const float*>(d));
    store8<DT>(out + ff, c, ff, vec, reinterpret_cast<const float*>(up));
    store8<DT>(static_cast<E*>(hidden) + row * ff, c, ff, vec, reinterpret_cast<const float*>(h));
  }
}

template <int DT>
__global__ void __launch_bounds__(256) packed_gelu_bwd_kernel(const int8_t* q, int64_t q_stride, const float* scale,
                                                              const void* grad, int64_t g_stride, void* grad_h,
                                                              void* hidden, int total, int D, int groups,
                                                              FastDiv per_row, int vec) {
  using E = typename Elem<DT>::type;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * 8;
    const int64_t row = row_of;
    float2 x2[4];
    float g[8], h[8];
    load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, D, vec, g);
    dequantise8(*reinterpret_cast<const uint2*>(q + row * q_stride + c), scale[row * groups + c / kGroup], x2);
    const float* x = reinterpret_cast<const float*>(x2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float bell;
      const float cdf = normal_cdf(x[j], &bell);
      h[j] = x[j] * cdf;
      g[j] *= cdf + x[j] * 0.39894228040143268f * bell;  // 1 / sqrt(2 pi)
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
  FMOE_REQUIRE(T >= 0 && D > 0 && T < (1ll << 31) && D < (1ll << 30), FMOE_ERR_ARG, name ": bad sizes");     \
  if (T == 0) return FMOE_OK;                                                                               \
  FMOE_REQUIRE(T * ((D + 7) / 8) < (1ll << 31) - 1024, FMOE_ERR_UNSUPPORTED, name ": too many values");    \
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
  const int64_t total = T * groups;
  const unsigned grid = stream_grid((total + 31) / 32);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool full = vec && D % kGroup == 0 && total % 4 == 0;
  FMOE_DISPATCH_DTYPE(dtype, DT, {
    if (full)
      pack_kernel<DT, true><<<grid, 256, 0, st>>>(x, x_stride, q, q_stride, scale, static_cast<int>(total),
                                                  static_cast<int>(D), FastDiv(groups), vec);
    else
      pack_kernel<DT, false><<<grid, 256, 0, st>>>(x, x_stride, q, q_stride, scale, static_cast<int>(total),
                                                   static_cast<int>(D), FastDiv(groups), vec);
  });
  return check_launch("pack_kernel");
}

extern "C" int fmoe_unpack_activation(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t T, int64_t D,
                                      int dtype, void* stream) {
  FMOE_RANGE("fmoe_unpack_activation");
  FMOE_PACKED_SIZES("fmoe_unpack_activation");
  FMOE_REQUIRE(out != nullptr, FMOE_ERR_ARG, "fmoe_unpack_activation: null pointer argument");
  const int vec = D % 8 == 0 && aligned_to(out, 16);
  FMOE_DISPATCH_DTYPE(dtype, DT, unpack_kernel<DT><<<stream_grid((T * ((D + 7) / 8) + 255) / 256), 256, 0,
                                                     static_cast<cudaStream_t>(stream)>>>(
      q, q_stride, scale, out, static_cast<int>(T * ((D + 7) / 8)), static_cast<int>(D), packed_groups(D), FastDiv((D + 7) / 8), vec));
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
  const int total = static_cast<int>(T * ((cols + 7) / 8));
  const FastDiv per_row((cols + 7) / 8);
  const unsigned grid = stream_grid((static_cast<int64_t>(total) + 255) / 256);
  const int groups = packed_groups(D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (swiglu) {
    FMOE_DISPATCH_DTYPE(dtype, DT, packed_swiglu_bwd_kernel<DT><<<grid, 256, 0, st>>>(q, q_stride, scale, grad, g_stride,
                                                                                    grad_h, hidden, total, static_cast<int>(cols), groups,
                                                                                    per_row, vec));
  } else {
    FMOE_DISPATCH_DTYPE(dtype, DT, packed_gelu_bwd_kernel<DT><<<grid, 256, 0, st>>>(q, q_stride, scale, grad, g_stride,
                                                                                  grad_h, hidden, total, static_cast<int>(cols), groups,
                                                                                    per_row, vec));
  }
  return check_launch("packed_act_bwd_kernel");
}
