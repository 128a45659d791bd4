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

// Eight values of a row in 16-byte vectors.
template <int DT>
__device__ __forceinline__ void load8(const void* row, int c, float* f) {
  const typename Elem<DT>::type* p = static_cast<const typename Elem<DT>::type*>(row) + c;
#pragma unroll
  for (int j = 0; j < 8; j += Elem<DT>::kVec) unpack16<DT>(ld_stream16(reinterpret_cast<const uint4*>(p + j)), f + j);
}
template <int DT>
__device__ __forceinline__ void store8(void* row, int c, const float* f) {
  typename Elem<DT>::type* p = static_cast<typename Elem<DT>::type*>(row) + c;
#pragma unroll
  for (int j = 0; j < 8; j += Elem<DT>::kVec) st_stream16(reinterpret_cast<uint4*>(p + j), pack16<DT>(f + j));
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

// Each kernel below comes in two forms. Vectors: widths and addresses that allow 16-byte accesses, eight or
// sixteen columns to a thread. Columns: any width; a warp takes 128 columns of a row, a lane every 32nd
// of them, so that each access of a warp is one contiguous piece wherever the row starts. (Eight
// neighbouring columns to a lane, read one by one, took 49 us for 5122 x 1189 fp32 in the GELU derivative.)

// Vectors: eight lanes share a group, sixteen columns each, four groups to a warp. RAGGED: a width that is
// a multiple of 16 but not of 128, or groups that do not fill the last warp.
template <int DT, bool RAGGED>
__global__ void __launch_bounds__(256) pack_kernel(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride,
                                                   float* scale, int total, int D, FastDiv groups) {
  using E = typename Elem<DT>::type;
  constexpr int VE = Elem<DT>::kVec;
  const int sub = threadIdx.x & 7;
  // the four groups of a warp stay in the loop together: the shuffles below need all 32 lanes
  for (int64_t g0 = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 5) * 4; g0 < total;
       g0 += static_cast<int64_t>(gridDim.x) * 32) {
    const int g = static_cast<int>(g0) + ((threadIdx.x >> 3) & 3);
    const int row_of = !RAGGED || g < total ? groups.div(g) : 0;
    const int64_t row = row_of;
    const int c = (g - row_of * groups.d) * kGroup + sub * 16;
    const bool live = !RAGGED || (g < total && c < D);
    const E* p = static_cast<const E*>(x) + row * x_stride + c;
    uint4 v[16 / VE];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16 / VE; ++i) v[i] = live ? ld_stream16(reinterpret_cast<const uint4*>(p + i * VE)) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 16 / VE; ++i) top = vec_top<DT>(v[i], top);
    top = top_bits<DT>(top);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const Quantiser quant(top);
    if (live) {
      float f[16];
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 16 / VE; ++i) unpack16<DT>(v[i], f + i * VE);
      if constexpr (DT == FMOE_F32) quant.template operator()<16>(f, w);
      else quant.template from16<16>(f, w);
      st_stream16(reinterpret_cast<uint4*>(q + row * q_stride + c), make_uint4(w[0], w[1], w[2], w[3]));
      if (sub == 0) scale[g] = quant.scale();
    }
  }
}

constexpr int kPackAhead = 4;  // groups a warp has loads in flight for

template <int DT>
__global__ void __launch_bounds__(256) pack_columns_kernel(const void* x, int64_t x_stride, int8_t* q, int64_t q_stride,
                                                           float* scale, int total, int D, FastDiv groups) {
  using E = typename Elem<DT>::type;
  const int lane = threadIdx.x & 31;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), warps = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t g0 = warp * kPackAhead; g0 < total; g0 += warps * kPackAhead) {
    float f[kPackAhead][4];
#pragma unroll
    for (int u = 0; u < kPackAhead; ++u) {
      const int g = static_cast<int>(g0) + u, row = g < total ? groups.div(g) : 0, c = (g - row * groups.d) * kGroup + lane;
      const E* p = static_cast<const E*>(x) + static_cast<int64_t>(row) * x_stride + c;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[u][j] = g < total && c + 32 * j < D ? to_float<DT>(p[32 * j]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kPackAhead; ++u) {
      const int g = static_cast<int>(g0) + u;
      if (g >= total) break;  // the whole warp
      const int row = groups.div(g), c = (g - row * groups.d) * kGroup + lane;
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, abs_bits(f[u][j]));
      const Quantiser quant(__reduce_max_sync(0xffffffffu, top));
      uint32_t w;
      if constexpr (DT == FMOE_F32) quant.template operator()<4>(f[u], &w);
      else quant.template from16<4>(f[u], &w);
      int8_t* out = q + static_cast<int64_t>(row) * q_stride + c;
#pragma unroll
      for (int j = 0; j < 4; ++j)  // past D: zeros up to the 16-byte step
        if (c + 32 * j < q_stride) out[32 * j] = static_cast<int8_t>(w >> (8 * j));
      if (lane == 0) scale[g] = quant.scale();
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(256) unpack_kernel(const int8_t* q, int64_t q_stride, const float* scale, void* out,
                                                     int total, int D, int groups, FastDiv per_row) {
  using E = typename Elem<DT>::type;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * 8;
    const int64_t row = row_of;
    float2 f[4];
    dequantise8(*reinterpret_cast<const uint2*>(q + row * q_stride + c), scale[row * groups + c / kGroup], f);
    store8<DT>(static_cast<E*>(out) + row * D, c, reinterpret_cast<const float*>(f));
  }
}

// The 128 columns from `block` on of a row, four to a lane: calls f(row, c) for each.
template <typename F>
__device__ __forceinline__ void for_columns(int total, int cols, const FastDiv& blocks, F f) {
  const int64_t warps = static_cast<int64_t>(gridDim.x) * 8;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); b < total; b += warps) {
    const int row = blocks.div(static_cast<int>(b));
    const int c0 = (static_cast<int>(b) - row * blocks.d) * kGroup + (threadIdx.x & 31);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + 32 * j < cols) f(static_cast<int64_t>(row), c0 + 32 * j);
  }
}

template <int DT>
__global__ void __launch_bounds__(256) unpack_columns_kernel(const int8_t* __restrict__ q, int64_t q_stride,
                                                             const float* __restrict__ scale, void* __restrict__ out, int total,
                                                             int D, int groups, FastDiv blocks) {
  typename Elem<DT>::type* o = static_cast<typename Elem<DT>::type*>(out);
  for_columns(total, D, blocks, [&](int64_t row, int c) {
    o[row * D + c] = from_float<DT>(static_cast<float>(q[row * q_stride + c]) * scale[row * groups + c / kGroup]);
  });
}

// One value each, as in the vector kernels.
__device__ __forceinline__ void swiglu_bwd(float gate, float up, float g, float* d_gate, float* d_up, float* hidden) {
  const float s = sigmoid(gate), act = gate * s;
  *hidden = act * up;
  *d_gate = g * up * s * fmaf(gate, 1.f - s, 1.f);
  *d_up = g * act;
}
__device__ __forceinline__ void gelu_bwd(float x, float g, float* d, float* hidden) {
  float bell;
  const float cdf = normal_cdf(x, &bell);
  *hidden = x * cdf;
  *d = g * (cdf + x * 0.39894228040143268f * bell);  // 1 / sqrt(2 pi)
}

// Vectors: eight columns of the gate half and the same columns of the up half to a thread.
template <int DT>
__global__ void __launch_bounds__(256) packed_swiglu_bwd_kernel(const int8_t* q, int64_t q_stride, const float* scale,
                                                                const void* grad, int64_t g_stride, void* grad_h,
                                                                void* hidden, int total, int ff, int groups,
                                                                FastDiv per_row) {
  using E = typename Elem<DT>::type;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * 8;
    const int64_t row = row_of;
    const int8_t* qr = q + row * q_stride;
    const float* sr = scale + row * groups;
    float2 gate[4], up[4], g[4], d[4], h[4];
    const uint2 qg = *reinterpret_cast<const uint2*>(qr + c), qu = *reinterpret_cast<const uint2*>(qr + ff + c);
    load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, reinterpret_cast<float*>(g));
    dequantise8(qu, sr[(ff + c) / kGroup], up);
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
    store8<DT>(out, c, reinterpret_cast<const float*>(d));
    store8<DT>(out + ff, c, reinterpret_cast<const float*>(up));
    store8<DT>(static_cast<E*>(hidden) + row * ff, c, reinterpret_cast<const float*>(h));
  }
}
template <int DT>
__global__ void __launch_bounds__(256)
    packed_swiglu_bwd_columns_kernel(const int8_t* __restrict__ q, int64_t q_stride, const float* __restrict__ scale,
                                     const void* __restrict__ grad, int64_t g_stride, void* __restrict__ grad_h,
                                     void* __restrict__ hidden, int total, int ff, int groups, FastDiv blocks) {
  using E = typename Elem<DT>::type;
  for_columns(total, ff, blocks, [&](int64_t row, int c) {
    const int8_t* qr = q + row * q_stride;
    const float* sr = scale + row * groups;
    const float gate = static_cast<float>(qr[c]) * sr[c / kGroup];
    const float up = static_cast<float>(qr[ff + c]) * sr[(ff + c) / kGroup];
    float d_gate, d_up, h;
    swiglu_bwd(gate, up, to_float<DT>(static_cast<const E*>(grad)[row * g_stride + c]), &d_gate, &d_up, &h);
    static_cast<E*>(grad_h)[row * 2 * ff + c] = from_float<DT>(d_gate);
    static_cast<E*>(grad_h)[row * 2 * ff + ff + c] = from_float<DT>(d_up);
    static_cast<E*>(hidden)[row * ff + c] = from_float<DT>(h);
  });
}

template <int DT>
__global__ void __launch_bounds__(256) packed_gelu_bwd_kernel(const int8_t* q, int64_t q_stride, const float* scale,
                                                              const void* grad, int64_t g_stride, void* grad_h,
                                                              void* hidden, int total, int D, int groups,
                                                              FastDiv per_row) {
  using E = typename Elem<DT>::type;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int row_of = per_row.div(static_cast<int>(i)), c = (static_cast<int>(i) - row_of * per_row.d) * 8;
    const int64_t row = row_of;
    float2 x2[4];
    float g[8], h[8];
    load8<DT>(static_cast<const E*>(grad) + row * g_stride, c, g);
    dequantise8(*reinterpret_cast<const uint2*>(q + row * q_stride + c), scale[row * groups + c / kGroup], x2);
    const float* x = reinterpret_cast<const float*>(x2);
#pragma unroll
    for (int j = 0; j < 8; ++j) gelu_bwd(x[j], g[j], &g[j], &h[j]);
    store8<DT>(static_cast<E*>(grad_h) + row * D, c, g);
    store8<DT>(static_cast<E*>(hidden) + row * D, c, h);
  }
}
template <int DT>
__global__ void __launch_bounds__(256)
    packed_gelu_bwd_columns_kernel(const int8_t* __restrict__ q, int64_t q_stride, const float* __restrict__ scale,
                                   const void* __restrict__ grad, int64_t g_stride, void* __restrict__ grad_h,
                                   void* __restrict__ hidden, int total, int D, int groups, FastDiv blocks) {
  using E = typename Elem<DT>::type;
  for_columns(total, D, blocks, [&](int64_t row, int c) {
    const float x = static_cast<float>(q[row * q_stride + c]) * scale[row * groups + c / kGroup];
    float d, h;
    gelu_bwd(x, to_float<DT>(static_cast<const E*>(grad)[row * g_stride + c]), &d, &h);
    static_cast<E*>(grad_h)[row * D + c] = from_float<DT>(d);
    static_cast<E*>(hidden)[row * D + c] = from_float<DT>(h);
  });
}

// Several rounds of CTAs rather than one or two that walk the tensor in step: SwiGLU derivative 65536 x 4096 bf16
// 228 us with 16 CTAs to an SM, 212 with 64, 214 with 256; GELU fp32 867 and 722. Packing 16-bit values, which is bound
// by its instructions, does not gain: 22.8 us for 8192 x 4096, 24.6 with 64 (fp32 65536 x 4096 236 and 216).
static unsigned stream_grid(int64_t blocks, int per_sm = 64) {
  const int64_t most = static_cast<int64_t>(per_sm) * kNumSMs;
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
  const int64_t total = T * groups;
  const bool vec = D % 16 == 0 && aligned_to(x, 16) && x_stride * dtype_size(dtype) % 16 == 0;
  const bool whole = D % kGroup == 0 && total % 4 == 0;
  const unsigned vec_grid = stream_grid((total + 31) / 32, dtype == FMOE_F32 ? 64 : 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FMOE_DISPATCH_DTYPE(dtype, DT, {
    if (vec && whole)
      pack_kernel<DT, false><<<vec_grid, 256, 0, st>>>(x, x_stride, q, q_stride, scale, static_cast<int>(total),
                                                       static_cast<int>(D), FastDiv(groups));
    else if (vec)
      pack_kernel<DT, true><<<vec_grid, 256, 0, st>>>(x, x_stride, q, q_stride, scale, static_cast<int>(total),
                                                      static_cast<int>(D), FastDiv(groups));
    else
      pack_columns_kernel<DT><<<stream_grid((total + 8 * kPackAhead - 1) / (8 * kPackAhead)), 256, 0, st>>>(
          x, x_stride, q, q_stride, scale, static_cast<int>(total), static_cast<int>(D), FastDiv(groups));
  });
  return check_launch("pack_kernel");
}

extern "C" int fmoe_unpack_activation(const int8_t* q, int64_t q_stride, const float* scale, void* out, int64_t T, int64_t D,
                                      int dtype, void* stream) {
  FMOE_RANGE("fmoe_unpack_activation");
  FMOE_PACKED_SIZES("fmoe_unpack_activation");
  FMOE_REQUIRE(out != nullptr, FMOE_ERR_ARG, "fmoe_unpack_activation: null pointer argument");
  const bool vec = D % 8 == 0 && aligned_to(out, 16);
  const int groups = packed_groups(D);
  const int64_t total = T * (vec ? D / 8 : groups);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FMOE_DISPATCH_DTYPE(dtype, DT, {
    if (vec)
      unpack_kernel<DT><<<stream_grid((total + 255) / 256), 256, 0, st>>>(q, q_stride, scale, out, static_cast<int>(total),
                                                                          static_cast<int>(D), groups, FastDiv(D / 8));
    else
      unpack_columns_kernel<DT><<<stream_grid((total + 7) / 8), 256, 0, st>>>(
          q, q_stride, scale, out, static_cast<int>(total), static_cast<int>(D), groups, FastDiv(groups));
  });
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
  const bool vec = cols % 8 == 0 && aligned_to(grad, 16) && g_stride * dtype_size(dtype) % 16 == 0 && aligned_to(grad_h, 16) &&
                   aligned_to(hidden, 16);
  const int64_t per_row = vec ? cols / 8 : (cols + kGroup - 1) / kGroup;
  const int total = static_cast<int>(T * per_row), width = static_cast<int>(cols), groups = packed_groups(D);
  const FastDiv div(per_row);
  const unsigned grid = stream_grid(vec ? (static_cast<int64_t>(total) + 255) / 256 : (static_cast<int64_t>(total) + 7) / 8);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define FMOE_PACKED_BWD(kernel) \
  kernel<DT><<<grid, 256, 0, st>>>(q, q_stride, scale, grad, g_stride, grad_h, hidden, total, width, groups, div)
  FMOE_DISPATCH_DTYPE(dtype, DT, {
    if (swiglu && vec) FMOE_PACKED_BWD(packed_swiglu_bwd_kernel);
    else if (swiglu) FMOE_PACKED_BWD(packed_swiglu_bwd_columns_kernel);
    else if (vec) FMOE_PACKED_BWD(packed_gelu_bwd_kernel);
    else FMOE_PACKED_BWD(packed_gelu_bwd_columns_kernel);
  });
#undef FMOE_PACKED_BWD
  return check_launch("packed_act_bwd_kernel");
}
