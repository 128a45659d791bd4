// Matrix product in 8-bit integers on the 5th-generation tensor cores (tcgen05, kind::i8), dense or
// grouped by expert:
//   C[r, n] = act( (sum_k Aq[r, k] * Wq[e, n, k]) * sa[r] * sw[e, n] )     e = expert of row r
// Aq [R, K] int8 with a scale per row (token), Wq [E, N, K] int8 with a scale per row (output
// channel), C bf16 / fp16 / fp32. The sum is exact in 32-bit integers (|q| <= 128, K < 131072), so a
// result does not depend on how K is split or in which order parts arrive; the two scales are
// applied in fp32 and the result is rounded once.
//
// int8_gemm_kernel, per CTA (192 threads, one CTA per SM):
//   warp 0      TMA producer: A tile 128 x 128 bytes and W tile 256 x 128 bytes per stage, 128-byte
//               swizzle, 4 stages, mbarrier full/empty pairs; rows and columns past the ends of
//               the tensors read as zeros, so R, N and K need not be multiples of the tile
//   warp 1      MMA issuer: one thread issues tcgen05.mma (M=128, N=256, K=32, s8 x s8 -> s32) into
//               one of two 256-column TMEM accumulators
//   warps 2-5   epilogue: tcgen05.ld, integer -> float, scales, activation, stores of the valid
//               rows and columns while the next tile's MMAs fill the other accumulator
// Every mbarrier wait is bounded, as in grouped_gemm.cu.
#include "int8.cuh"
#include "tcgen05.cuh"

namespace fmoe {

extern int g_gemm_sms, g_gemm_skip_loads, g_gemm_spin_limit;

namespace i8 {

constexpr int kBM = 128, kBN = 256, kBK = 128, kStages = 4, kUmmaK = 32;
constexpr int kABytes = kBM * kBK;  // 16 KB
constexpr int kBBytes = kBN * kBK;  // 32 KB
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kThreads = 192;
constexpr int kEpiStageBytes = 4 * 32 * 128;  // one 32-row x 128-byte block per epilogue warp
constexpr int kMaxExperts = 1024;
constexpr int kRowGroup = 16;  // row blocks that share their column blocks' weight tiles, see locate()

struct Args {
  const int64_t* offsets;  // [E] first row of each expert; nullptr: one expert with all rows
  const int64_t* counts;
  const float* a_scale;    // [R]
  const float* w_scale;    // [E, N]
  void* C;                 // [R, cols]
  int64_t cols;            // N, or N / 2 for SwiGLU: also the row stride of C
  int64_t R, N;
  int E;
  int n_blocks;            // column tiles per expert
  int k_blocks;
  int act, out_dtype;
  int vec_ok;              // rows of C start on 16-byte boundaries
  int skip_loads;
  uint32_t spin_limit;
  int32_t* status;
};

// Instruction descriptor: D s32, A and B signed 8 bits, both K-major, M=128, N=256.
constexpr uint32_t kIdesc = (2u << 4) | (1u << 7) | (1u << 10) | ((kBN >> 3) << 17) | ((kBM >> 4) << 24);

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ int64_t rows_of(const Args& a, int e) {
  return a.offsets == nullptr ? a.R : expert_rows(a.offsets, a.counts, a.R, e);
}

struct Tile {
  int expert, nb, rows;
  int64_t row0;
};

// Tiles are numbered expert by expert; inside an expert in groups of kRowGroup row blocks, column
// block by column block, row block by row block. The tiles that run at the same time then touch
// about kRowGroup row blocks and 148 / kRowGroup column blocks: 36 MB of operands at K = 8192,
// which L2 holds, where one column block against all rows of a 32768-row matrix would stream
// 268 MB of rows per column block.
__device__ __forceinline__ Tile locate(int tile, const int* mb_prefix, const Args& a) {
  int lo = 0, hi = a.E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (static_cast<int64_t>(mb_prefix[mid]) * a.n_blocks <= tile) lo = mid; else hi = mid;
  }
  const int mblocks = mb_prefix[lo + 1] - mb_prefix[lo];
  int local = tile - mb_prefix[lo] * a.n_blocks;
  const int group = local / (kRowGroup * a.n_blocks);
  local -= group * kRowGroup * a.n_blocks;
  const int left = mblocks - group * kRowGroup;
  const int height = left < kRowGroup ? left : kRowGroup;
  Tile t;
  t.expert = lo;
  t.nb = local / height;
  const int64_t first = static_cast<int64_t>(group * kRowGroup + local - t.nb * height) * kBM;
  t.row0 = (a.offsets == nullptr ? 0 : a.offsets[lo]) + first;
  const int64_t rows = rows_of(a, lo) - first;
  t.rows = static_cast<int>(rows < kBM ? rows : kBM);
  return t;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                     const Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kStages * kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* tmem_full = empty + kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_base_slot + 1);
  uint64_t* drain = reinterpret_cast<uint64_t*>(abort_flag + 1);
  uint4* stage_buf = reinterpret_cast<uint4*>(smem + kStages * kStageBytes + 256);
  int* mb_prefix = reinterpret_cast<int*>(smem + kStages * kStageBytes + 256 + kEpiStageBytes);  // [E + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool swiglu = a.act == FMOE_ACT_SWIGLU;
  int fills = 0;
  bool mma_issued = false;

  // ---- set-up: tile table, barriers, TMEM ----------------------------------------------
  for (int e = threadIdx.x; e < a.E; e += kThreads) {
    const int64_t n = rows_of(a, e);
    if (a.counts != nullptr && n != a.counts[e] && a.counts[e] > 0 && a.status != nullptr && blockIdx.x == 0)
      atomicOr(a.status, FMOE_STATUS_BAD_EXPERT);  // rows past the end of A were cut off
    mb_prefix[e + 1] = static_cast<int>((n + kBM - 1) / kBM);
  }
  if (threadIdx.x == 0) {
    mb_prefix[0] = 0;
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], 4);
    }
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == 0) {  // inclusive scan of the per-expert block counts, 32 at a time
    int carry = 0;
    for (int base = 0; base < a.E; base += 32) {
      const int e = base + lane;
      int v = e < a.E ? mb_prefix[e + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += n;
      }
      if (e < a.E) mb_prefix[e + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_base_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int total_tiles = mb_prefix[a.E] * a.n_blocks;

  if (warp == 0 && lane == 0) {
    // ---- TMA producer ---------------------------------------------------------------
    int stage = 0;
    uint32_t phase = 0;
    for (int tile = blockIdx.x; tile < total_tiles && !a.skip_loads; tile += gridDim.x) {
      const Tile t = locate(tile, mb_prefix, a);
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, a.spin_limit)) goto timed_out;
        mbar_expect_tx(&full[stage], kStageBytes);
        tma_load_2d(smem_a + stage * kABytes, &map_a, kb * kBK, static_cast<int>(t.row0), &full[stage]);
        uint8_t* b = smem_b + stage * kBBytes;
        if (swiglu) {  // 128 gate rows, then the up rows of the same columns
          tma_load_3d(b, &map_w, kb * kBK, t.nb * 128, t.expert, &full[stage]);
          tma_load_3d(b + kBBytes / 2, &map_w, kb * kBK, static_cast<int>(a.cols) + t.nb * 128, t.expert, &full[stage]);
        } else {
          tma_load_3d(b, &map_w, kb * kBK, t.nb * kBN, t.expert, &full[stage]);
        }
        ++fills;
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1 && lane == 0) {
    // ---- MMA issuer -----------------------------------------------------------------
    int stage = 0;
    uint32_t phase = 0;
    int it = 0;
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++it) {
      const int acc = it & 1;
      if (!mbar_wait(&tmem_empty[acc], ((it >> 1) & 1) ^ 1, abort_flag, a.spin_limit)) goto timed_out;
      tcgen05_fence_after();
      const uint32_t tmem_d = tmem_base + acc * kBN;
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, a.spin_limit)) goto timed_out;
        tcgen05_fence_after();
        mma_issued = true;
        const uint64_t da = smem_desc(smem_u32(smem_a + stage * kABytes));
        const uint64_t db = smem_desc(smem_u32(smem_b + stage * kBBytes));
#pragma unroll
        for (int k = 0; k < kBK / kUmmaK; ++k)  // 32 bytes along K inside the swizzle atom: +2 encoded
          umma_i8(tmem_d, da + 2 * k, db + 2 * k, kIdesc, (kb | k) != 0 ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      umma_commit(&tmem_full[acc]);
    }
  } else if (warp >= 2) {
    // ---- epilogue -------------------------------------------------------------------
    using E = typename Elem<DT>::type;
    constexpr int kPiece = Elem<DT>::kVec;  // columns per 16 bytes of C
    constexpr int kChunk = 8 * kPiece;      // columns per 128-byte segment of a row of C: 64, or 32 in fp32
    const int quarter = warp & 3;
    uint4* stage_w = stage_buf + (warp - 2) * (32 * 8);
    const int out_cols = swiglu ? 128 : kBN;
    int it = 0;
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++it) {
      const int acc = it & 1;
      const Tile t = locate(tile, mb_prefix, a);
      const int row = quarter * 32 + lane;
      const int warp_rows = t.rows - quarter * 32;  // valid rows of this warp (may be <= 0)
      const float sa = row < t.rows ? a.a_scale[t.row0 + row] : 0.f;
      const float* sw = a.w_scale + static_cast<int64_t>(t.expert) * a.N;
      if (!mbar_wait(&tmem_full[acc], (it >> 1) & 1, abort_flag, a.spin_limit)) goto timed_out;
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + acc * kBN + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < out_cols && warp_rows > 0; c0 += kChunk) {
        const int64_t col0 = static_cast<int64_t>(t.nb) * out_cols + c0;
        const int cols = static_cast<int>(a.cols - col0 < kChunk ? a.cols - col0 : kChunk);
        if (cols <= 0) break;
#pragma unroll
        for (int h = 0; h < kChunk / 32; ++h) {
          float f[32];
          // lane j holds the channel scale of column 32 h + j and hands it round
          const int64_t mine = col0 + 32 * h + lane;
          const float s0 = mine < a.cols ? sw[mine] : 0.f;
          if (swiglu) {
            const float s1 = mine < a.cols ? sw[a.cols + mine] : 0.f;
            uint32_t g[32], u[32];
            tmem_ld32(taddr + c0 + 32 * h, g);
            tmem_ld32(taddr + 128 + c0 + 32 * h, u);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float gate = static_cast<float>(static_cast<int>(g[i])) * sa * __shfl_sync(0xffffffffu, s0, i);
              const float up = static_cast<float>(static_cast<int>(u[i])) * sa * __shfl_sync(0xffffffffu, s1, i);
              f[i] = silu(gate) * up;
            }
          } else {
            uint32_t r[32];
            tmem_ld32(taddr + c0 + 32 * h, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              f[i] = static_cast<float>(static_cast<int>(r[i])) * sa * __shfl_sync(0xffffffffu, s0, i);
            if (a.act == FMOE_ACT_GELU) {
#pragma unroll
              for (int i = 0; i < 32; ++i) f[i] = gelu_erf(f[i]);
            }
          }
#pragma unroll
          for (int v = 0; v < 32 / kPiece; ++v)
            stage_w[lane * 8 + (((32 / kPiece) * h + v) ^ (lane & 7))] = pack16<DT>(f + kPiece * v);
        }
        __syncwarp();
        // rows are regrouped through the swizzled staging block: four whole 128-byte segments a store
        const int q = lane & 7, left = cols - q * kPiece;
#pragma unroll
        for (int step = 0; step < 8; ++step) {
          const int r = step * 4 + (lane >> 3);
          if (r < warp_rows && left > 0) {
            const uint4 val = stage_w[r * 8 + (q ^ (r & 7))];
            E* p = static_cast<E*>(a.C) + (t.row0 + quarter * 32 + r) * a.cols + col0 + q * kPiece;
            if (a.vec_ok && left >= kPiece) {
              *reinterpret_cast<uint4*>(p) = val;
            } else {
              const E* from = reinterpret_cast<const E*>(&val);
#pragma unroll
              for (int j = 0; j < kPiece; ++j)
                if (j < left) p[j] = from[j];
            }
          }
        }
        __syncwarp();
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tmem_empty[acc]);
    }
  }
  goto done;

timed_out:
  *abort_flag = 1;
  if (a.status != nullptr) atomicOr(a.status, FMOE_STATUS_WAIT_TIMEOUT);

done:
  drain_on_exit(warp, lane, fills, mma_issued, full, drain, abort_flag, kStages, a.spin_limit);
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

// int8 tensor [depth, rows, cols] with the given strides in bytes (depth 1: [rows, cols]), box =
// 128 columns x box_rows rows, 128-byte swizzle; coordinates outside read as zeros.
static int make_map(CUtensorMap* map, const void* base, int64_t depth, int64_t rows, int64_t cols, int64_t row_stride,
                    int64_t depth_stride, int box_rows, int rank, const char* what) {
  if (const int rc = bind_context(); rc != 0) return rc;
  EncodeTiledFn fn = encode_tiled_fn();
  FMOE_REQUIRE(fn != nullptr, FMOE_ERR_DEVICE, "fmoe_int8_gemm: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(depth)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_stride), static_cast<cuuint64_t>(depth_stride)};
  const cuuint32_t box[3] = {kBK, static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, elem,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FMOE_REQUIRE(r == CUDA_SUCCESS, FMOE_ERR_ARG, "fmoe_int8_gemm: cuTensorMapEncodeTiled(%s) failed with %d", what,
               static_cast<int>(r));
  return FMOE_OK;
}

}  // namespace i8
}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_int8_gemm(const int8_t* a, int64_t a_stride, const float* a_scale, const int8_t* w, int64_t w_stride,
                              int64_t w_expert_stride, const float* w_scale, void* c, const int64_t* offsets,
                              const int64_t* counts, int64_t E, int64_t R, int64_t N, int64_t K, int activation,
                              int out_dtype, int32_t* status, void* stream) {
  FMOE_RANGE("fmoe_int8_gemm");
  FMOE_REQUIRE(activation >= FMOE_ACT_NONE && activation <= FMOE_ACT_GELU, FMOE_ERR_ARG,
               "fmoe_int8_gemm: activation must be FMOE_ACT_NONE, FMOE_ACT_SWIGLU or FMOE_ACT_GELU");
  FMOE_REQUIRE(valid_dtype(out_dtype), FMOE_ERR_ARG, "fmoe_int8_gemm: bad output dtype");
  FMOE_REQUIRE(E >= 0 && R >= 0 && N > 0 && K > 0, FMOE_ERR_ARG, "fmoe_int8_gemm: bad sizes");
  const bool swiglu = activation == FMOE_ACT_SWIGLU;
  FMOE_REQUIRE(!swiglu || N % 2 == 0, FMOE_ERR_ARG, "fmoe_int8_gemm: SwiGLU needs N = 2*ff, got N=%lld", (long long)N);
  FMOE_REQUIRE(E <= i8::kMaxExperts, FMOE_ERR_UNSUPPORTED, "fmoe_int8_gemm: supports E <= %d", i8::kMaxExperts);
  FMOE_REQUIRE(K < 131072, FMOE_ERR_UNSUPPORTED, "fmoe_int8_gemm: K=%lld could overflow the 32-bit sums (K < 131072)",
               (long long)K);
  FMOE_REQUIRE(R < (1ll << 31) && N < (1ll << 31) - 256, FMOE_ERR_UNSUPPORTED, "fmoe_int8_gemm: R and N must fit in int32");
  FMOE_REQUIRE((offsets == nullptr) == (counts == nullptr) && (offsets != nullptr || E <= 1), FMOE_ERR_ARG,
               "fmoe_int8_gemm: offsets and counts come together, and several experts need them");
  if (E == 0 || R == 0) return FMOE_OK;
  FMOE_REQUIRE(a && a_scale && w && w_scale && c, FMOE_ERR_ARG, "fmoe_int8_gemm: null pointer argument");
  FMOE_REQUIRE(aligned_to(a, 16) && aligned_to(w, 16) && a_stride % 16 == 0 && w_stride % 16 == 0 &&
                   w_expert_stride % 16 == 0 && a_stride >= K && w_stride >= K && (E == 1 || w_expert_stride >= w_stride),
               FMOE_ERR_ARG, "fmoe_int8_gemm: rows of a and w must lie at 16-byte steps of at least K");
  const int64_t cols = swiglu ? N / 2 : N;
  i8::Args g;
  g.offsets = offsets;
  g.counts = counts;
  g.a_scale = a_scale;
  g.w_scale = w_scale;
  g.C = c;
  g.cols = cols;
  g.R = R;
  g.N = N;
  g.E = static_cast<int>(E);
  g.n_blocks = static_cast<int>(swiglu ? (cols + 127) / 128 : (N + i8::kBN - 1) / i8::kBN);
  g.k_blocks = static_cast<int>((K + i8::kBK - 1) / i8::kBK);
  g.act = activation;
  g.out_dtype = out_dtype;
  g.vec_ok = aligned_to(c, 16) && cols * dtype_size(out_dtype) % 16 == 0;
  g.skip_loads = g_gemm_skip_loads;
  g.spin_limit = static_cast<uint32_t>(g_gemm_spin_limit);
  g.status = status;
  FMOE_REQUIRE((R / i8::kBM + E) * g.n_blocks < (1ll << 31), FMOE_ERR_UNSUPPORTED, "fmoe_int8_gemm: too many tiles");
  CUtensorMap map_a, map_w;
  int rc = i8::make_map(&map_a, a, 1, R, K, a_stride, R * a_stride, i8::kBM, 2, "A");
  if (rc != 0) return rc;
  rc = i8::make_map(&map_w, w, E, N, K, w_stride, E == 1 ? N * w_stride : w_expert_stride, swiglu ? 128 : i8::kBN, 3, "W");
  if (rc != 0) return rc;
  const int64_t max_tiles = ((R + i8::kBM - 1) / i8::kBM + E - 1) * g.n_blocks;
  const int grid = static_cast<int>(max_tiles < g_gemm_sms ? max_tiles : g_gemm_sms);
  const size_t smem = 1024 + static_cast<size_t>(i8::kStages) * i8::kStageBytes + 256 + i8::kEpiStageBytes +
                      sizeof(int) * (E + 2);
  const int smem_most = 1024 + i8::kStages * i8::kStageBytes + 256 + i8::kEpiStageBytes +
                        static_cast<int>(sizeof(int)) * (i8::kMaxExperts + 2);
  FMOE_DISPATCH_DTYPE(out_dtype, DT, {
    FMOE_CUDA(cudaFuncSetAttribute(i8::int8_gemm_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_most));
    i8::int8_gemm_kernel<DT><<<grid, i8::kThreads, smem, static_cast<cudaStream_t>(stream)>>>(map_a, map_w, g);
  });
  return check_launch("int8_gemm_kernel");
}
