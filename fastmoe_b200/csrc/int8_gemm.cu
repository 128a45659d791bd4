// Matrix product in 8-bit integers on the 5th-generation tensor cores (tcgen05, kind::i8), dense or
// grouped by expert:
//   C[r, n] = act( (sum_k Aq[r, k] * Wq[e, n, k]) * sa[r] * sw[e, n] )     e = expert of row r
// Aq [R, K] int8 with a scale per row (token), Wq [E, N, K] int8 with a scale per row (output
// channel), C bf16 / fp16 / fp32. The sum is exact in 32-bit integers (|q| <= 128, K < 131072), so a
// result does not depend on how K is split or in which order parts arrive; the two scales are
// applied in fp32 and the result is rounded once.
//
// int8_gemm_kernel, per CTA (320 threads, one CTA per SM):
//   warp 0      TMA producer: A tile 128 x 128 bytes and W tile 256 x 128 bytes per stage, 128-byte
//               swizzle, 4 stages, mbarrier full/empty pairs; rows and columns past the ends of
//               the tensors read as zeros, so R, N and K need not be multiples of the tile
//   warp 1      MMA issuer: one thread issues tcgen05.mma (M=128, N=256, K=32, s8 x s8 -> s32) into
//               one of two 256-column TMEM accumulators
//   warps 2-9   epilogue: tcgen05.ld, integer -> float, scales, activation, stores of the valid
//               rows and columns while the next tile's MMAs fill the other accumulator
// Every mbarrier wait is bounded, as in grouped_gemm.cu.
#include "int8.cuh"
#include "tcgen05.cuh"

namespace fmoe {

extern int g_gemm_sms, g_gemm_skip_loads, g_gemm_spin_limit;

namespace i8 {

constexpr int kBM = 128, kBN = 256, kBK = 128, kUmmaK = 32;
constexpr int kABytes = kBM * kBK;  // 16 KB
constexpr int kPipeBytes = 4 * 48 * 1024;  // pipeline of int8_gemm_kernel: 4 stages, or 6 of a pair
constexpr int kThreads = 192;      // int8_tn_kernel
constexpr int kEpiWarps = 8;       // of int8_gemm_kernel: two per quarter of tensor memory, half of the columns each
constexpr int kTileThreads = 64 + 32 * kEpiWarps;
constexpr int kEpiStageBytes = kEpiWarps * 32 * 64;  // one 32-row x 64-byte block per epilogue warp
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

// Instruction descriptor: D s32, A and B signed 8 bits, both K-major, M=128 (256 for a pair), N=256.
constexpr uint32_t kIdesc = (2u << 4) | (1u << 7) | (1u << 10) | ((kBN >> 3) << 17) | ((kBM >> 4) << 24);
constexpr uint32_t kIdescPair = (2u << 4) | (1u << 7) | (1u << 10) | ((kBN >> 3) << 17) | ((2 * kBM >> 4) << 24);

// Programmatic dependent launch: a kernel launched so may start while the one before it in the stream ends;
// everything it reads or writes comes after this wait.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address, in the cluster's window, of CTA 0's copy of a shared-memory object.
__device__ __forceinline__ uint32_t leader_addr(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_addr(bar)) : "memory");
}
// mbar_wait for arrivals from the other CTA of the cluster.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t limit) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t spin = 0; spin < limit; ++spin) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if ((spin & 1023u) == 1023u && *abort_flag) return false;
  }
  return false;
}
// Loads of a pair: into this CTA's memory, counted by the leader's barrier.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(kIdescPair), "r"(accumulate)
      : "memory");
}
// Arrives on `bar` of both CTAs once every MMA issued so far has completed.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

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
template <int BM>
__device__ __forceinline__ Tile locate(int tile, const int* mb_prefix, const Args& a) {
  int lo = 0, hi = a.E;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (static_cast<int64_t>(mb_prefix[mid]) * a.n_blocks <= tile) lo = mid; else hi = mid;
  }
  const int mblocks = mb_prefix[lo + 1] - mb_prefix[lo];
  int local = tile - mb_prefix[lo] * a.n_blocks;
  constexpr int kHeight = kRowGroup * kBM / BM;
  const int group = local / (kHeight * a.n_blocks);
  local -= group * kHeight * a.n_blocks;
  const int left = mblocks - group * kHeight;
  const int height = left < kHeight ? left : kHeight;
  Tile t;
  t.expert = lo;
  t.nb = local / height;
  const int64_t first = static_cast<int64_t>(group * kHeight + local - t.nb * height) * BM;
  t.row0 = (a.offsets == nullptr ? 0 : a.offsets[lo]) + first;
  const int64_t rows = rows_of(a, lo) - first;
  t.rows = static_cast<int>(rows < BM ? rows : BM);
  return t;
}

// PAIR: two CTAs of a cluster share a tile of 256 rows. Each loads its own 128 rows and half of the 256
// weight rows (32 KB per 128 bytes of K instead of 48: at 64 bytes a clock and SM the tensor pipe
// otherwise waits for its operands), CTA 0 issues the MMAs of both, and each keeps its rows'
// accumulators and writes them out. Barriers: `full` of CTA 0 counts the bytes of both; `empty` and
// `tmem_full` of each are arrived on by CTA 0's commits; `tmem_empty` of CTA 0 by the epilogue warps
// of both.
template <int DT, bool PAIR>
__global__ void __launch_bounds__(kTileThreads, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                     const Args a) {
  constexpr int kRows = PAIR ? 2 * kBM : kBM;              // rows of a tile
  constexpr int kBBytes = (PAIR ? kBN / 2 : kBN) * kBK;    // weights this CTA loads per stage
  constexpr int kStageBytes = kABytes + kBBytes, kStages = kPipeBytes / kStageBytes;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kStages * kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPipeBytes);
  uint64_t* empty = full + kStages;
  uint64_t* tmem_full = empty + kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_base_slot + 1);
  uint64_t* drain = reinterpret_cast<uint64_t*>(abort_flag + 1);
  uint4* stage_buf = reinterpret_cast<uint4*>(smem + kPipeBytes + 256);
  int* mb_prefix = reinterpret_cast<int*>(smem + kPipeBytes + 256 + kEpiStageBytes);  // [E + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
  const int worker = static_cast<int>(blockIdx.x) / (PAIR ? 2 : 1), workers = static_cast<int>(gridDim.x) / (PAIR ? 2 : 1);
  const bool swiglu = a.act == FMOE_ACT_SWIGLU;
  int fills = 0;
  bool mma_issued = false;

  // ---- set-up: tile table, barriers, TMEM ----------------------------------------------
  for (int e = threadIdx.x; e < a.E; e += kTileThreads) {
    const int64_t n = rows_of(a, e);
    if (a.counts != nullptr && n != a.counts[e] && a.counts[e] > 0 && a.status != nullptr && blockIdx.x == 0)
      atomicOr(a.status, FMOE_STATUS_BAD_EXPERT);  // rows past the end of A were cut off
    mb_prefix[e + 1] = static_cast<int>((n + kRows - 1) / kRows);
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
      mbar_init(&tmem_empty[i], (PAIR ? 2 : 1) * kEpiWarps);
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
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_base_slot))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_base_slot))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers are set up before either is signalled
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int total_tiles = mb_prefix[a.E] * a.n_blocks;

  if (warp == 0 && lane == 0) {
    // ---- TMA producer ---------------------------------------------------------------
    int stage = 0;
    uint32_t phase = 0;
    for (int tile = worker; tile < total_tiles && !a.skip_loads; tile += workers) {
      const Tile t = locate<kRows>(tile, mb_prefix, a);
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        if constexpr (PAIR) {
          if (!mbar_wait_cluster(&empty[stage], phase ^ 1, abort_flag, a.spin_limit)) goto timed_out;
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * kStageBytes);
          const uint32_t bar = leader_addr(&full[stage]);
          tma_load_2d_pair(smem_a + stage * kABytes, &map_a, kb * kBK, static_cast<int>(t.row0) + rank * kBM, bar);
          // columns 0 .. 127 of the tile are CTA 0's, 128 .. 255 (the up rows for SwiGLU) CTA 1's
          const int w_row = swiglu ? rank * static_cast<int>(a.cols) + t.nb * 128 : t.nb * kBN + rank * 128;
          tma_load_3d_pair(smem_b + stage * kBBytes, &map_w, kb * kBK, w_row, t.expert, bar);
        } else {
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
        }
        ++fills;
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- MMA issuer -----------------------------------------------------------------
    int stage = 0;
    uint32_t phase = 0;
    int it = 0;
    for (int tile = worker; tile < total_tiles; tile += workers, ++it) {
      const int acc = it & 1;
      if (!mbar_wait_cluster(&tmem_empty[acc], ((it >> 1) & 1) ^ 1, abort_flag, a.spin_limit)) goto timed_out;
      tcgen05_fence_after();
      const uint32_t tmem_d = tmem_base + acc * kBN;
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        if (!mbar_wait_cluster(&full[stage], phase, abort_flag, a.spin_limit)) goto timed_out;
        tcgen05_fence_after();
        mma_issued = true;
        const uint64_t da = smem_desc(smem_u32(smem_a + stage * kABytes));
        const uint64_t db = smem_desc(smem_u32(smem_b + stage * kBBytes));
#pragma unroll
        for (int k = 0; k < kBK / kUmmaK; ++k) {  // 32 bytes along K inside the swizzle atom: +2 encoded
          if constexpr (PAIR) umma_i8_pair(tmem_d, da + 2 * k, db + 2 * k, (kb | k) != 0 ? 1u : 0u);
          else umma_i8(tmem_d, da + 2 * k, db + 2 * k, kIdesc, (kb | k) != 0 ? 1u : 0u);
        }
        if constexpr (PAIR) umma_commit_pair(&empty[stage]);
        else umma_commit(&empty[stage]);
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      if constexpr (PAIR) umma_commit_pair(&tmem_full[acc]);
      else umma_commit(&tmem_full[acc]);
    }
  } else if (warp >= 2) {
    // ---- epilogue -------------------------------------------------------------------
    using E = typename Elem<DT>::type;
    constexpr int kPiece = Elem<DT>::kVec;  // columns per 16 bytes of C
    constexpr int kPart = 4 * kPiece;       // columns per 64-byte segment of a row of C: 32, or 16 in fp32
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint4* stage_w = stage_buf + (warp - 2) * (32 * 4);
    const int out_cols = swiglu ? 128 : kBN;
    int it = 0;
    for (int tile = worker; tile < total_tiles; tile += workers, ++it) {
      const int acc = it & 1;
      Tile t = locate<kRows>(tile, mb_prefix, a);
      t.row0 += rank * kBM;  // this CTA's half of a pair's rows
      t.rows -= rank * kBM;
      const int row = quarter * 32 + lane;
      const int warp_rows = t.rows - quarter * 32;  // valid rows of this warp (may be <= 0)
      const float sa = row < t.rows ? a.a_scale[t.row0 + row] : 0.f;
      const float* sw = a.w_scale + static_cast<int64_t>(t.expert) * a.N;
      if (!mbar_wait_cluster(&tmem_full[acc], (it >> 1) & 1, abort_flag, a.spin_limit)) goto timed_out;
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + acc * kBN + (static_cast<uint32_t>(quarter * 32) << 16);
      const int c_end = (half + 1) * (out_cols / 2);
#pragma unroll 1
      for (int c0 = half * (out_cols / 2); c0 < c_end && warp_rows > 0; c0 += 32) {
        const int64_t col0 = static_cast<int64_t>(t.nb) * out_cols + c0;
        const int cols = static_cast<int>(a.cols - col0 < 32 ? a.cols - col0 : 32);
        if (cols <= 0) break;
        float f[32];
        // lane j holds the channel scale of column j and hands it round
        const float s0 = lane < cols ? sw[col0 + lane] : 0.f;
        if (swiglu) {
          const float s1 = lane < cols ? sw[a.cols + col0 + lane] : 0.f;
          uint32_t g[32], u[32];
          tmem_ld32(taddr + c0, g);
          tmem_ld32(taddr + 128 + c0, u);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float gate = static_cast<float>(static_cast<int>(g[i])) * sa * __shfl_sync(0xffffffffu, s0, i);
            const float up = static_cast<float>(static_cast<int>(u[i])) * sa * __shfl_sync(0xffffffffu, s1, i);
            f[i] = gate * sigmoid(gate) * up;
          }
        } else {
          uint32_t r[32];
          tmem_ld32(taddr + c0, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            f[i] = static_cast<float>(static_cast<int>(r[i])) * sa * __shfl_sync(0xffffffffu, s0, i);
          if (a.act == FMOE_ACT_GELU) {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = gelu(f[i]);
          }
        }
        // rows are regrouped through a swizzled staging block: whole 64-byte segments a store
#pragma unroll
        for (int h = 0; h < 32 / kPart; ++h) {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            stage_w[lane * 4 + (v ^ ((lane >> 1) & 3))] = pack16<DT>(f + h * kPart + kPiece * v);
          __syncwarp();
          E* out = static_cast<E*>(a.C) + (t.row0 + quarter * 32) * a.cols + col0 + h * kPart;
          const int n = cols - h * kPart;
          if (a.vec_ok && n >= kPart) {
#pragma unroll
            for (int step = 0; step < 4; ++step) {
              const int r = step * 8 + (lane >> 2), q = lane & 3;
              if (r < warp_rows)
                *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r) * a.cols + q * kPiece) = stage_w[r * 4 + (q ^ ((r >> 1) & 3))];
            }
          } else {  // rows off the 16-byte grid, or the last columns: an element a lane
            constexpr int kRows = 32 / kPart;  // rows a store covers: 1, or 2 in fp32
            const int j = lane & (kPart - 1);
#pragma unroll 4
            for (int r = lane / kPart; r < warp_rows && r < 32; r += kRows) {
              const E* from = reinterpret_cast<const E*>(&stage_w[r * 4 + ((j / kPiece) ^ ((r >> 1) & 3))]);
              if (j < n) out[static_cast<int64_t>(r) * a.cols + j] = from[j & (kPiece - 1)];
            }
          }
          __syncwarp();
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_leader(&tmem_empty[acc]);
        else mbar_arrive(&tmem_empty[acc]);
      }
    }
  }
  goto done;

timed_out:
  *abort_flag = 1;
  if (a.status != nullptr) atomicOr(a.status, FMOE_STATUS_WAIT_TIMEOUT);

done:
  if constexpr (PAIR) {
    // CTA 0 sees the pair's loads land and its MMAs finish; CTA 1 waits for it at the cluster's barrier,
    // after which nothing is on its way into either CTA's memory.
    if (rank == 0 && warp == 0 && lane == 0 && *abort_flag) {
      for (int s = 0; s < kStages && s < fills; ++s) {
        const int last = (fills - 1 - s) / kStages * kStages + s;  // last fill that used stage s
        mbar_wait_plain(&full[s], (last / kStages) & 1, a.spin_limit);
      }
    }
    if (mma_issued) {
      umma_commit_pair(drain);
      mbar_wait_plain(drain, 0, a.spin_limit);
    }
  } else {
    drain_on_exit(warp, lane, fills, mma_issued, full, drain, abort_flag, kStages, a.spin_limit);
  }
  tcgen05_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tcgen05_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
  if constexpr (PAIR) {
    __syncwarp();
    cluster_sync_all();  // neither leaves before both have given the tensor memory back
  }
}

// ---- few rows per expert: weights streamed past a handful of tokens ------------------------------
// With a few rows the product is bound by reading the weights once, and a 128 x 256 tile per CTA leaves
// most SMs without one (21504 x 7168 weights are 84 tiles; 7168 x 7168 are 28). Here a CTA takes 32
// weight rows and all of up to 8 * NT tokens, its eight warps each every eighth 128-byte piece of K:
// weights are the 16-row operand of mma.sync m16n8k32 and go from global memory straight into its
// fragments, tokens are the 8-column operand. A product's K order is free as long as both operands
// agree, so a thread's fragment words are the 16 consecutive bytes that one load brings:
// lane (g, t) takes bytes 16 t .. 16 t + 15 of a 64-byte step of rows g and g + 8, word 0 and 1 as
// the first MMA's two k halves, word 2 and 3 as the second's. The warps' integer sums meet in shared
// memory: exact, so the split changes nothing. The legacy MMA's rate does not matter here: it is the
// tile shape that counts.
constexpr int kFewThreads = 256, kFewWarps = 8, kFewRows = 32;  // weight rows per CTA
constexpr int kFewStep = 128;                                  // bytes of K per warp and step
constexpr int kFewPad = 4;  // columns of padding in the reduction buffer: fragment stores without bank conflicts

struct FewArgs {
  const int8_t* A;
  const int8_t* W;
  int64_t a_stride, w_stride, w_expert_stride;
  int64_t K;
  int n_blocks;  // groups of 32 weight rows (16 gate + 16 up rows for SwiGLU) per expert
  Args g;
};

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a token from byte k on, with zeros from K on: what lies behind a row does not count.
__device__ __forceinline__ uint4 load_token(const int8_t* row, int k, int K) {
  if (row == nullptr || k >= K) return make_uint4(0, 0, 0, 0);
  uint4 v = __ldg(reinterpret_cast<const uint4*>(row + k));
  if (k + 16 > K) {
    auto keep = [&](int i) { return K - k >= 4 * i + 4 ? ~0u : K - k <= 4 * i ? 0u : ~0u >> (32 - 8 * (K - k - 4 * i)); };
    v.x &= keep(0), v.y &= keep(1), v.z &= keep(2), v.w &= keep(3);
  }
  return v;
}

template <int DT, int NT>
__global__ void __launch_bounds__(kFewThreads) int8_few_rows_kernel(const FewArgs f) {
  using E = typename Elem<DT>::type;
  constexpr int kTokens = 8 * NT, kLine = kFewRows + kFewPad;
  __shared__ int red[kFewWarps][kTokens][kLine];
  extern __shared__ int chunk_prefix[];  // [E + 1] chunks of kTokens rows before each expert
  const Args& a = f.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int K = static_cast<int>(f.K);
  const bool swiglu = a.act == FMOE_ACT_SWIGLU;

  wait_for_previous_kernel();
  for (int e = threadIdx.x; e < a.E; e += kFewThreads) {
    const int64_t n = rows_of(a, e);
    if (a.counts != nullptr && n != a.counts[e] && a.counts[e] > 0 && a.status != nullptr && blockIdx.x == 0)
      atomicOr(a.status, FMOE_STATUS_BAD_EXPERT);  // rows past the end of A were cut off
    chunk_prefix[e + 1] = static_cast<int>((n + kTokens - 1) / kTokens);
  }
  if (threadIdx.x == 0) chunk_prefix[0] = 0;
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int base = 0; base < a.E; base += 32) {
      const int e = base + lane;
      int v = e < a.E ? chunk_prefix[e + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += n;
      }
      if (e < a.E) chunk_prefix[e + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const int items = chunk_prefix[a.E] * f.n_blocks;
  const int out_cols = swiglu ? kFewRows / 2 : kFewRows;

  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    int lo = 0, hi = a.E;  // last e with chunk_prefix[e] * n_blocks <= item
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<int64_t>(chunk_prefix[mid]) * f.n_blocks <= item) lo = mid; else hi = mid;
    }
    const int chunks = chunk_prefix[lo + 1] - chunk_prefix[lo];
    const int local = item - chunk_prefix[lo] * f.n_blocks;
    const int nb = local / chunks, chunk = local - nb * chunks;  // chunks that share weights run together
    const int64_t row0 = (a.offsets == nullptr ? 0 : a.offsets[lo]) + static_cast<int64_t>(chunk) * kTokens;
    const int64_t left = rows_of(a, lo) - static_cast<int64_t>(chunk) * kTokens;
    const int rows = static_cast<int>(left < kTokens ? left : kTokens);

    // this lane's four weight rows: g and g + 8 of each 16-row operand; past the end the last row again
    const int8_t* w_row[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int64_t n = swiglu ? static_cast<int64_t>(nb) * 16 + 8 * h + g : static_cast<int64_t>(nb) * kFewRows + 16 * m + 8 * h + g;
        if (n >= a.cols) n = a.cols - 1;
        if (swiglu) n += m * a.cols;
        w_row[m][h] = f.W + lo * f.w_expert_stride + n * f.w_stride + 16 * t;
      }
    const int8_t* tok[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) tok[j] = 8 * j + g < rows ? f.A + (row0 + 8 * j + g) * f.a_stride : nullptr;

    int acc[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0;

    // One step ahead: the next step's weights and tokens are on their way while this one's are multiplied.
    uint4 w[2][2][2], b[2][NT];  // weights [m][g or g + 8][64-byte half of the step]; tokens [half][j]
    auto load = [&](int k) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bool in = k + 64 * s + 16 * t < K;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            w[m][h][s] = in ? ld_stream16(reinterpret_cast<const uint4*>(w_row[m][h] + k + 64 * s)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < NT; ++j) b[s][j] = load_token(tok[j], k + 64 * s + 16 * t, K);
    };
    int k = warp * kFewStep;
    if (k < K) load(k);
    while (k < K) {
      uint4 cw[2][2][2], cb[2][NT];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) cw[m][h][s] = w[m][h][s];
#pragma unroll
        for (int j = 0; j < NT; ++j) cb[s][j] = b[s][j];
      }
      k += kFewWarps * kFewStep;
      if (k < K) load(k);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int m = 0; m < 2; ++m)
            mma_s8(acc[m][j], cw[m][0][s].x, cw[m][1][s].x, cw[m][0][s].y, cw[m][1][s].y, cb[s][j].x, cb[s][j].y);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int m = 0; m < 2; ++m)
            mma_s8(acc[m][j], cw[m][0][s].z, cw[m][1][s].z, cw[m][0][s].w, cw[m][1][s].w, cb[s][j].z, cb[s][j].w);
      }
    }
    __syncthreads();  // the previous item's sums have been read
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][8 * j + 2 * t + (i & 1)][16 * m + g + 8 * (i >> 1)] = acc[m][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < kTokens * out_cols; i += kFewThreads) {
      const int token = i / out_cols, c = i - token * out_cols;
      const int64_t col = static_cast<int64_t>(nb) * out_cols + c;
      if (token < rows && col < a.cols) {
        int sum = 0, up = 0;
#pragma unroll
        for (int v = 0; v < kFewWarps; ++v) {
          sum += red[v][token][c];
          if (swiglu) up += red[v][token][16 + c];
        }
        const float sa = a.a_scale[row0 + token];
        const float* sw = a.w_scale + static_cast<int64_t>(lo) * a.N;
        float y = static_cast<float>(sum) * sa * sw[col];
        if (swiglu) y = y * sigmoid(y) * (static_cast<float>(up) * sa * sw[a.cols + col]);
        else if (a.act == FMOE_ACT_GELU) y = gelu(y);
        static_cast<E*>(a.C)[(row0 + token) * a.cols + col] = from_float<DT>(y);
      }
    }
  }
}

// ---- up to a few hundred rows: weight rows as the MMA's M, tokens as its N, K split over a cluster ----
// A 128 x 256 tile streams 48 KB of operands per 128 bytes of K through one SM at 64 bytes a clock, and
// with few tiles most SMs watch: 7168 x 7168 weights took 32 us for any number of rows up to 512. Here
// the tile is 128 weight rows (64 gate + 64 up rows for SwiGLU) x NB tokens, so that for few tokens
// nearly all of an SM's traffic is weights, two CTAs share an SM, and where even that leaves SMs idle
// the K range is split over the S CTAs of a cluster. Their integer sums meet in distributed
// shared memory: exact, whatever the split.
// The accumulator arrives with lane = output column and column = token: a warp's stores of one token
// are 32 consecutive columns as they come.
constexpr int kTnRows = 128;
constexpr int kTnWBytes = kTnRows * kBK;  // 16 KB
template <int NB>
struct Tn {
  static constexpr int kStages = NB <= 32 ? 5 : NB <= 64 ? 4 : 3;  // two CTAs fit an SM
  static constexpr int kStageBytes = kTnWBytes + NB * kBK;
  static constexpr int kTmemCols = 2 * NB < 32 ? 32 : 2 * NB;  // two accumulators
};
constexpr int kTnExchange = 16 * 64;  // floats: up halves of 16 tokens on their way to the gate warps

struct TnArgs {
  Args g;
  int n_blocks;  // tiles of 128 weight rows (64 output columns for SwiGLU) per expert
  int splits;    // CTAs per cluster, each with its share of K; 1: a persistent grid
};

// One integer into CTA `rank`'s shared memory, at the place that `saddr` is in this CTA's.
__device__ __forceinline__ void st_cluster(uint32_t saddr, uint32_t rank, uint32_t v) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(saddr), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote), "r"(v) : "memory");
}
// Barrier of the four epilogue warps that also tells whether one of them gave up: a warp must not wait
// here for one that has left.
__device__ __forceinline__ bool epilogue_any(bool gave_up) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(gave_up))
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Up to four neighbouring outputs.
__device__ __forceinline__ void store4(void* C, int64_t i, int dt, const float* y, int n, bool whole) {
  if (whole && n == 4) {
    if (dt == FMOE_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(C) + i) = make_float4(y[0], y[1], y[2], y[3]);
    } else if (dt == FMOE_BF16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(C) + i) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      const __half2 lo = __floats2half2_rn(y[0], y[1]), hi = __floats2half2_rn(y[2], y[3]);
      *reinterpret_cast<uint2*>(static_cast<__half*>(C) + i) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) store_scalar_from_float(C, i + j, dt, y[j]);
  }
}

// The first n of 16 outputs of one column.
template <int DT>
__device__ __forceinline__ void store_column(void* C, int64_t at, int64_t stride, const float* y, int n) {
  typename Elem<DT>::type* p = static_cast<typename Elem<DT>::type*>(C) + at;
#pragma unroll
  for (int i = 0; i < 16; ++i, p += stride)
    if (i < n) *p = from_float<DT>(y[i]);
}

template <int NB>
__global__ void __launch_bounds__(kThreads, 2)
    int8_tn_kernel(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_w, const TnArgs f) {
  constexpr int kS = Tn<NB>::kStages, kStage = Tn<NB>::kStageBytes, kTmemCols = Tn<NB>::kTmemCols;
  constexpr uint32_t kIdescTn = (2u << 4) | (1u << 7) | (1u << 10) | ((NB >> 3) << 17) | ((kTnRows >> 4) << 24);
  static_assert(kS * kStage >= NB * kTnRows * 4, "the partial sums take the place of the pipeline");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kS * kStage);
  uint64_t* empty = full + kS;
  uint64_t* tmem_full = empty + kS;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_base_slot + 1);
  uint64_t* drain = reinterpret_cast<uint64_t*>(abort_flag + 1);
  float* exchange = reinterpret_cast<float*>(smem + kS * kStage + 256);
  int* chunk_prefix = reinterpret_cast<int*>(exchange + kTnExchange);  // [E + 1]
  // partial sums from each CTA of the cluster for this CTA's tokens, after the pipelines have drained
  int* part = reinterpret_cast<int*>(smem);                            // [splits][NB / splits][128]

  const Args& a = f.g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool swiglu = a.act == FMOE_ACT_SWIGLU;
  const int out_cols = swiglu ? kTnRows / 2 : kTnRows;
  const int split = f.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int k_begin = a.k_blocks * split / f.splits, k_end = a.k_blocks * (split + 1) / f.splits;
  int fills = 0;
  bool mma_issued = false;

  // ---- set-up: barriers and TMEM, which need nobody's results, then the chunk table ------------
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kS; ++s) {
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
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)),
                 "n"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  wait_for_previous_kernel();
  for (int e = threadIdx.x; e < a.E; e += kThreads) {
    const int64_t n = rows_of(a, e);
    if (a.counts != nullptr && n != a.counts[e] && a.counts[e] > 0 && a.status != nullptr && blockIdx.x == 0)
      atomicOr(a.status, FMOE_STATUS_BAD_EXPERT);  // rows past the end of A were cut off
    chunk_prefix[e + 1] = static_cast<int>((n + NB - 1) / NB);
  }
  if (threadIdx.x == 0) chunk_prefix[0] = 0;
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int base = 0; base < a.E; base += 32) {
      const int e = base + lane;
      int v = e < a.E ? chunk_prefix[e + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += n;
      }
      if (e < a.E) chunk_prefix[e + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int items = chunk_prefix[a.E] * f.n_blocks;
  const int first = static_cast<int>(blockIdx.x) / f.splits, stride = static_cast<int>(gridDim.x) / f.splits;
  // one item per cluster: there are enough of them unless experts claim the same rows
  if (f.splits > 1 && items > stride && blockIdx.x == 0 && threadIdx.x == 0 && a.status != nullptr)
    atomicOr(a.status, FMOE_STATUS_BAD_EXPERT);

  struct Item {
    int expert, nb, rows;
    int64_t row0;
  };
  auto find = [&](int item) {  // the chunks of an expert's rows that read the same weights are neighbours
    int lo = 0, hi = a.E;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<int64_t>(chunk_prefix[mid]) * f.n_blocks <= item) lo = mid; else hi = mid;
    }
    const int chunks = chunk_prefix[lo + 1] - chunk_prefix[lo];
    const int local = item - chunk_prefix[lo] * f.n_blocks;
    Item t;
    t.expert = lo;
    t.nb = local / chunks;
    const int64_t begin = static_cast<int64_t>(local - t.nb * chunks) * NB;
    t.row0 = (a.offsets == nullptr ? 0 : a.offsets[lo]) + begin;
    const int64_t rows = rows_of(a, lo) - begin;
    t.rows = static_cast<int>(rows < NB ? rows : NB);
    return t;
  };

  if (warp == 0 && lane == 0) {
    // ---- TMA producer ---------------------------------------------------------------
    int stage = 0;
    uint32_t phase = 0;
    for (int item = first; item < items && !a.skip_loads; item += stride) {
      const Item t = find(item);
      for (int kb = k_begin; kb < k_end; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, a.spin_limit)) goto timed_out;
        mbar_expect_tx(&full[stage], kStage);
        uint8_t* w = smem + stage * kStage;
        if (swiglu) {  // 64 gate rows, then the up rows of the same columns
          tma_load_3d(w, &map_w, kb * kBK, t.nb * 64, t.expert, &full[stage]);
          tma_load_3d(w + kTnWBytes / 2, &map_w, kb * kBK, static_cast<int>(a.cols) + t.nb * 64, t.expert, &full[stage]);
        } else {
          tma_load_3d(w, &map_w, kb * kBK, t.nb * kTnRows, t.expert, &full[stage]);
        }
        tma_load_2d(w + kTnWBytes, &map_t, kb * kBK, static_cast<int>(t.row0), &full[stage]);
        ++fills;
        if (++stage == kS) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1 && lane == 0) {
    // ---- MMA issuer -----------------------------------------------------------------
    int stage = 0;
    uint32_t phase = 0;
    int it = 0;
    for (int item = first; item < items; item += stride, ++it) {
      const int acc = it & 1;
      if (!mbar_wait(&tmem_empty[acc], ((it >> 1) & 1) ^ 1, abort_flag, a.spin_limit)) goto timed_out;
      tcgen05_fence_after();
      for (int kb = k_begin; kb < k_end; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, a.spin_limit)) goto timed_out;
        tcgen05_fence_after();
        mma_issued = true;
        const uint64_t dw = smem_desc(smem_u32(smem + stage * kStage));
        const uint64_t dt = smem_desc(smem_u32(smem + stage * kStage + kTnWBytes));
#pragma unroll
        for (int k = 0; k < kBK / kUmmaK; ++k)
          umma_i8(tmem_base + acc * NB, dw + 2 * k, dt + 2 * k, kIdescTn, kb > k_begin || k > 0 ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == kS) { stage = 0; phase ^= 1; }
      }
      umma_commit(&tmem_full[acc]);
    }
  } else if (warp >= 2) {
    // ---- epilogue -------------------------------------------------------------------
    const int quarter = warp & 3, line = quarter * 32 + lane;  // line: weight row of the tile
    int it = 0;
    for (int item = first; item < items; item += stride, ++it) {
      const int acc = it & 1;
      const Item t = find(item);
      const int64_t col = static_cast<int64_t>(t.nb) * out_cols + (line & (out_cols - 1));
      const bool up = swiglu && line >= 64;
      const float sw = col < a.cols ? a.w_scale[static_cast<int64_t>(t.expert) * a.N + (up ? a.cols : 0) + col] : 0.f;
      // lane j has the scales of tokens j, j + 32, ..: here, not where they are used, 0.7 us away from memory each
      float sa[(NB + 31) / 32];
#pragma unroll
      for (int j = 0; j < (NB + 31) / 32; ++j) sa[j] = 32 * j + lane < t.rows ? a.a_scale[t.row0 + 32 * j + lane] : 0.f;
      if (epilogue_any(!mbar_wait(&tmem_full[acc], (it >> 1) & 1, abort_flag, a.spin_limit))) goto timed_out;
      if (f.splits > 1) break;  // one item per cluster: its sums meet below
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + acc * NB + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < t.rows; c0 += 16) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_ld_wait();
        float mine = sa[0];
#pragma unroll
        for (int j = 1; j < (NB + 31) / 32; ++j) mine = c0 >= 32 * j ? sa[j] : mine;
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          y[i] = static_cast<float>(static_cast<int>(r[i])) * __shfl_sync(0xffffffffu, mine, (c0 & 16) + i) * sw;
        if (swiglu) {
          if (up) {
#pragma unroll
            for (int i = 0; i < 16; ++i) exchange[i * 64 + line - 64] = y[i];
          }
          epilogue_sync();
          if (!up) {
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = y[i] * sigmoid(y[i]) * exchange[i * 64 + line];
          }
          epilogue_sync();
        } else if (a.act == FMOE_ACT_GELU) {
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = gelu(y[i]);
        }
        if (!up && col < a.cols) {
          const int64_t at = (t.row0 + c0) * a.cols + col;
          const int n = t.rows - c0;
          if (a.out_dtype == FMOE_F32) store_column<FMOE_F32>(a.C, at, a.cols, y, n);
          else if (a.out_dtype == FMOE_BF16) store_column<FMOE_BF16>(a.C, at, a.cols, y, n);
          else store_column<FMOE_F16>(a.C, at, a.cols, y, n);
        }
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
  drain_on_exit(warp, lane, fills, mma_issued, full, drain, abort_flag, kS, a.spin_limit);
  tcgen05_fence_before();
  __syncthreads();
  // A cluster's CTAs each finish every splits-th token: they send each other their partial sums, and each adds
  // up what it got from its own shared memory. (Fetching the others' sums instead, a round trip for every
  // one, took 20.0 us where this takes 18.4 for 128 rows of 7168 x 7168 in four parts.)
  // All threads of all its CTAs come here, also after a wait gave up.
  const int quads = out_cols / 4, c = static_cast<int>(threadIdx.x) % quads * 4;  // kThreads is a multiple of quads
  Item t{0, 0, 0, 0};
  int64_t col = 0;
  float sg[4], su[4];
  if (f.splits > 1) {
    if (first < items) {
      t = find(first);
      col = static_cast<int64_t>(t.nb) * out_cols + c;
      const float* scales = a.w_scale + static_cast<int64_t>(t.expert) * a.N;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sg[j] = col + j < a.cols ? scales[col + j] : 0.f;
        su[j] = swiglu && col + j < a.cols ? scales[a.cols + col + j] : 0.f;
      }
    }
    __syncwarp();
    cluster_sync_all();  // every CTA's pipeline has drained
    tcgen05_fence_after();
    if (warp >= 2) {
      const int quarter = warp & 3, shift = __ffs(f.splits) - 1;
      const uint32_t mine = smem_u32(part + split * (NB * kTnRows >> shift) + quarter * 32 + lane);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < t.rows; c0 += 16) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c0 + i < t.rows) st_cluster(mine + 4 * kTnRows * ((c0 + i) >> shift), i & (f.splits - 1), r[i]);
      }
    }
    tcgen05_fence_before();
    __syncwarp();
    cluster_sync_all();
  }
  if (warp == 1) {
    __syncwarp();
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(kTmemCols) : "memory");
  }
  if (f.splits == 1 || col >= a.cols) return;
  // four neighbouring columns of a token to a thread
  for (int i = static_cast<int>(threadIdx.x) / quads; i * f.splits + split < t.rows; i += kThreads / quads) {
    const int64_t row = t.row0 + i * f.splits + split;
    const float sa = a.a_scale[row];
    const int* from = part + i * kTnRows + c;
    int4 sum = make_int4(0, 0, 0, 0), up = sum;
    for (int r = 0; r < f.splits; ++r, from += NB * kTnRows / f.splits) {
      const int4 v = *reinterpret_cast<const int4*>(from);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
      if (swiglu) {
        const int4 w = *reinterpret_cast<const int4*>(from + 64);
        up.x += w.x, up.y += w.y, up.z += w.z, up.w += w.w;
      }
    }
    const int sums[4] = {sum.x, sum.y, sum.z, sum.w}, ups[4] = {up.x, up.y, up.z, up.w};
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[j] = static_cast<float>(sums[j]) * sa * sg[j];
      if (swiglu) y[j] = y[j] * sigmoid(y[j]) * (static_cast<float>(ups[j]) * sa * su[j]);
      else if (a.act == FMOE_ACT_GELU) y[j] = gelu(y[j]);
    }
    store4(a.C, row * a.cols + col, a.out_dtype, y, static_cast<int>(a.cols - col < 4 ? a.cols - col : 4),
           a.cols % 4 == 0 && a.vec_ok != 0);
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

template <int DT, int NT>
static int launch_few(const FewArgs& f, int64_t items, cudaStream_t st) {
  static_assert(sizeof(int) * kFewWarps * 8 * NT * (kFewRows + kFewPad) <= 40 * 1024, "static and dynamic part within 48 KB");
  int per_sm = 0;
  const int smem = static_cast<int>(sizeof(int)) * (f.g.E + 1);
  FMOE_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, int8_few_rows_kernel<DT, NT>, kFewThreads, smem));
  const int64_t most = static_cast<int64_t>(per_sm > 0 ? per_sm : 1) * kNumSMs;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(items < most ? items : most));
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FMOE_CUDA(cudaLaunchKernelEx(&cfg, int8_few_rows_kernel<DT, NT>, f));
  return check_launch("int8_few_rows_kernel");
}

template <int NB>
static int launch_tn(const CUtensorMap& map_t, const CUtensorMap& map_w, const TnArgs& f, int64_t items, cudaStream_t st) {
  constexpr int kFixed = 1024 + Tn<NB>::kStages * Tn<NB>::kStageBytes + 256 + 4 * kTnExchange;
  const size_t smem = kFixed + sizeof(int) * (f.g.E + 2);
  FMOE_CUDA(cudaFuncSetAttribute(int8_tn_kernel<NB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kFixed + static_cast<int>(sizeof(int)) * (kMaxExperts + 2)));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  const int64_t most = 2 * static_cast<int64_t>(g_gemm_sms);
  cfg.gridDim = dim3(static_cast<unsigned>(f.splits > 1 ? items * f.splits : items < most ? items : most));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = f.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = f.splits > 1 ? 2 : 1;
  FMOE_CUDA(cudaLaunchKernelEx(&cfg, int8_tn_kernel<NB>, map_t, map_w, f));
  return check_launch("int8_tn_kernel");
}

template <int DT, bool PAIR>
static int launch_tiles(const CUtensorMap& map_a, const CUtensorMap& map_w, const Args& g, cudaStream_t st) {
  constexpr int kFixed = 1024 + kPipeBytes + 256 + kEpiStageBytes, kRows = PAIR ? 2 * kBM : kBM, kCtas = PAIR ? 2 : 1;
  FMOE_CUDA(cudaFuncSetAttribute(int8_gemm_kernel<DT, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kFixed + static_cast<int>(sizeof(int)) * (kMaxExperts + 2)));
  // upper bound of the tile count, known without reading the counts: one partial block per expert
  const int64_t tiles = ((g.R + kRows - 1) / kRows + g.E - 1) * g.n_blocks;
  const int64_t most = g_gemm_sms / kCtas > 0 ? g_gemm_sms / kCtas : 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(static_cast<unsigned>(kCtas * (tiles < most ? tiles : most)));
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = kFixed + sizeof(int) * (g.E + 2);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 1 : 0;
  FMOE_CUDA(cudaLaunchKernelEx(&cfg, int8_gemm_kernel<DT, PAIR>, map_a, map_w, g));
  return check_launch("int8_gemm_kernel");
}

// Kernel 0 (tiles), 1 (few rows), 2 (weight rows as M) or 3 (pairs) for E experts of which `reached` can have rows,
// `mean` rows each. The first two by an estimate of their times in us, fitted to (few / 2 / tiles): 512 x
// 4096, 16 rows 3.2 / 4.2 / 6.9, 64 rows 7.6 / 5.1 / 7.2; 2048 x 7168, 8 rows 5.9 / 8.2 / 12.9, 24 rows 10.5 /
// 8.5 / 13.2; 7168 x 7168, 8 rows 13.9 / 15.4 / 33, 16 rows 20.8 / 15.5 / 33; 8192 x 1024, 1 row 7.6 / 6.8 / 26;
// 1008 x 515, 256 rows 6.0 / 8.3 / 13.8: few rows pays for every 8 tokens by 32 weight rows, kernel 2 for the weights
// once and for its start and end. The tiled kernel (2 / tiles / pairs) streams fewer bytes per product but
// needs tiles for most SMs and starts 2 us later: 7168 x 7168, 256 rows 24.7 / 29.5 / 27.2, 512 rows 30.0 / 29.2 / 27.3;
// 2048 x 7168, 1024 rows 19.7 / 20.4 / 20.4, 2048 rows 31.2 / 29.9 / 30.9; 64 experts of 7168 x 4096 with SwiGLU, 64 rows
// each 294 / 293, 128 each 375 / 361. Pairs of CTAs gain on a long K where their tiles of 256 rows do not cost a round
// more: 7168 x 21504, 256 rows 55.8 / 49.8, 384 rows 54.7 / 62.7, 512 rows 75 / 65; 8192 x 8192, 32768 rows for seconds on
// end (at the power limit) 1680 / 1620; experts' rows come in ragged numbers, and pad them at a few hundred
// (32 experts of 7168 x 4096, 256 rows each 263 / 292, 2048 rows for seconds on end 1490 / 1440).
static int pick_kernel(const Args& g, int64_t K, int64_t reached, int64_t mean, int64_t few_items, int nb, int64_t tn_items) {
  const double weights = static_cast<double>(reached) * static_cast<double>(g.N) * static_cast<double>(K);
  const double rounds = few_items > kNumSMs ? static_cast<double>(few_items) / kNumSMs : 1.0;
  const double few = 2.4 + fmax(rounds * (0.45 + 0.55 * static_cast<double>(K) / 1024), weights / 5e6);
  const double tn = 4.2 + fmax(0.245 * (g.k_blocks < 12 ? g.k_blocks : 12) - 1.0, weights / 6e6) + nb / 64.0;
  const bool long_k = K >= 4096;
  if (mean <= 64 || tn_items <= (long_k || g.act == FMOE_ACT_SWIGLU ? 1 : 4) * kNumSMs) return few < tn ? 1 : 2;
  if (!long_k) return 0;
  if (g.E > 1) return mean < 1024 ? 0 : 3;
  const int64_t tiles = (g.R + kBM - 1) / kBM * g.n_blocks, pairs = (g.R + 2 * kBM - 1) / (2 * kBM) * g.n_blocks;
  return (pairs + kNumSMs / 2 - 1) / (kNumSMs / 2) <= (tiles + kNumSMs - 1) / kNumSMs ? 3 : 0;
}

// Parts of K for the CTAs of a cluster, for as long as there are CTAs to spare (two to an SM). A part saves its k
// blocks (0.25 us each); the exchange costs 1.5 us, 2 to 4 in two parts, and more when the SMs are full.
// Measured (1 / 2 / 4 / 8 parts, us; 128 rows): 1024 x 512 7.2 / 10.4 / 8.2 / 7.4, 2048 x 512 9.3 / 11.4 / 8.7 / 7.5, 2048 x
// 2048 9.3 / 11.4 / 8.8 / 9.6, 7168 x 2048 24.6 / 19.4 / 13.3 / 12.3, 2048 x 7168 11.3 / 13.2 / 12.8, 4096 x 7168 17.4 / 17.0 /
// 15.2; 256 rows: 4096 x 7168 17.6 / 19.2, 7168 x 7168 26.4 / 24.5.
static int pick_splits(int64_t items, int k_blocks) {
  for (int parts = 8; parts > 1 && k_blocks >= 12; parts /= 2) {
    const int64_t ctas = items * parts;
    const int least = parts == 2 ? 20 : ctas > kNumSMs ? 8 : 2 * ctas > kNumSMs ? 4 : 2;  // k blocks of a part
    if (ctas <= 2 * kNumSMs && k_blocks / parts >= least) return parts;
  }
  return 1;
}

}  // namespace i8

int g_int8_kernel = -1;  // fmoe_tune "int8_kernel": 0 tiles, 1 few rows, 2 split K, 3 pairs; -1 = by the sizes

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
  // Which kernel: the host knows the rows and the experts, not how the rows are spread.
  const int64_t reached = R < E ? R : E, mean = (R + E - 1) / E;
  const int64_t tokens = E == 1 ? R : 2 * mean;  // rows that an expert may well have
  const int few_blocks = static_cast<int>(swiglu ? (cols + 15) / 16 : (N + i8::kFewRows - 1) / i8::kFewRows);
  const int64_t few_items = (E == 1 ? (R + 7) / 8 : R / 8 + reached) * few_blocks;
  const int tn_blocks = static_cast<int>(swiglu ? (cols + 63) / 64 : (N + i8::kTnRows - 1) / i8::kTnRows);
  const int nb = tokens <= 16 ? 16 : tokens <= 32 ? 32 : tokens <= 64 ? 64 : 128;
  const int64_t tn_items = (E == 1 ? (R + nb - 1) / nb : R / nb + reached) * tn_blocks;
  int which = g_int8_kernel;
  if (which < 0) which = i8::pick_kernel(g, K, reached, mean, few_items, nb, tn_items);
  if (which == 1) {
    i8::FewArgs f;
    f.A = a;
    f.W = w;
    f.a_stride = a_stride;
    f.w_stride = w_stride;
    f.w_expert_stride = E == 1 ? 0 : w_expert_stride;
    f.K = K;
    f.n_blocks = few_blocks;
    f.g = g;
    FMOE_REQUIRE(few_items < (1ll << 31), FMOE_ERR_UNSUPPORTED, "fmoe_int8_gemm: too many tiles");
    int rc = FMOE_OK;
    FMOE_DISPATCH_DTYPE(out_dtype, DT, rc = (i8::launch_few<DT, 1>(f, few_items, static_cast<cudaStream_t>(stream))));
    return rc;
  }
  if (which == 2) {
    i8::TnArgs f;
    f.g = g;
    f.n_blocks = tn_blocks;
    FMOE_REQUIRE(tn_items < (1ll << 31) / 8, FMOE_ERR_UNSUPPORTED, "fmoe_int8_gemm: too many tiles");
    f.splits = i8::pick_splits(tn_items, g.k_blocks);
    CUtensorMap map_t, map_w;
    int rc = i8::make_map(&map_t, a, 1, R, K, a_stride, R * a_stride, nb, 2, "A");
    if (rc != 0) return rc;
    rc = i8::make_map(&map_w, w, E, N, K, w_stride, E == 1 ? N * w_stride : w_expert_stride, swiglu ? 64 : i8::kTnRows, 3, "W");
    if (rc != 0) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (nb == 16) return i8::launch_tn<16>(map_t, map_w, f, tn_items, st);
    if (nb == 32) return i8::launch_tn<32>(map_t, map_w, f, tn_items, st);
    if (nb == 64) return i8::launch_tn<64>(map_t, map_w, f, tn_items, st);
    return i8::launch_tn<128>(map_t, map_w, f, tn_items, st);
  }
  CUtensorMap map_a, map_w;
  int rc = i8::make_map(&map_a, a, 1, R, K, a_stride, R * a_stride, i8::kBM, 2, "A");
  if (rc != 0) return rc;
  rc = i8::make_map(&map_w, w, E, N, K, w_stride, E == 1 ? N * w_stride : w_expert_stride,
                    swiglu || which == 3 ? 128 : i8::kBN, 3, "W");
  if (rc != 0) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FMOE_DISPATCH_DTYPE(out_dtype, DT, {
    rc = which == 3 ? i8::launch_tiles<DT, true>(map_a, map_w, g, st) : i8::launch_tiles<DT, false>(map_a, map_w, g, st);
  });
  return rc;
}
