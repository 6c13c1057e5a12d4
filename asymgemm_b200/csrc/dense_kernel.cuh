// Dense matrix product D[r, c] = sum_k A(r, k) * B(c, k) for bf16 or fp16 operands on the tensor cores, with an epilogue of
// bias, activation and residual. One kernel body serves y = x W^T, dx = dz W and dW = dz^T x: an operand is either
// "K-major" (the contraction index is the contiguous one in memory) or "MN-major" (the row index of the operand is), which only
// changes the boxes TMA fetches, the descriptors' strides and two bits of the instruction descriptor. Nothing is transposed in
// memory.
//
// Accumulation. The tensor core adds to its fp32 accumulators by truncation, which loses about K / 16 * 2^-24 of a sum of
// terms of one sign (measured here: 2.8e-5 relative at K = 7168, 2.2e-6 at 1024). So it accumulates kChunkSteps * 64 terms
// at a time into one of two TMEM buffers, and the drain warps add those to fp32 accumulators in registers, rounded to
// nearest, while it fills the other: the error stays that of one chunk whatever K is.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mgrouped_pair_kernel.cuh"

namespace agb {

constexpr int kStepK = 64;         // contraction elements per pipeline step: one 128-byte row of the swizzled tiles
constexpr int kChunkSteps = 8;     // steps accumulated in TMEM before they are added to the registers
constexpr int kTileA = 128;        // operand A rows per CTA = TMEM lanes

enum : int { T_BF16 = 0, T_FP16 = 1, T_FP32 = 2 };
enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

struct DenseParams {
  int rows_a, rows_b;        // extents of the product
  int steps;                 // ceil(K / kStepK)
  int tiles_b;               // tiles along B
  int swapped;               // 0: D is the output; 1: D is its transpose (A's rows are the output's columns)
  uint32_t idesc;
  const void* bias;          // per output column, or null
  const void* residual;      // like the output, rows ldr apart, or null
  void* out;
  void* pre;                 // value before the activation, in the operands' type, rows ldp apart, or null
  long long ldr, ldo, ldp;
  int bias_type, out_type, pre_type, act;
  int* status;
  unsigned long long timeout_ns;
};

__device__ __forceinline__ float load_as_float(const void* p, long long i, int type) {
  if (type == T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (type == T_FP16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_from_float(void* p, long long i, int type, float v) {
  if (type == T_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (type == T_FP16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : z;                       // NaN stays NaN
  if (act == ACT_GELU) return z * normcdff(z);                       // x Phi(x), exact also where Phi is small
  if (act == ACT_SILU) return z / (1.f + expf(-z));
  return z;
}

// One output element: z = acc + bias, y = act(z) + residual.
__device__ __forceinline__ void finish(const DenseParams& p, long long m, long long n, float acc) {
  float z = acc;
  if (p.bias != nullptr) z += load_as_float(p.bias, n, p.bias_type);
  if (p.pre != nullptr) store_from_float(p.pre, m * p.ldp + n, p.pre_type, z);
  float y = activate(z, p.act);
  if (p.residual != nullptr) y += load_as_float(p.residual, m * p.ldr + n, p.out_type);
  store_from_float(p.out, m * p.ldo + n, p.out_type, y);
}

// Descriptor of an MN-major tile: blocks of 64 rows (128 bytes, the contiguous direction) x kStepK contraction indices, each
// block 64 x 128 bytes with the 128-byte swizzle. 8 contraction indices are 1024 bytes apart (stride offset), 64-row blocks
// 8192 (leading offset).
__device__ __forceinline__ uint64_t make_mnmajor_sw128_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((kStepK * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr) {
  if constexpr (MN) return make_mnmajor_sw128_desc(smem_addr);
  else return make_kmajor_sw128_desc(smem_addr);
}
// bytes from one MMA's 16 contraction indices to the next within a step's tile
template <bool MN>
__host__ __device__ constexpr int operand_k_bytes() { return MN ? 16 * 128 : 32; }

// One step of an operand: ROWS rows from `row`, contraction indices from `k`.
template <bool MN, int ROWS>
__device__ __forceinline__ void load_operand(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int k) {
  if constexpr (MN) {
#pragma unroll
    for (int b = 0; b < ROWS / 64; ++b) tma_load_2d(dst + b * kStepK * 128, map, bar, row + b * 64, k);
  } else {
    tma_load_2d(dst, map, bar, k, row);
  }
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// ------------------------------------------------------------------------------------------------ one tile per CTA
// 128 x BN tile per CTA, the contraction split over the CTAs of a cluster (1, 2, 4 or 8). The CTAs' partial tiles meet in
// shared memory: each sums an equal share of the tile over the cluster in the order of the splits (so the result does not
// depend on timing), applies the epilogue and stores it. No workspace, no atomics, one launch.
template <int BN>
constexpr int tile_stages() { return BN >= 128 ? 6 : BN == 64 ? 4 : 5; }   // BN <= 64: two CTAs fit on an SM

template <int BN>
struct TileSmem {
  static constexpr int stages = tile_stages<BN>();
  static constexpr int a_bytes = kTileA * 128, b_bytes = BN * 128, stage_bytes = a_bytes + b_bytes;
  static constexpr int pitch = BN + 1;                            // of the fp32 tile, which takes the ring's place at the end
  static constexpr int bar_off = stages * stage_bytes;
  static constexpr int total = bar_off + (2 * stages + 4) * 8 + 16;
  static constexpr int dyn_bytes = total + 1024;
  static_assert(kTileA * pitch * 4 <= bar_off, "the fp32 tile must fit into the ring");
};

constexpr int kTileThreads = 256;
template <int BN>
__host__ __device__ constexpr uint32_t tile_tmem_cols() { return 2 * BN < 32 ? 32 : 2 * BN; }

template <int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kTileThreads, BN >= 128 ? 1 : 2)
dense_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const DenseParams p, const int splits) {
  static_assert(!B_MN || BN >= 64, "an MN-major tile is made of 64-row blocks");
  using L = TileSmem<BN>;
  constexpr int ST = L::stages;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::bar_off);
  uint64_t* empty = full + ST;
  uint64_t* tm_full = empty + ST;
  uint64_t* tm_empty = tm_full + 2;
  uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(tm_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_smem + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(cluster_cta_rank());       // the cluster runs along the splits
  const int tile = blockIdx.x / splits;
  const int a0 = (tile / p.tiles_b) * kTileA, b0 = (tile % p.tiles_b) * BN;
  const int step0 = static_cast<int>(static_cast<long long>(p.steps) * split / splits);
  const int steps = static_cast<int>(static_cast<long long>(p.steps) * (split + 1) / splits) - step0;
  const int chunks = (steps + kChunkSteps - 1) / kChunkSteps;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tm_full[i], 1); mbar_init(&tm_empty[i], 4); }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 2) {
    tmem_alloc(tmem_base_smem, tile_tmem_cols<BN>());
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_smem;
  const WaitCtx wc{p.status, abort_flag, p.timeout_ns};
  float* tile_smem = reinterpret_cast<float*>(smem);

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < steps; ++i) {
        const int s = i % ST;
        if (!wait_bar(&empty[s], ((i / ST) & 1) ^ 1, wc, ST_TIMEOUT_A_EMPTY)) break;
        mbar_arrive_expect_tx(&full[s], L::stage_bytes);
        uint8_t* dst = smem + s * L::stage_bytes;
        load_operand<A_MN, kTileA>(dst, &map_a, &full[s], a0, (step0 + i) * kStepK);
        load_operand<B_MN, BN>(dst + L::a_bytes, &map_b, &full[s], b0, (step0 + i) * kStepK);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < steps; ++i) {
        const int s = i % ST, j = i % kChunkSteps, chunk = i / kChunkSteps, slot = chunk & 1;
        if (j == 0 && !wait_bar(&tm_empty[slot], ((chunk >> 1) & 1) ^ 1, wc, ST_TIMEOUT_TM_EMPTY)) break;
        if (!wait_bar(&full[s], (i / ST) & 1, wc, ST_TIMEOUT_A_FULL)) break;
        tc_fence_after_sync();
        const uint32_t at = smem_u32(smem + s * L::stage_bytes);
        const uint64_t da = operand_desc<A_MN>(at), db = operand_desc<B_MN>(at + L::a_bytes);
#pragma unroll
        for (int q = 0; q < kStepK / 16; ++q)
          umma<MmaKind::F16>(tmem_base + slot * BN, da + ((q * operand_k_bytes<A_MN>()) >> 4), db + ((q * operand_k_bytes<B_MN>()) >> 4),
                             p.idesc, j > 0 || q > 0);
        umma_commit(&empty[s]);
        if (j == kChunkSteps - 1 || i == steps - 1) umma_commit(&tm_full[slot]);
      }
    }
  } else if (warp >= 4) {
    constexpr int W = BN < 32 ? BN : 32;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float acc[BN];
#pragma unroll
    for (int c = 0; c < BN; ++c) acc[c] = 0.f;
    bool ok = true;
    for (int chunk = 0; chunk < chunks; ++chunk) {
      const int slot = chunk & 1;
      ok = wait_bar(&tm_full[slot], (chunk >> 1) & 1, wc, ST_TIMEOUT_TM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += W) {
        uint32_t r[W];
        tmem_ld_cols(lane_addr + slot * BN + c0, r);
        tmem_wait_ld_into(r);
#pragma unroll
        for (int c = 0; c < W; ++c) acc[c0 + c] += __uint_as_float(r[c]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tm_empty[slot]);
    }
    // the last chunk is complete: every load has landed and every MMA has read it, so the ring is free
    if (ok) {
      float* row = tile_smem + ((warp & 3) * 32 + lane) * L::pitch;
#pragma unroll
      for (int c = 0; c < BN; ++c) row[c] = acc[c];
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  if (*abort_flag) {
    // loads of this CTA may still be on their way into its shared memory: they take a few microseconds
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  } else {
    uint32_t part[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) part[s] = map_to_cta(smem_u32(tile_smem), s < splits ? s : 0);
    auto sum_of = [&](int r, int c) {
      const uint32_t off = static_cast<uint32_t>(r * L::pitch + c) * 4;
      if (splits == 1) return tile_smem[r * L::pitch + c];
      float v = ld_cluster_f32(part[0] + off);
#pragma unroll
      for (int s = 1; s < 8; ++s)
        if (s < splits) v += ld_cluster_f32(part[s] + off);
      return v;
    };
    if (p.swapped) {
      const int share = BN / splits;
      for (int e = threadIdx.x; e < share * kTileA; e += kTileThreads) {
        const int r = e % kTileA, c = split * share + e / kTileA;
        if (a0 + r < p.rows_a && b0 + c < p.rows_b) finish(p, b0 + c, a0 + r, sum_of(r, c));
      }
    } else {
      const int share = kTileA / splits;
      for (int e = threadIdx.x; e < share * BN; e += kTileThreads) {
        const int r = split * share + e / BN, c = e % BN;
        if (a0 + r < p.rows_a && b0 + c < p.rows_b) finish(p, a0 + r, b0 + c, sum_of(r, c));
      }
    }
  }
  __syncthreads();
  cluster_sync_all();        // no CTA leaves while another may read its tile
  if (warp == 2) tmem_dealloc(tmem_base, tile_tmem_cols<BN>());
}

}  // namespace agb
