// Dense matrix product D[r, c] = sum_k A(r, k) * B(c, k) for bf16 or fp16 operands on the tensor cores, with an epilogue of
// bias, activation and residual. One kernel body serves y = x W^T, dx = dz W and dW = dz^T x: an operand is either
// "K-major" (the contraction index is the contiguous one in memory) or "MN-major" (the row index of the operand is), which only
// changes the boxes TMA fetches, the descriptors' strides and two bits of the instruction descriptor. Nothing is transposed in
// memory.
//
// Accumulation. The tensor core adds to its fp32 accumulators by truncation, which loses about K / 16 * 2^-24 of a sum of
// terms of one sign (measured here: 2.8e-5 relative at K = 7168, 2.2e-6 at 1024). So it accumulates `chunk_steps` * 64 terms
// at a time into one of two TMEM buffers, and the drain warps add those to fp32 accumulators in registers, rounded to
// nearest, while it fills the other: the error stays that of one chunk whatever K is. fp32 outputs take chunks of 512
// terms (1.1e-6 at worst). For outputs that are rounded to 16 bits (half a step is 4.9e-4 or 3.9e-3) chunks of 8192 terms
// (3.2e-5) change nothing, and the usual product is then one chunk: its epilogue has the whole next tile to run in. The exception is
// a relu whose z is kept for its gradient, which depends on z's sign: chunks of 512.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mgrouped_pair_kernel.cuh"

namespace agb {

constexpr int kStepK = 64;         // contraction elements per pipeline step: one 128-byte row of the swizzled tiles
constexpr int kChunkStepsFp32 = 8, kChunkSteps16Bit = 128;   // DenseParams::chunk_steps
constexpr int kTileA = 128;        // operand A rows per CTA = TMEM lanes

enum : int { T_BF16 = 0, T_FP16 = 1, T_FP32 = 2 };
enum : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

struct DenseParams {
  int rows_a, rows_b;        // extents of the product
  int steps;                 // ceil(K / kStepK)
  int chunk_steps;           // steps accumulated in TMEM before they are added to the registers
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

__device__ __forceinline__ void store_from_float(void* p, long long i, int type, float v) {
  if (type == T_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (type == T_FP16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float reciprocal(float x) {      // 1 ulp, 0 for infinity
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Phi(z) = erfc(-z / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (absolute error of erfc 1.5e-7): five products and one exponential
// without a branch; the library's function cost an epilogue twice its time. z Phi(z) is off by 2.2e-7 at most, which is what
// 1 + erf loses by cancellation in fp32, and by 5e-4 of itself down to z = -4. `bell` is exp(-z^2 / 2), which the density
// needs too.
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  bell = __expf(-0.5f * z * z);
  const float t = reciprocal(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
  float c = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
  c = fmaf(c, t, 0.5f * 1.421413741f);
  c = fmaf(c, t, 0.5f * -0.284496736f);
  c = fmaf(c, t, 0.5f * 0.254829592f);
  const float tail = c * t * bell;
  return z < 0.f ? tail : 1.f - tail;
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == ACT_RELU) return z < 0.f ? 0.f : z;                       // NaN stays NaN
  if (act == ACT_GELU) {
    float bell;
    return z * normal_cdf(z, bell);
  }
  if (act == ACT_SILU) return z * reciprocal(1.f + __expf(-z));
  return z;
}

// ------------------------------------------------------------------------------------------------ epilogue
// VW consecutive elements as the words they are in memory (fp32: VW words, 16 bits: (VW + 1) / 2), aligned to their size together.
// Loading and converting are apart so that many loads are under way before the first is waited for.
template <int VW, bool FP32>
__device__ __forceinline__ void load_raw(const void* at, uint32_t (&w)[VW]) {
  constexpr int kBytes = VW * (FP32 ? 4 : 2);
  if constexpr (kBytes == 16) {
    const uint4 u = __ldcs(static_cast<const uint4*>(at));
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (kBytes == 8) {
    const uint2 u = __ldcs(static_cast<const uint2*>(at));
    w[0] = u.x; w[1] = u.y;
  } else if constexpr (kBytes == 4) {
    w[0] = __ldcs(static_cast<const uint32_t*>(at));
  } else {
    w[0] = __ldcs(static_cast<const uint16_t*>(at));
  }
}
template <int VW>
__device__ __forceinline__ void store_pack(void* base, long long i, int type, const float (&v)[VW]) {
  if constexpr (VW == 1) {
    store_from_float(base, i, type, v[0]);
  } else if (type == T_FP32) {
    float* dst = static_cast<float*>(base) + i;
    if constexpr (VW == 4) __stcs(reinterpret_cast<float4*>(dst), make_float4(v[0], v[1], v[2], v[3]));
    else __stcs(reinterpret_cast<float2*>(dst), make_float2(v[0], v[1]));
  } else {
    uint32_t w[VW / 2];
#pragma unroll
    for (int j = 0; j < VW / 2; ++j) {
      if (type == T_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    uint16_t* dst = static_cast<uint16_t*>(base) + i;
    if constexpr (VW == 4) __stcs(reinterpret_cast<uint2*>(dst), make_uint2(w[0], w[1]));
    else __stcs(reinterpret_cast<uint32_t*>(dst), w[0]);
  }
}

template <int VW>
__device__ __forceinline__ void load_bias(const DenseParams& p, int n, float (&bias)[VW]) {
#pragma unroll
  for (int j = 0; j < VW; ++j) bias[j] = 0.f;
  if (p.bias == nullptr) return;
  if (p.bias_type == T_FP32) {
#pragma unroll
    for (int j = 0; j < VW; ++j) bias[j] = __ldg(static_cast<const float*>(p.bias) + n + j);
  } else {
    uint32_t raw[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) raw[j] = __ldg(static_cast<const uint16_t*>(p.bias) + n + j);
#pragma unroll
    for (int j = 0; j < VW; ++j)
      bias[j] = p.bias_type == T_BF16 ? __uint_as_float(raw[j] << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(raw[j])));
  }
}

// Epilogue of a lane's packs of VW columns n .. in the rows m + i * row_step below `rows`, i < PACKS: z = v + bias,
// y = act(z) + residual. Every choice (activation,
// types, what there is) is made once for all packs: a branch per pack would cost more than the arithmetic between them.
template <int VW, int PACKS>
__device__ __forceinline__ void load_residual(const DenseParams& p, int rows, int m, int row_step, int n, uint32_t (&raw)[PACKS][VW]) {
  if (p.residual == nullptr) return;
  auto all = [&](auto fp32) {
    constexpr bool kFp32 = decltype(fp32)::value;
    constexpr int kSize = kFp32 ? 4 : 2;
    const char* at = static_cast<const char*>(p.residual) + (m * p.ldr + n) * kSize;
    const long long step = row_step * p.ldr * kSize;
#pragma unroll
    for (int i = 0; i < PACKS; ++i, at += step)
      if (m + i * row_step < rows) load_raw<VW, kFp32>(at, raw[i]);
  };
  if (p.out_type == T_FP32) all(std::true_type{});
  else all(std::false_type{});
}
template <int VW, int PACKS>
__device__ __forceinline__ void store_packs(void* out, long long ld, int type, int m, int rows, int row_step, int n, const float (&v)[PACKS][VW]) {
  const int size = type == T_FP32 ? 4 : 2;
  char* at = static_cast<char*>(out) + (m * ld + n) * size;
  const long long step = row_step * ld * size;
  auto all = [&](auto t) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i, at += step)
      if (m + i * row_step < rows) store_pack<VW>(at, 0, decltype(t)::value, v[i]);
  };
  if (type == T_BF16) all(std::integral_constant<int, T_BF16>{});
  else if (type == T_FP16) all(std::integral_constant<int, T_FP16>{});
  else all(std::integral_constant<int, T_FP32>{});
}
template <int VW, int PACKS>
__device__ __forceinline__ void finish_packs(const DenseParams& p, void* out, int rows, int m, int row_step, int n, const float (&bias)[VW],
                                             const uint32_t (&residual)[PACKS][VW], float (&v)[PACKS][VW]) {
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < PACKS; ++i) {
#pragma unroll
      for (int j = 0; j < VW; ++j) v[i][j] = f(v[i][j], i, j);
    }
  };
  if (p.bias != nullptr) each([&](float z, int, int j) { return z + bias[j]; });
  if (p.pre != nullptr) store_packs<VW, PACKS>(p.pre, p.ldp, p.pre_type, m, rows, row_step, n, v);
  if (p.act == ACT_RELU) each([](float z, int, int) { return activate(z, ACT_RELU); });
  else if (p.act == ACT_GELU) each([](float z, int, int) { return activate(z, ACT_GELU); });
  else if (p.act == ACT_SILU) each([](float z, int, int) { return activate(z, ACT_SILU); });
  if (p.residual != nullptr) {
    // element j of the raw words: bits 16 (j & 1) .. of word j / 2
    auto bits = [&](int i, int j) { return residual[i][j / 2] >> (16 * (j & 1)); };
    if (p.out_type == T_FP32) each([&](float y, int i, int j) { return y + __uint_as_float(residual[i][j]); });
    else if (p.out_type == T_BF16) each([&](float y, int i, int j) { return y + __uint_as_float(bits(i, j) << 16); });
    else each([&](float y, int i, int j) { return y + __half2float(__ushort_as_half(static_cast<unsigned short>(bits(i, j)))); });
  }
  store_packs<VW, PACKS>(out, p.ldo, p.out_type, m, rows, row_step, n, v);
}

// ------------------------------------------------------------------------------------------------ operands
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

// A wait of a whole warp with one answer for all of it: a lane that gave up takes the others along, so that they meet at the
// warp's next synchronisation.
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity, const WaitCtx& c, int code) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, c, code));
}

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

template <int VW>
__device__ __forceinline__ void ld_cluster(uint32_t addr, float (&v)[VW]) {
  if constexpr (VW == 4)
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory");
}

// ------------------------------------------------------------------------------------------------ one tile per CTA
// 128 x BN tile per CTA, the contraction split over the CTAs of a cluster (1, 2, 4 or 8). The CTAs' partial tiles meet in
// shared memory: each sums an equal share of the tile over the cluster in the order of the splits (so the result does not
// depend on timing), applies the epilogue and stores it. No workspace, no atomics, one launch. Measured: 64 x 7168 x 2048
// 10.0 us, 4 x 256 x 7168 8.6, 128 x 1024 x 512 6.7: launch, pipeline fill, join and epilogue are most of these.
template <int BN>
constexpr int tile_stages() { return BN >= 128 ? 6 : BN == 64 ? 4 : 5; }   // BN <= 64: two CTAs fit on an SM

template <int BN>
struct TileSmem {
  static constexpr int stages = tile_stages<BN>();
  static constexpr int a_bytes = kTileA * 128, b_bytes = BN * 128, stage_bytes = a_bytes + b_bytes;
  // The fp32 tile takes the ring's place at the end, laid out like the output: rows of `cols` outputs, 4 more between rows so
  // that lanes on different rows start on different banks.
  __host__ __device__ static constexpr int pitch(bool swapped) { return (swapped ? kTileA : BN) + 4; }
  static constexpr int bar_off = stages * stage_bytes;
  static constexpr int total = bar_off + (2 * stages + 4) * 8 + 16;
  static constexpr int dyn_bytes = total + 1024;
  static_assert(kTileA * (BN + 4) * 4 <= bar_off && BN * (kTileA + 4) * 4 <= bar_off, "the fp32 tile must fit into the ring");
};

constexpr int kTileThreads = 256;

// This CTA's share of an output tile of ROWS x COLS at (m0, n0): the rows' packs of VW columns, each summed over the cluster's
// partial tiles in the order of the splits. A thread's packs lie in one column.
template <int VW, int ROWS, int COLS>
__device__ __forceinline__ void store_tile(const DenseParams& p, const float* tile, int split, int splits, int m0, int n0, int rows, int cols) {
  constexpr int kAcross = COLS / VW, kRowStep = kTileThreads / kAcross, kPitch = COLS + 4;
  constexpr int kPacks = ROWS / kRowStep < 4 ? (ROWS / kRowStep < 1 ? 1 : ROWS / kRowStep) : 4;
  const int share = ROWS / splits, row0 = split * share;
  const int col = static_cast<int>(threadIdx.x) % kAcross * VW, n = n0 + col;
  if (n >= cols) return;
  float bias[VW];
  load_bias<VW>(p, n, bias);
  const uint32_t base = smem_u32(tile);
  for (int r = static_cast<int>(threadIdx.x) / kAcross; r < share; r += kRowStep * kPacks) {
    const int m = m0 + row0 + r;
    const int live = min(rows, m0 + row0 + share);      // rows past this CTA's share or the output are left out
    if (m >= live) break;
    uint32_t residual[kPacks][VW];
    load_residual<VW, kPacks>(p, live, m, kRowStep, n, residual);
    float v[kPacks][VW];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
#pragma unroll
      for (int j = 0; j < VW; ++j) v[i][j] = 0.f;
    }
    for (int s = 0; s < splits; ++s) {
      const uint32_t at = map_to_cta(base, static_cast<uint32_t>(s)) + static_cast<uint32_t>(((row0 + r) * kPitch + col) * 4);
      float u[kPacks][VW];
#pragma unroll
      for (int i = 0; i < kPacks; ++i)
        if (r + i * kRowStep < share) ld_cluster<VW>(at + i * kRowStep * kPitch * 4, u[i]);
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
#pragma unroll
        for (int j = 0; j < VW; ++j) v[i][j] += u[i][j];
      }
    }
    finish_packs<VW, kPacks>(p, p.out, live, m, kRowStep, n, bias, residual, v);
  }
}

template <int BN>
__host__ __device__ constexpr uint32_t tile_tmem_cols() { return 2 * BN < 32 ? 32 : 2 * BN; }

template <int BN, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kTileThreads, BN >= 128 ? 1 : 2)
dense_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const DenseParams p, const int splits,
                  const int vector_width) {
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
  const int chunks = (steps + p.chunk_steps - 1) / p.chunk_steps;

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

  // The whole warp runs the loops of the two issuing roles and one elected lane issues: with control flow and addresses
  // uniform across the warp an MMA costs its issuer far less than from a lone thread's branch.
  if (warp == 0) {
    const bool issuer = elect_one();
    for (int i = 0; i < steps; ++i) {
      const int s = i % ST;
      if (!wait_bar_warp(&empty[s], ((i / ST) & 1) ^ 1, wc, ST_TIMEOUT_A_EMPTY)) break;
      if (!issuer) continue;
      mbar_arrive_expect_tx(&full[s], L::stage_bytes);
      uint8_t* dst = smem + s * L::stage_bytes;
      load_operand<A_MN, kTileA>(dst, &map_a, &full[s], a0, (step0 + i) * kStepK);
      load_operand<B_MN, BN>(dst + L::a_bytes, &map_b, &full[s], b0, (step0 + i) * kStepK);
    }
  } else if (warp == 1) {
    const bool issuer = elect_one();
    const uint64_t da0 = operand_desc<A_MN>(smem_u32(smem)), db0 = operand_desc<B_MN>(smem_u32(smem) + L::a_bytes);
    for (int i = 0, chunk = 0, j = 0; i < steps; ++i) {
      const int s = i % ST, slot = chunk & 1;
      if (j == 0 && !wait_bar_warp(&tm_empty[slot], ((chunk >> 1) & 1) ^ 1, wc, ST_TIMEOUT_TM_EMPTY)) break;
      if (!wait_bar_warp(&full[s], (i / ST) & 1, wc, ST_TIMEOUT_A_FULL)) break;
      tc_fence_after_sync();
      const uint64_t da = da0 + ((s * L::stage_bytes) >> 4), db = db0 + ((s * L::stage_bytes) >> 4);
      const bool last = j + 1 == p.chunk_steps || i == steps - 1;
      if (issuer) {
#pragma unroll
        for (int q = 0; q < kStepK / 16; ++q)
          umma<MmaKind::F16>(tmem_base + slot * BN, da + ((q * operand_k_bytes<A_MN>()) >> 4), db + ((q * operand_k_bytes<B_MN>()) >> 4),
                             p.idesc, j > 0 || q > 0);
        umma_commit(&empty[s]);
        if (last) umma_commit(&tm_full[slot]);
      }
      __syncwarp();
      chunk += last;
      j = last ? 0 : j + 1;
    }
  } else if (warp >= 4) {
    constexpr int W = BN < 32 ? BN : 32;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const int r = (warp & 3) * 32 + lane;
    // W columns of this lane's row into the fp32 tile
    auto put = [&](int c0, const float (&v)[W]) {
      if (p.swapped) {
#pragma unroll
        for (int c = 0; c < W; ++c) tile_smem[(c0 + c) * L::pitch(true) + r] = v[c];
      } else {
#pragma unroll
        for (int c = 0; c < W; c += 4)
          *reinterpret_cast<float4*>(tile_smem + r * L::pitch(false) + c0 + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
      }
    };
    [[maybe_unused]] float acc[BN];
    bool ok = true;
    for (int chunk = 0; chunk < chunks; ++chunk) {
      const int slot = chunk & 1;
      ok = wait_bar_warp(&tm_full[slot], (chunk >> 1) & 1, wc, ST_TIMEOUT_TM_FULL);
      if (!ok) break;
      tc_fence_after_sync();
      // once the last chunk is complete every load has landed and every MMA has read it, so the ring is free for the tile
      const bool last = chunk == chunks - 1;
#pragma unroll
      for (int c0 = 0; c0 < BN; c0 += W) {
        uint32_t u[W];
        tmem_ld_cols(lane_addr + slot * BN + c0, u);
        tmem_wait_ld_into(u);
        float v[W];
#pragma unroll
        for (int c = 0; c < W; ++c) {
          v[c] = chunk == 0 ? __uint_as_float(u[c]) : acc[c0 + c] + __uint_as_float(u[c]);
          acc[c0 + c] = v[c];
        }
        if (last) put(c0, v);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tm_empty[slot]);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (splits > 1) cluster_sync_all();
  tc_fence_after_sync();
  if (*abort_flag) {
    // loads of this CTA may still be on their way into its shared memory: they take a few microseconds
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  } else if (p.swapped) {
    if (vector_width == 4) store_tile<4, BN, kTileA>(p, tile_smem, split, splits, b0, a0, p.rows_b, p.rows_a);
    else store_tile<1, BN, kTileA>(p, tile_smem, split, splits, b0, a0, p.rows_b, p.rows_a);
  } else {
    if (vector_width == 4) store_tile<4, kTileA, BN>(p, tile_smem, split, splits, a0, b0, p.rows_a, p.rows_b);
    else store_tile<1, kTileA, BN>(p, tile_smem, split, splits, a0, b0, p.rows_a, p.rows_b);
  }
  __syncthreads();
  if (splits > 1) cluster_sync_all();        // no CTA leaves while another may read its tile
  if (warp == 2) tmem_dealloc(tmem_base, tile_tmem_cols<BN>());
}

// ------------------------------------------------------------------------------------------------ pairs of CTAs
// 256 x 256 tile per pair of CTAs (tcgen05.mma.cta_group::2): each CTA holds 128 rows of A, 128 of B's 256 rows and the 128 x 256
// accumulator of its own rows, so an SM fetches 64 operand bytes per 128-cycle MMA row of work where a 128 x 128 tile of one
// CTA fetches 128: what a product of this size is bound by otherwise is operand traffic out of L2. Persistent: pairs take
// (tile, split of the contraction) items in turn, in blocks of 8 tile rows so that the tiles under way together share
// operands in L2. The drain's last pass over a tile -- bias, activation, residual, stores -- runs while the MMAs fill the
// two TMEM buffers of the next tile.
// With splits > 1 every split writes its fp32 partial to a workspace plane of its own and join_splits_kernel adds them in order.
// Measured: 8192 x 4096 x 7168 bf16 with silu 312 us (1540 TFLOP/s) in short runs, 388 under the power cap; 16384 x 256 x 7168 with
// fp32 outputs 57 us (39 of memory traffic; 64 tiles on 74 pairs, which pull 695 MB through L2); 2048 x 256 x 65536 split over 8:
// 62 us and 8 more for the join.
constexpr int kPairTile = 256, kPairStages = 6, kPairRowBlock = 8;
struct PairDenseSmem {
  static constexpr int box_bytes = 128 * 128;                    // one CTA's 128 rows of an operand, one step
  static constexpr int stage_bytes = 2 * box_bytes;
  static constexpr int turn_off = kPairStages * stage_bytes;     // per drain warp: a TurnBlock
  static constexpr int bar_off = turn_off + 8 * 32 * 32 * 4;
  static constexpr int total = bar_off + (2 * kPairStages + 6) * 8 + 16;
  static constexpr int dyn_bytes = total + 1024;
};
static_assert(PairDenseSmem::dyn_bytes <= 232448, "pair configuration does not fit in shared memory");

struct PairItem {
  int a0, b0, step0, steps, split;
};
__device__ __forceinline__ PairItem pair_item(const DenseParams& p, int w, int tiles_a, int splits) {
  PairItem it;
  it.split = w % splits;
  const int tile = w / splits;
  const int per_block = kPairRowBlock * p.tiles_b;
  const int block = tile / per_block, in = tile - block * per_block;
  const int rows = min(kPairRowBlock, tiles_a - block * kPairRowBlock);
  it.a0 = (block * kPairRowBlock + in % rows) * kPairTile;
  it.b0 = in / rows * kPairTile;
  it.step0 = static_cast<int>(static_cast<long long>(p.steps) * it.split / splits);
  it.steps = static_cast<int>(static_cast<long long>(p.steps) * (it.split + 1) / splits) - it.step0;
  return it;
}

// 32 rows x 32 columns of fp32 per drain warp, turned from row-per-lane (as TMEM gives them) to column-per-lane for coalesced
// stores. The 16-byte pieces of row r are at piece ^ (r & 7), which keeps the 16-byte accesses of both directions free of bank
// conflicts.
struct TurnBlock {
  float* base;
  __device__ __forceinline__ float* piece(int r, int c4) const { return base + r * 32 + ((c4 ^ (r & 7)) << 2); }
  __device__ __forceinline__ void put_row(int r, const uint32_t (&v)[32]) const {
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<uint4*>(piece(r, c)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
  }
  template <int VW>
  __device__ __forceinline__ void get(int r, int c, float (&v)[VW]) const {
    const float* at = piece(r, c >> 2) + (c & 3);
    if constexpr (VW == 4) {
      const float4 u = *reinterpret_cast<const float4*>(at);
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else if constexpr (VW == 2) {
      const float2 u = *reinterpret_cast<const float2*>(at);
      v[0] = u.x; v[1] = u.y;
    } else {
      v[0] = *at;
    }
  }
};

// One 32 x 32 block of a drain warp: 32 / VW lanes per row, VW rows per pass, kPacks passes at a time. `fill` puts the block into
// `turn`; the residual is on its way meanwhile.
template <int VW, int kPacks, typename Fill>
__device__ __forceinline__ void store_block(const DenseParams& p, void* out, const TurnBlock& turn, int lane, int m0, int n0, Fill fill) {
  constexpr int kLanes = 32 / VW;
  const int col = (lane % kLanes) * VW, n = n0 + col, row = lane / kLanes;
  const bool live = n < p.rows_b;
  float bias[VW];
  uint32_t residual[kPacks][VW];
  if (live) {
    load_bias<VW>(p, n, bias);
    load_residual<VW, kPacks>(p, p.rows_a, m0 + row, VW, n, residual);
  }
  fill();
  __syncwarp();
  if (live) {
#pragma unroll 1
    for (int r0 = 0; r0 < 32; r0 += kPacks * VW) {
      if (r0 > 0) load_residual<VW, kPacks>(p, p.rows_a, m0 + r0 + row, VW, n, residual);
      float v[kPacks][VW];
#pragma unroll
      for (int i = 0; i < kPacks; ++i) turn.get<VW>(r0 + i * VW + row, col, v[i]);
      finish_packs<VW, kPacks>(p, out, p.rows_a, m0 + r0 + row, VW, n, bias, residual, v);
    }
  }
  __syncwarp();
}

// ONE_CHUNK: no product of the launch has more steps than a chunk, so the drain needs no accumulators in registers.
template <bool A_MN, bool B_MN, bool ONE_CHUNK>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
dense_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const DenseParams params, const int splits,
                  const int vector_width) {
  using L = PairDenseSmem;
  constexpr int ST = kPairStages;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::bar_off);   // used in the first CTA: the bytes of both CTAs' loads
  uint64_t* empty = full + ST;                                       // in both: the MMA thread commits to both
  uint64_t* tm_full = empty + ST;                                    // in both
  uint64_t* tm_empty = tm_full + 2;                                  // in both: this CTA's drain warps are done with a buffer
  uint64_t* tm_empty_peer = tm_empty + 2;                            // used in the first CTA: the second CTA's are
  uint32_t* tmem_base_smem = reinterpret_cast<uint32_t*>(tm_empty_peer + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_smem + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_cta_rank();
  const int tiles_a = (params.rows_a + kPairTile - 1) / kPairTile;
  const int items = tiles_a * params.tiles_b * splits;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tm_full[i], 1); mbar_init(&tm_empty[i], 8); mbar_init(&tm_empty_peer[i], 1); }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 2) {
    tmem_alloc_pair(tmem_base_smem, 2 * kPairTile);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_base_smem;
  const WaitCtx wc{params.status, abort_flag, params.timeout_ns};

  if (warp == 0) {
    // ---------------------------------------------------------------- loads: this CTA's 128 rows of both operands
    {
      const bool issuer = elect_one();
      uint32_t it = 0;
      bool ok = true;
      for (int w = first; w < items && ok; w += stride) {
        const PairItem item = pair_item(params, w, tiles_a, splits);
        const int a = item.a0 + static_cast<int>(rank) * 128, b = item.b0 + static_cast<int>(rank) * 128;
        for (int i = 0; i < item.steps; ++i, ++it) {
          const uint32_t s = it % ST;
          ok = wait_bar_warp(&empty[s], ((it / ST) & 1) ^ 1, wc, ST_TIMEOUT_A_EMPTY);
          if (!ok) break;
          const uint32_t bar = map_to_cta(smem_u32(&full[s]), 0);
          uint8_t* dst = smem + s * L::stage_bytes;
          const int k = (item.step0 + i) * kStepK;
          if (!issuer) continue;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::stage_bytes);
          if constexpr (A_MN) {
            tma_load_2d_pair(dst, &map_a, bar, a, k);
            tma_load_2d_pair(dst + L::box_bytes / 2, &map_a, bar, a + 64, k);
          } else {
            tma_load_2d_pair(dst, &map_a, bar, k, a);
          }
          if constexpr (B_MN) {
            tma_load_2d_pair(dst + L::box_bytes, &map_b, bar, b, k);
            tma_load_2d_pair(dst + L::box_bytes + L::box_bytes / 2, &map_b, bar, b + 64, k);
          } else {
            tma_load_2d_pair(dst + L::box_bytes, &map_b, bar, k, b);
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issue, first CTA of the pair only
    if (rank == 0) {
      const bool issuer = elect_one();
      uint32_t it = 0, chunk = 0;
      bool ok = true;
      const uint64_t da0 = operand_desc<A_MN>(smem_u32(smem)), db0 = operand_desc<B_MN>(smem_u32(smem) + L::box_bytes);
      for (int w = first; w < items && ok; w += stride) {
        const PairItem item = pair_item(params, w, tiles_a, splits);
        for (int i = 0, j = 0; i < item.steps; ++i, ++it) {
          const uint32_t s = it % ST, slot = chunk & 1;
          if (j == 0) ok = wait_bar_warp(&tm_empty[slot], ((chunk >> 1) & 1) ^ 1, wc, ST_TIMEOUT_TM_EMPTY) &&
                           wait_bar_warp(&tm_empty_peer[slot], ((chunk >> 1) & 1) ^ 1, wc, ST_TIMEOUT_TM_EMPTY);
          if (ok) ok = wait_bar_warp(&full[s], (it / ST) & 1, wc, ST_TIMEOUT_A_FULL);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t da = da0 + ((s * L::stage_bytes) >> 4), db = db0 + ((s * L::stage_bytes) >> 4);
          const bool last = j + 1 == params.chunk_steps || i == item.steps - 1;
          if (issuer) {
#pragma unroll
            for (int q = 0; q < kStepK / 16; ++q)
              umma_pair<MmaKind::F16>(tmem_base + slot * kPairTile, da + ((q * operand_k_bytes<A_MN>()) >> 4), db + ((q * operand_k_bytes<B_MN>()) >> 4),
                                      params.idesc, j > 0 || q > 0);
            umma_commit_pair(&empty[s]);
            if (last) umma_commit_pair(&tm_full[slot]);
          }
          __syncwarp();
          chunk += last;
          j = last ? 0 : j + 1;
        }
      }
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- second CTA: pass "buffer drained" on to the first
    // An arrival on another CTA's barrier waits for all earlier stores of its thread. The drain warps have output stores under
    // way, so they arrive on their own CTA's barrier and this warp, which has none, carries the news over.
    if (rank == 1) {
      uint32_t chunk = 0;
      bool ok = true;
      for (int w = first; w < items && ok; w += stride) {
        const PairItem item = pair_item(params, w, tiles_a, splits);
        const int chunks = ONE_CHUNK ? 1 : (item.steps + params.chunk_steps - 1) / params.chunk_steps;
        for (int c = 0; c < chunks && ok; ++c, ++chunk) {
          const uint32_t slot = chunk & 1;
          ok = wait_bar_warp(&tm_empty[slot], (chunk >> 1) & 1, wc, ST_TIMEOUT_TM_EMPTY);
          if (ok && lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tm_empty_peer[slot]), 0));
          __syncwarp();
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- drain: this CTA's 128 rows, 128 columns per warpgroup
    const int q = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + half * 128;
    const TurnBlock turn{reinterpret_cast<float*>(smem + L::turn_off) + (warp - 4) * 32 * 32};
    uint32_t chunk = 0;
    bool ok = true;
    auto release = [&](uint32_t slot) {      // hand a TMEM buffer back to the MMA warp
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tm_empty[slot]);
    };
    for (int w = first; w < items && ok; w += stride) {
      const PairItem item = pair_item(params, w, tiles_a, splits);
      const int chunks = ONE_CHUNK ? 1 : (item.steps + params.chunk_steps - 1) / params.chunk_steps;
      [[maybe_unused]] float acc[ONE_CHUNK ? 1 : 128];
#pragma unroll
      for (float& v : acc) v = 0.f;
      uint32_t slot = 0;
      for (int c = 0; c < chunks; ++c, ++chunk) {
        slot = chunk & 1;
        ok = wait_bar_warp(&tm_full[slot], (chunk >> 1) & 1, wc, ST_TIMEOUT_TM_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        if constexpr (!ONE_CHUNK) {
          // the sum ends up in the last chunk's buffer, so that the epilogue below has the registers to itself
          const bool last = c == chunks - 1;
#pragma unroll
          for (int cc = 0; cc < 128; cc += 8) {
            uint32_t r[8];
            tmem_ld_cols(lane_addr + slot * kPairTile + cc, r);
            tmem_wait_ld_into(r);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[cc + i] += __uint_as_float(r[i]);
          }
          if (last) {
#pragma unroll
            for (int cc = 0; cc < 128; cc += 32) {
              uint32_t r[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(acc[cc + i]);
              tmem_st_32x32b_x32(lane_addr + slot * kPairTile + cc, r);
            }
          }
          if (last) tmem_wait_st();
          else release(slot);
        }
      }
      if (!ok) break;
      void* out = params.out;
      if (splits > 1) out = static_cast<float*>(params.out) + static_cast<long long>(item.split) * params.rows_a * params.ldo;
      const int m0 = item.a0 + static_cast<int>(rank) * 128 + q * 32, n0 = item.b0 + half * 128;
      uint32_t r[32];
      tmem_ld_32x32b_x32(lane_addr + slot * kPairTile, r);
#pragma unroll 1
      for (int cc = 0; cc < 128; cc += 32) {
        auto fill = [&] {
          tmem_wait_ld_into(r);
          turn.put_row(lane, r);
          // the next 32 columns are on their way while these are finished
          if (cc < 96) tmem_ld_32x32b_x32(lane_addr + slot * kPairTile + cc + 32, r);
          else release(slot);
        };
        if (vector_width == 4) store_block<4, 8>(params, out, turn, lane, m0, n0 + cc, fill);
        else if (vector_width == 2) store_block<2, 8>(params, out, turn, lane, m0, n0 + cc, fill);
        else store_block<1, 8>(params, out, turn, lane, m0, n0 + cc, fill);
      }
    }
  }

  if (*abort_flag) {
    // loads and MMAs of the pair may still be in flight, counted on barriers the second CTA cannot wait on: give them a fixed
    // 200 us (they take a few) before shared memory and TMEM are given back
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 200000ull) {
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc_pair(tmem_base, 2 * kPairTile);
}

// out = epilogue(sum of the splits' partials [splits, m, n], in order). VW columns per thread; bound by memory.
template <int VW>
__global__ void __launch_bounds__(256) join_splits_kernel(const float* __restrict__ partial, int splits, const DenseParams p) {
  const long long packs = static_cast<long long>(p.rows_b) / VW, plane = static_cast<long long>(p.rows_a) * p.rows_b;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= packs * p.rows_a) return;
  const long long m = i / packs, n = (i - m * packs) * VW;
  float v[1][VW], bias[VW];
  uint32_t residual[1][VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) v[0][j] = 0.f;
  load_bias<VW>(p, static_cast<int>(n), bias);
  load_residual<VW, 1>(p, p.rows_a, static_cast<int>(m), 1, static_cast<int>(n), residual);
  for (int s = 0; s < splits; ++s) {
    uint32_t u[VW];
    load_raw<VW, true>(partial + s * plane + m * p.rows_b + n, u);
#pragma unroll
    for (int j = 0; j < VW; ++j) v[0][j] += __uint_as_float(u[j]);
  }
  finish_packs<VW, 1>(p, p.out, p.rows_a, static_cast<int>(m), 1, static_cast<int>(n), bias, residual, v);
}

}  // namespace agb
