// Dense products of the layer around the grouped GEMMs (router logits, shared experts, projections): y = act(x W^T + b) + r and
// its gradients. Operands bf16 or fp16, fp32 accumulation, output in the operands' type or fp32; see dense_kernel.cuh.
#include "dense_kernel.cuh"

#include <atomic>

#include "../../include/asymgemm_b200.h"

int agb_fail(int code, const char* message);
int agb_device_sm_count(int* out);
int32_t* agb_default_status_word();
int agb_encode_16bit_2d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t rows, uint64_t pitch_bytes, uint32_t box_rows, const char* what);

namespace agb {

// ------------------------------------------------------------------------------------------------ gradient before the activation
// dz = dy * act'(z), rounded to the operands' type because the tensor core takes it as an operand of the two products that
// follow (half a step of that type per element, like the operands themselves), with rows padded to 16 bytes; and, in the
// same pass over dy, the column sums of the unrounded dz that make the bias gradient. A thread owns columns and walks rows,
// so the sums are fp32 additions in a fixed order: per block of rows here, over the blocks in column_sums_kernel.
// dy and z are read once, dz is written once: 7.5 us of memory traffic for 3990 x 2050 fp16, where gelu's slope makes the kernel
// bound by instructions instead (19.5 us, issue slots 66 % used).
constexpr int kDzCols = 256, kDzThreads = 256;

__device__ __forceinline__ float slope(float z, int act) {
  if (act == ACT_RELU) return z > 0.f ? 1.f : z != z ? z : 0.f;
  if (act == ACT_GELU) {
    float bell;
    const float cdf = normal_cdf(z, bell);
    return fmaf(z * 0.39894228f, bell, cdf);
  }
  if (act == ACT_SILU) {
    const float s = reciprocal(1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

struct DzParams {
  const void* dy;
  const void* pre;
  void* dz;             // or null: only the sums are wanted
  float* partial;       // [row blocks, n] or null
  long long m, n, ld_dy, ld_pre, ld_dz;
  int dy_type, type, act, rows_per_block;
};

// A thread's 8 columns are 8 / V pieces of V consecutive ones, 32 V columns apart: V = 8 for rows on 16-byte boundaries, 2 for rows
// on 4-byte ones, 1 for any. 3990 x 2050 fp16 with gelu: 57 us with a branch on the type at every element, 19.5 so.
template <int V, bool FP32>
__device__ __forceinline__ void load_columns(const void* row, long long n, long long c0, uint32_t (&raw)[8]) {
#pragma unroll
  for (int i = 0; i < 8 / V; ++i) {
    const long long c = c0 + 32 * V * i;
    if (c >= n) continue;
    if constexpr (FP32) {
      const uint32_t* src = static_cast<const uint32_t*>(row) + c;
      if constexpr (V == 8) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(src)), b = __ldcs(reinterpret_cast<const uint4*>(src) + 1);
        raw[0] = a.x; raw[1] = a.y; raw[2] = a.z; raw[3] = a.w; raw[4] = b.x; raw[5] = b.y; raw[6] = b.z; raw[7] = b.w;
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) raw[i * V + j] = __ldcs(src + j);
      }
    } else {
      const uint16_t* src = static_cast<const uint16_t*>(row) + c;
      if constexpr (V == 8) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(src));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j] = j % 2 == 0 ? w[j / 2] & 0xffffu : w[j / 2] >> 16;
      } else if constexpr (V == 2) {
        const uint32_t w = __ldcs(reinterpret_cast<const uint32_t*>(src));
        raw[2 * i] = w & 0xffffu;
        raw[2 * i + 1] = w >> 16;
      } else {
        raw[i] = __ldcs(src);
      }
    }
  }
}
__device__ __forceinline__ float from_bits(uint32_t raw, int type) {
  if (type == T_BF16) return __uint_as_float(raw << 16);
  if (type == T_FP16) return __half2float(__ushort_as_half(static_cast<unsigned short>(raw)));
  return __uint_as_float(raw);
}

template <int V>
__global__ void __launch_bounds__(kDzThreads) dz_kernel(const DzParams p) {
  __shared__ float sums[8][kDzCols];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long r0 = static_cast<long long>(blockIdx.y) * p.rows_per_block, r1 = min(r0 + p.rows_per_block, p.m);
  const long long c0 = static_cast<long long>(blockIdx.x) * kDzCols + tx * V;      // n is a multiple of V
  auto column = [&](int i) { return c0 + 32 * V * (i / V) + i % V; };
  const int dy_size = p.dy_type == T_FP32 ? 4 : 2;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  for (long long r = r0 + ty; r < r1; r += 8) {
    uint32_t graw[8], zraw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) graw[i] = zraw[i] = 0;
    const void* dy = static_cast<const char*>(p.dy) + r * p.ld_dy * dy_size;
    if (p.dy_type == T_FP32) load_columns<V, true>(dy, p.n, c0, graw);
    else load_columns<V, false>(dy, p.n, c0, graw);
    if (p.act != ACT_NONE) load_columns<V, false>(static_cast<const uint16_t*>(p.pre) + r * p.ld_pre, p.n, c0, zraw);
    float g[8];
    auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = f(i);
    };
    if (p.dy_type == T_BF16) each([&](int i) { return from_bits(graw[i], T_BF16); });
    else if (p.dy_type == T_FP16) each([&](int i) { return from_bits(graw[i], T_FP16); });
    else each([&](int i) { return from_bits(graw[i], T_FP32); });
    if (p.act != ACT_NONE) {
      float z[8];
      if (p.type == T_BF16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = from_bits(zraw[i], T_BF16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = from_bits(zraw[i], T_FP16);
      }
      if (p.act == ACT_RELU) each([&](int i) { return g[i] * slope(z[i], ACT_RELU); });
      else if (p.act == ACT_GELU) each([&](int i) { return g[i] * slope(z[i], ACT_GELU); });
      else each([&](int i) { return g[i] * slope(z[i], ACT_SILU); });
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] += g[i];
    if (p.dz != nullptr) {
      uint16_t* dst = static_cast<uint16_t*>(p.dz) + r * p.ld_dz;
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) {
        uint16_t h[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
          h[j] = p.type == T_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(g[i * V + j])) : __half_as_ushort(__float2half_rn(g[i * V + j]));
        const long long c = c0 + 32 * V * i;
        if (c >= p.n) continue;
        if constexpr (V == 8)
          *reinterpret_cast<uint4*>(dst + c) = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        else if constexpr (V == 2)
          *reinterpret_cast<uint32_t*>(dst + c) = h[0] | h[1] << 16;
        else
          dst[c] = h[0];
      }
    }
  }
  if (p.partial == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[ty][column(i) - static_cast<long long>(blockIdx.x) * kDzCols] = acc[i];
  __syncthreads();
  const long long c = static_cast<long long>(blockIdx.x) * kDzCols + threadIdx.x;
  if (c >= p.n) return;
  float s = 0.f;
#pragma unroll
  for (int y = 0; y < 8; ++y) s += sums[y][threadIdx.x];
  p.partial[blockIdx.y * p.n + c] = s;
}

// out[c] = sum over the row blocks of partial[., c]; 32 columns x 8 interleaved shares of the blocks per CTA, joined in order.
__global__ void __launch_bounds__(256) column_sums_kernel(const float* __restrict__ partial, long long blocks, long long n, void* out, int type) {
  __shared__ float sums[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long c = static_cast<long long>(blockIdx.x) * 32 + tx;
  float s = 0.f;
  if (c < n)
    for (long long b = ty; b < blocks; b += 8) s += partial[b * n + c];
  sums[ty][tx] = s;
  __syncthreads();
  if (ty != 0 || c >= n) return;
#pragma unroll
  for (int y = 1; y < 8; ++y) s += sums[y][tx];
  store_from_float(out, c, type, s);
}

}  // namespace agb

namespace {

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// An operand of a product: element (row, k) at p[row * ld + k], or, MN-major, at p[k * ld + row].
struct Operand {
  const void* p;
  int64_t ld, rows;
  bool mn;
  const char* what;
};

struct Plan {
  bool pair;        // 256 x 256 tiles on pairs of CTAs, else 128 x bn tiles
  int bn, splits;
  bool swapped;     // tiles of 128 x bn: A and B change places
};

// Tile and split of a product: the candidate that a simple model of its time (microseconds, fitted to a sweep over 54 shapes and 12
// plans, see the figures beside it) finds fastest.
//   pairs: a step takes 0.30 (0.28 is the tensor core's own time), a tile's epilogue 4.3 that overlaps the next tile's steps, a
//   launch 5; split, the fp32 planes are written and read at about 4 TB/s by a second kernel.
//   128 x bn: a step takes 0.21 (bn 16 .. 64) or 0.26 (128), limited by what an SM pulls out of L2, 1.6 times that where two
//   CTAs share an SM; a launch and its epilogue 4.3 + bn / 64; joining s splits 0.35 s.
// Measured at m, n, k (pairs / 128 x 128 / 128 x 64): 2048^3 17.5 / 28 / 26; 512, 2048, 2048 17.2 / 12.1 / 11.6; 128, 256, 7168
// 39 / 12.8 / 10.2; 64, 7168, 2048 at bn 64, 32, 16: 10.0, 11.0, 12.9.
Plan plan_product(const Operand& a, const Operand& b, int64_t steps, int sms) {
  Plan best{};
  double best_us = 1e30;
  auto consider = [&](const Plan& pl, double us) {
    if (us < best_us) {
      best = pl;
      best_us = us;
    }
  };
  auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
  const int64_t pair_tiles = up(a.rows, agb::kPairTile) * up(b.rows, agb::kPairTile);
  for (int s = 1; s <= 8 && (s == 1 || steps >= 8 * s); ++s) {
    const double waves = static_cast<double>(up(pair_tiles * s, sms / 2));
    const double loop = 0.30 * static_cast<double>(up(steps, s));
    const double join = s > 1 ? 3.0 + s * 8e-6 * static_cast<double>(a.rows) * static_cast<double>(b.rows) / 4.0 : 0.0;
    consider({true, agb::kPairTile, s, false}, 5.0 + (waves - 1) * (loop > 4.3 ? loop : 4.3) + loop + 4.3 + join);
  }
  // 128 x bn tiles exist with A MN-major, or both operands, not B alone; of two K-major operands either may be A
  for (int swapped = 0; swapped < 2; ++swapped) {
    if (a.mn == b.mn ? (a.mn && swapped) : swapped != (b.mn ? 1 : 0)) continue;
    const int64_t ra = swapped ? b.rows : a.rows, rb = swapped ? a.rows : b.rows;
    for (int bn = a.mn && b.mn ? 64 : 16; bn <= 128; bn *= 2) {
      if (!swapped && !b.mn && bn < 64) continue;      // rows of 16 outputs would be stored in 32-byte pieces
      if (bn > 64 && rb <= bn / 2) continue;
      const int64_t tiles = up(ra, agb::kTileA) * up(rb, bn);
      for (int s = 1; s <= 8 && (s == 1 || steps >= 4 * s); s *= 2) {
        const int64_t ctas = tiles * s;
        const bool shared = bn < 128 && ctas > sms;
        const double waves = static_cast<double>(up(ctas, bn < 128 ? 2 * sms : sms));
        const double step = (bn < 128 ? 0.21 : 0.26) * (shared ? 1.6 : 1.0);
        consider({false, bn, s, swapped != 0}, waves * (4.3 + bn / 64.0 + step * static_cast<double>(up(steps, s))) + (s > 1 ? 0.35 * s : 0.0));
      }
    }
  }
  return best;
}

template <typename K>
cudaError_t allow_shared_memory(K kernel, int bytes, std::atomic<bool> (&configured)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && configured[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_relaxed);
  return e;
}

template <bool A_MN, bool B_MN, bool ONE_CHUNK>
cudaError_t launch_pair_as(const CUtensorMap& ma, const CUtensorMap& mb, const agb::DenseParams& p, int splits, int vector_width, int sms, cudaStream_t stream) {
  auto kernel = agb::dense_pair_kernel<A_MN, B_MN, ONE_CHUNK>;
  static std::atomic<bool> configured[64];
  if (cudaError_t e = allow_shared_memory(kernel, agb::PairDenseSmem::dyn_bytes, configured)) return e;
  const int64_t items = (static_cast<int64_t>(p.rows_a) + agb::kPairTile - 1) / agb::kPairTile * p.tiles_b * splits;
  const int64_t pairs = sms / 2 < items ? sms / 2 : items;
  kernel<<<static_cast<unsigned>(2 * pairs), agb::PAIR_THREADS, agb::PairDenseSmem::dyn_bytes, stream>>>(ma, mb, p, splits, vector_width);
  return cudaGetLastError();
}

template <int BN, bool A_MN, bool B_MN>
cudaError_t launch_tile(const CUtensorMap& ma, const CUtensorMap& mb, const agb::DenseParams& p, int splits, int vector_width, cudaStream_t stream) {
  using L = agb::TileSmem<BN>;
  static_assert(L::dyn_bytes * (BN >= 128 ? 1 : 2) <= 232448, "tile configuration does not fit in shared memory");
  auto kernel = agb::dense_tile_kernel<BN, A_MN, B_MN>;
  static std::atomic<bool> configured[64];
  if (cudaError_t e = allow_shared_memory(kernel, L::dyn_bytes, configured)) return e;
  const int64_t tiles = (static_cast<int64_t>(p.rows_a) + agb::kTileA - 1) / agb::kTileA * p.tiles_b;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * splits));
  cfg.blockDim = dim3(agb::kTileThreads);
  cfg.dynamicSmemBytes = L::dyn_bytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, p, splits, vector_width);
}

int64_t steps_of(int64_t k) { return (k + agb::kStepK - 1) / agb::kStepK; }

template <bool A_MN, bool B_MN>
cudaError_t launch_pair(const CUtensorMap& ma, const CUtensorMap& mb, const agb::DenseParams& p, int splits, int vector_width, int sms, cudaStream_t stream) {
  return (p.steps + splits - 1) / splits <= p.chunk_steps ? launch_pair_as<A_MN, B_MN, true>(ma, mb, p, splits, vector_width, sms, stream)
                                                          : launch_pair_as<A_MN, B_MN, false>(ma, mb, p, splits, vector_width, sms, stream);
}

// Bytes of partial results a product needs: one fp32 plane per split of the pair kernel.
uint64_t product_workspace(const Operand& a, const Operand& b, int64_t k, int sms) {
  const Plan pl = plan_product(a, b, steps_of(k), sms);
  return pl.pair && pl.splits > 1 ? static_cast<uint64_t>(pl.splits) * a.rows * b.rows * 4 : 0;
}

// Columns a lane can write at once: rows of every output-shaped tensor aligned for them together.
int vector_width(const agb::DenseParams& p, int64_t n) {
  for (int vw = 4; vw > 1; vw /= 2) {
    auto fits = [&](const void* base, int64_t ld, int type) {
      const int64_t bytes = vw * (type == AG_T_FP32 ? 4 : 2);
      return base == nullptr || (reinterpret_cast<uintptr_t>(base) % bytes == 0 && ld * (type == AG_T_FP32 ? 4 : 2) % bytes == 0);
    };
    if (n % vw == 0 && fits(p.out, p.ldo, p.out_type) && fits(p.residual, p.ldr, p.out_type) && fits(p.pre, p.ldp, p.pre_type)) return vw;
  }
  return 1;
}

template <int VW>
void launch_join(const float* partial, int splits, const agb::DenseParams& p, cudaStream_t stream) {
  const int64_t packs = static_cast<int64_t>(p.rows_a) * (p.rows_b / VW);
  agb::join_splits_kernel<VW><<<static_cast<unsigned>((packs + 255) / 256), 256, 0, stream>>>(partial, splits, p);
}

// out[r, c] = sum_k a(r, k) b(c, k) with the epilogue that `p` names; the rest of DenseParams follows from the operands.
int run_product(Operand a, Operand b, int64_t k, int type, agb::DenseParams p, void* workspace, cudaStream_t stream) {
  int sms = 0;
  if (int rc = agb_device_sm_count(&sms)) return rc;
  const Plan pl = plan_product(a, b, steps_of(k), sms);
  if (pl.swapped) {
    const Operand t = a;
    a = b;
    b = t;
  }
  auto encode = [&](CUtensorMap* map, const Operand& o, int box_rows) {
    return o.mn ? agb_encode_16bit_2d(map, o.p, static_cast<uint64_t>(o.rows), static_cast<uint64_t>(k), static_cast<uint64_t>(o.ld) * 2, agb::kStepK, o.what)
                : agb_encode_16bit_2d(map, o.p, static_cast<uint64_t>(k), static_cast<uint64_t>(o.rows), static_cast<uint64_t>(o.ld) * 2,
                                      static_cast<uint32_t>(box_rows), o.what);
  };
  CUtensorMap ma, mb;
  if (int rc = encode(&ma, a, agb::kTileA)) return rc;
  if (int rc = encode(&mb, b, pl.pair ? 128 : pl.bn)) return rc;
  p.rows_a = static_cast<int>(a.rows);
  p.rows_b = static_cast<int>(b.rows);
  p.steps = static_cast<int>(steps_of(k));
  // relu's slope turns on the sign of z, which the error of a long run flips for a few in a million -- 1.3e-3 of the gradient, where the
  // roundings to 16 bits make 2e-4. Runs of 512 flip as few as an fp32 product does (2000 x 2048 x 4096: 1 sign, 6 in one run of all);
  // 4096 x 4096 x 7168 takes 184 us so, and silu in one run 177.
  const bool sign_matters = p.act == agb::ACT_RELU && p.pre != nullptr;
  p.chunk_steps = p.out_type == AG_T_FP32 || sign_matters ? agb::kChunkStepsFp32 : agb::kChunkSteps16Bit;
  p.tiles_b = static_cast<int>((b.rows + pl.bn - 1) / pl.bn);
  p.swapped = pl.swapped;
  // operand format 0 = fp16, 1 = bf16; bits 15 and 16: A, B are MN-major
  const uint32_t format = type == AG_T_BF16 ? 1u : 0u;
  p.idesc = (pl.pair ? agb::make_idesc_pair(1, format, agb::kPairTile) : agb::make_idesc(1, format, static_cast<uint32_t>(pl.bn))) |
            (a.mn ? 1u << 15 : 0u) | (b.mn ? 1u << 16 : 0u);
  cudaError_t e = cudaErrorInvalidValue;
  const int64_t out_cols = pl.swapped ? a.rows : b.rows;
  int vw = vector_width(p, out_cols);
  if (pl.pair) {
    agb::DenseParams q = p;
    if (pl.splits > 1) {      // raw partials now, the epilogue when they are joined
      q.bias = q.residual = nullptr;
      q.pre = nullptr;
      q.act = agb::ACT_NONE;
      q.out = workspace;
      q.ldo = b.rows;
      q.out_type = AG_T_FP32;
    }
    const int join_vw = vw;
    vw = vector_width(q, out_cols);
    if (!a.mn && !b.mn) e = launch_pair<false, false>(ma, mb, q, pl.splits, vw, sms, stream);
    else if (!a.mn) e = launch_pair<false, true>(ma, mb, q, pl.splits, vw, sms, stream);
    else if (b.mn) e = launch_pair<true, true>(ma, mb, q, pl.splits, vw, sms, stream);
    if (e == cudaSuccess && pl.splits > 1) {
      if (join_vw == 4) launch_join<4>(static_cast<const float*>(workspace), pl.splits, p, stream);
      else if (join_vw == 2) launch_join<2>(static_cast<const float*>(workspace), pl.splits, p, stream);
      else launch_join<1>(static_cast<const float*>(workspace), pl.splits, p, stream);
      e = cudaGetLastError();
    }
  } else if (!a.mn && !b.mn) {
    if (pl.bn == 16) e = launch_tile<16, false, false>(ma, mb, p, pl.splits, vw, stream);
    else if (pl.bn == 32) e = launch_tile<32, false, false>(ma, mb, p, pl.splits, vw, stream);
    else if (pl.bn == 64) e = launch_tile<64, false, false>(ma, mb, p, pl.splits, vw, stream);
    else e = launch_tile<128, false, false>(ma, mb, p, pl.splits, vw, stream);
  } else if (!b.mn) {
    if (pl.bn == 16) e = launch_tile<16, true, false>(ma, mb, p, pl.splits, vw, stream);
    else if (pl.bn == 32) e = launch_tile<32, true, false>(ma, mb, p, pl.splits, vw, stream);
    else if (pl.bn == 64) e = launch_tile<64, true, false>(ma, mb, p, pl.splits, vw, stream);
    else e = launch_tile<128, true, false>(ma, mb, p, pl.splits, vw, stream);
  } else {
    if (pl.bn == 64) e = launch_tile<64, true, true>(ma, mb, p, pl.splits, vw, stream);
    else e = launch_tile<128, true, true>(ma, mb, p, pl.splits, vw, stream);
  }
  return e == cudaSuccess ? AG_OK : agb_fail(AG_E_CUDA, cudaGetErrorString(e));
}

int size_of(int type) { return type == AG_T_FP32 ? 4 : 2; }

int check_common(const ag_linear_desc_t* g) {
  if (g == nullptr) return agb_fail(AG_E_INVALID, "desc is NULL");
  if (g->dtype != AG_T_BF16 && g->dtype != AG_T_FP16) return agb_fail(AG_E_INVALID, "x and weight must be bf16 or fp16");
  if (g->out_dtype != g->dtype && g->out_dtype != AG_T_FP32) return agb_fail(AG_E_INVALID, "the output is of the operands' type or fp32");
  if (g->bias_dtype != g->dtype && g->bias_dtype != AG_T_FP32) return agb_fail(AG_E_INVALID, "the bias is of the operands' type or fp32");
  if (g->activation < AG_ACT_NONE || g->activation > AG_ACT_SILU) return agb_fail(AG_E_INVALID, "unknown activation");
  if (g->m < 0 || g->n <= 0 || g->k <= 0 || g->m > 0x7fffff00LL || g->n > 0x7fffff00LL || g->k > 0x7fffff00LL) return agb_fail(AG_E_INVALID, "bad sizes");
  if (g->k % 8 != 0) return agb_fail(AG_E_INVALID, "k must be a multiple of 8 (16-byte rows)");
  if (g->ldw < g->k || g->ldw % 8 != 0 || (g->m > 0 && (g->ldx < g->k || g->ldx % 8 != 0)))
    return agb_fail(AG_E_INVALID, "rows of x and weight must start on 16-byte boundaries and not overlap");
  if (!aligned_to(g->x, 16) || !aligned_to(g->weight, 16)) return agb_fail(AG_E_INVALID, "x and weight must be 16-byte aligned");
  return AG_OK;
}

// How the gradient before the activation is had: as dy itself where the products can take that, else from dz_kernel.
bool needs_dz(const ag_linear_desc_t* g) {
  return g->activation != AG_ACT_NONE || g->out_dtype != g->dtype || g->lddy % 8 != 0 || !aligned_to(g->dy, 16);
}
int64_t dz_ld(const ag_linear_desc_t* g) { return (g->n + 7) / 8 * 8; }
// Rows per block of dz_kernel: enough blocks to fill the GPU a few times, and no more partial sums than 512 blocks make.
int64_t dz_rows(const ag_linear_desc_t* g) {
  const int64_t col_blocks = (g->n + agb::kDzCols - 1) / agb::kDzCols;
  int64_t rows = (g->m * col_blocks + 1183) / 1184;
  if (rows < (g->m + 511) / 512) rows = (g->m + 511) / 512;
  return (rows < 8 ? 8 : rows + 7) / 8 * 8;
}
uint64_t align256(uint64_t v) { return (v + 255) / 256 * 256; }

// The three products; dz [m, n] with rows `ld` apart.
Operand x_rows(const ag_linear_desc_t* g) { return {g->x, g->ldx, g->m, false, "x"}; }
Operand weight_rows(const ag_linear_desc_t* g) { return {g->weight, g->ldw, g->n, false, "weight"}; }
Operand weight_columns(const ag_linear_desc_t* g) { return {g->weight, g->ldw, g->k, true, "weight"}; }
Operand x_columns(const ag_linear_desc_t* g) { return {g->x, g->ldx, g->k, true, "x"}; }
Operand dz_by_row(const ag_linear_desc_t* g, const void* dz, int64_t ld) { return {dz, ld, g->m, false, "dz"}; }
Operand dz_by_column(const ag_linear_desc_t* g, const void* dz, int64_t ld) { return {dz, ld, g->n, true, "dz"}; }

struct BackwardSpace {
  uint64_t dz, partial, product, total;     // product: shared by the two products, which run one after the other
};
BackwardSpace backward_space(const ag_linear_desc_t* g, int sms) {
  BackwardSpace s{};
  if (needs_dz(g) && (g->dx != nullptr || g->dweight != nullptr)) s.dz = align256(static_cast<uint64_t>(g->m) * dz_ld(g) * 2);
  if (g->dbias != nullptr) s.partial = align256(static_cast<uint64_t>((g->m + dz_rows(g) - 1) / dz_rows(g)) * g->n * 4);
  if (g->dx != nullptr) s.product = product_workspace(dz_by_row(g, nullptr, 0), weight_columns(g), g->n, sms);
  if (g->dweight != nullptr) {
    const uint64_t need = product_workspace(dz_by_column(g, nullptr, 0), x_columns(g), g->m, sms);
    if (need > s.product) s.product = need;
  }
  s.total = s.dz + s.partial + s.product;
  return s;
}

agb::DenseParams plain_output(const ag_linear_desc_t* g, void* out, int64_t ld, int type) {
  agb::DenseParams p{};
  p.out = out;
  p.ldo = ld;
  p.out_type = type;
  p.status = g->status != nullptr ? g->status : agb_default_status_word();
  p.timeout_ns = static_cast<unsigned long long>(g->timeout_ms ? g->timeout_ms : 4000u) * 1000000ull;
  return p;
}

}  // namespace

extern "C" {

uint64_t ag_linear_desc_size(void) { return sizeof(ag_linear_desc_t); }

int ag_linear(const ag_linear_desc_t* g) {
  if (int rc = check_common(g)) return rc;
  if (g->m == 0) return AG_OK;
  if (g->x == nullptr || g->weight == nullptr || g->y == nullptr) return agb_fail(AG_E_INVALID, "x, weight and y must be non-NULL");
  const int out_size = size_of(g->out_dtype);
  if (g->ldy < g->n || (g->residual != nullptr && g->ldr < g->n) || (g->pre != nullptr && g->ldp < g->n))
    return agb_fail(AG_E_INVALID, "rows of y, residual and pre must not overlap");
  if (!aligned_to(g->y, out_size) || !aligned_to(g->residual, out_size) || !aligned_to(g->pre, 2) || !aligned_to(g->bias, size_of(g->bias_dtype)))
    return agb_fail(AG_E_INVALID, "pointers must be aligned to their element type");
  agb::DenseParams p = plain_output(g, g->y, g->ldy, g->out_dtype);
  if (p.status == nullptr) return agb_fail(AG_E_CUDA, "no status word");
  p.bias = g->bias;
  p.bias_type = g->bias_dtype;
  p.residual = g->residual;
  p.ldr = g->ldr;
  p.pre = g->pre;
  p.ldp = g->ldp;
  p.pre_type = g->dtype;
  p.act = g->activation;
  int sms = 0;
  if (int rc = agb_device_sm_count(&sms)) return rc;
  const uint64_t need = product_workspace(x_rows(g), weight_rows(g), g->k, sms);
  if (need > 0 && (g->workspace == nullptr || g->workspace_bytes < need || !aligned_to(g->workspace, 256)))
    return agb_fail(AG_E_INVALID, "workspace too small or not 256-byte aligned (ag_linear_workspace_bytes)");
  return run_product(x_rows(g), weight_rows(g), g->k, g->dtype, p, g->workspace, static_cast<cudaStream_t>(g->stream));
}

uint64_t ag_linear_workspace_bytes(const ag_linear_desc_t* g, int32_t backward) {
  int sms = 0;
  if (check_common(g) != AG_OK || g->m == 0 || agb_device_sm_count(&sms) != AG_OK) return 0;
  return backward ? backward_space(g, sms).total : product_workspace(x_rows(g), weight_rows(g), g->k, sms);
}

int ag_linear_backward(const ag_linear_desc_t* g) {
  if (int rc = check_common(g)) return rc;
  if (g->dx == nullptr && g->dweight == nullptr && g->dbias == nullptr) return AG_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(g->stream);
  if (!aligned_to(g->dbias, size_of(g->bias_dtype)) || !aligned_to(g->dx, 2) || !aligned_to(g->dweight, 2))
    return agb_fail(AG_E_INVALID, "pointers must be aligned to their element type");
  if (g->m == 0) {      // a sum over no rows
    cudaError_t e = cudaSuccess;
    if (g->dweight != nullptr) e = cudaMemsetAsync(g->dweight, 0, static_cast<size_t>(g->n) * g->k * 2, stream);
    if (e == cudaSuccess && g->dbias != nullptr) e = cudaMemsetAsync(g->dbias, 0, static_cast<size_t>(g->n) * size_of(g->bias_dtype), stream);
    return e == cudaSuccess ? AG_OK : agb_fail(AG_E_CUDA, cudaGetErrorString(e));
  }
  if (g->x == nullptr || g->weight == nullptr || g->dy == nullptr) return agb_fail(AG_E_INVALID, "x, weight and dy must be non-NULL");
  if (g->activation != AG_ACT_NONE && g->pre == nullptr) return agb_fail(AG_E_INVALID, "the gradient of an activation wants `pre` of the forward call");
  if (g->lddy < g->n || (g->pre != nullptr && g->ldp < g->n)) return agb_fail(AG_E_INVALID, "rows of dy and pre must not overlap");
  if (!aligned_to(g->dy, size_of(g->out_dtype)) || !aligned_to(g->pre, 2)) return agb_fail(AG_E_INVALID, "pointers must be aligned to their element type");
  int sms = 0;
  if (int rc = agb_device_sm_count(&sms)) return rc;
  const BackwardSpace space = backward_space(g, sms);
  if (space.total > 0 && (g->workspace == nullptr || g->workspace_bytes < space.total || !aligned_to(g->workspace, 256)))
    return agb_fail(AG_E_INVALID, "workspace too small or not 256-byte aligned (ag_linear_workspace_bytes)");

  const void* dz = g->dy;
  int64_t ld = g->lddy;
  if (space.dz > 0 || space.partial > 0) {
    agb::DzParams p{};
    p.dy = g->dy;
    p.pre = g->pre;
    p.m = g->m;
    p.n = g->n;
    p.ld_dy = g->lddy;
    p.ld_pre = g->ldp;
    p.dy_type = g->out_dtype;
    p.type = g->dtype;
    p.act = g->activation;
    p.rows_per_block = static_cast<int>(dz_rows(g));
    if (space.dz > 0) {
      dz = p.dz = g->workspace;
      ld = p.ld_dz = dz_ld(g);
    }
    if (space.partial > 0) p.partial = reinterpret_cast<float*>(static_cast<char*>(g->workspace) + space.dz);
    const int64_t blocks = (g->m + p.rows_per_block - 1) / p.rows_per_block;
    // the widest pieces that every row of dy, pre and dz allows (dz rows are padded to 16 bytes)
    auto fits = [&](int v) {
      const int dy_bytes = v * size_of(g->out_dtype) < 16 ? v * size_of(g->out_dtype) : 16;
      return g->n % v == 0 && aligned_to(g->dy, dy_bytes) && g->lddy * size_of(g->out_dtype) % dy_bytes == 0 &&
             (g->activation == AG_ACT_NONE || (aligned_to(g->pre, 2 * v) && g->ldp % v == 0));
    };
    const dim3 grid(static_cast<unsigned>((g->n + agb::kDzCols - 1) / agb::kDzCols), static_cast<unsigned>(blocks));
    if (fits(8)) agb::dz_kernel<8><<<grid, agb::kDzThreads, 0, stream>>>(p);
    else if (fits(2)) agb::dz_kernel<2><<<grid, agb::kDzThreads, 0, stream>>>(p);
    else agb::dz_kernel<1><<<grid, agb::kDzThreads, 0, stream>>>(p);
    if (g->dbias != nullptr)
      agb::column_sums_kernel<<<static_cast<unsigned>((g->n + 31) / 32), 256, 0, stream>>>(p.partial, blocks, g->n, g->dbias, g->bias_dtype);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return agb_fail(AG_E_CUDA, cudaGetErrorString(e));
  }
  void* product_space = static_cast<char*>(g->workspace) + space.dz + space.partial;
  if (g->dx != nullptr) {      // dx[m, k] = sum_n dz[m, n] W[n, k]
    agb::DenseParams p = plain_output(g, g->dx, g->k, g->dtype);
    if (p.status == nullptr) return agb_fail(AG_E_CUDA, "no status word");
    if (int rc = run_product(dz_by_row(g, dz, ld), weight_columns(g), g->n, g->dtype, p, product_space, stream)) return rc;
  }
  if (g->dweight != nullptr) {      // dW[n, k] = sum_m dz[m, n] x[m, k]
    agb::DenseParams p = plain_output(g, g->dweight, g->k, g->dtype);
    if (p.status == nullptr) return agb_fail(AG_E_CUDA, "no status word");
    if (int rc = run_product(dz_by_column(g, dz, ld), x_columns(g), g->m, g->dtype, p, product_space, stream)) return rc;
  }
  return AG_OK;
}

}  // extern "C"
