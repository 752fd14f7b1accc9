// Matrix products with bias, activation and residual in the epilogue, and their gradient.
//
//   z = op(a) op(b) + bias          op(a) [m, k], op(b) [k, n]
//   y = act(z) + residual           act in {identity, relu, sigmoid, silu, gelu}
//
// 16-bit factors (half, bfloat16), or e4m3 factors with one fp32 scale per row of a and
// per column of the product.  The products run on the tensor cores (tcgen05, fp32
// accumulators in tensor memory), fed by TMA through a ring of shared-memory stages;
// everything after the product is fp32 arithmetic on the accumulators, rounded once.
// A factor stored transposed is read as it lies: the matrix instructions take both
// orders.  A factor whose lines do not start on 16-byte boundaries, which TMA cannot
// address, is first copied to lines that do.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "matmul.h"
#include "partial_rows.cuh"
#include "tcgen05_dev.cuh"
#include "trace.h"
#include "tuning.h"
#include "../../include/musa_plugin_kernels.h"

namespace musa_b200 {
namespace {

// Set by a kernel whose wait ran out (see BarWait); read by MusaMatMulStatus.
__device__ int g_status;

// ------------------------------------------------------------- activations --

// The 16-bit outputs keep 8 or 11 bits; the hardware exp2 and reciprocal are good to about
// 2^-22.
__device__ __forceinline__ float Exp2Of(float v) {
  float out;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(out) : "f"(v));
  return out;
}
__device__ __forceinline__ float ReciprocalOf(float v) {
  float out;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(out) : "f"(v));
  return out;
}
constexpr float kLog2E = 1.44269504f;

__device__ __forceinline__ float2 SigmoidOf(float2 z) {
  const float2 p = Mul2(z, make_float2(-kLog2E, -kLog2E));
  const float2 d = Add2(make_float2(Exp2Of(p.x), Exp2Of(p.y)), make_float2(1.0f, 1.0f));
  return make_float2(ReciprocalOf(d.x), ReciprocalOf(d.y));
}

// Phi(-|z|), and exp(-z^2 / 2) in `*bell`.  Hastings' rational form of the error function
// (Abramowitz and Stegun 7.1.26): with t = 1 / (1 + p |z| / sqrt 2), erfc(|z| / sqrt 2) is
// a polynomial of degree five in t times the bell, to 1.5e-7 (the polynomial alone; with the
// roundings of fp32 and the two hardware functions z Phi(z) is off by up to 8e-7 of |z|).  The
// bound is absolute: where the value itself is small, below z = -5, it is good to 0.4 % down to
// -6 and to 1 % down to -8 (an fp32 1 + erf has lost it all there).  erff, which takes a branch at
// 1 and some 40 instructions, made the epilogue of a tile three times as long (8192 x 16384
// outputs of depth 64: 225 us against 108 without an activation).
__device__ __forceinline__ float2 NormalTail(float2 z, float2* bell) {
  constexpr float kP = 0.3275911f * 0.70710678f;
  const float2 t = make_float2(ReciprocalOf(fmaf(kP, fabsf(z.x), 1.0f)),
                               ReciprocalOf(fmaf(kP, fabsf(z.y), 1.0f)));
  const auto Both = [](float v) { return make_float2(v, v); };
  float2 q = Fma2(t, Both(0.5f * 1.061405429f), Both(0.5f * -1.453152027f));
  q = Fma2(t, q, Both(0.5f * 1.421413741f));
  q = Fma2(t, q, Both(0.5f * -0.284496736f));
  q = Fma2(t, q, Both(0.5f * 0.254829592f));
  const float2 w = Mul2(Mul2(z, z), Both(-0.5f * kLog2E));
  *bell = make_float2(Exp2Of(w.x), Exp2Of(w.y));
  return Mul2(Mul2(t, q), *bell);
}
// z Phi(z) = max(z, 0) - |z| Phi(-|z|); an infinite z times its tail of 0 is 0.
__device__ __forceinline__ float GeluOf(float z, float tail) {
  return fmaf(-fminf(fabsf(z), 1e30f), tail, fmaxf(z, 0.0f));
}

template <int kN>
__device__ __forceinline__ void Activate(float (&v)[kN], int act) {
  switch (act) {
    case MUSA_ACT_RELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // NaN goes through
      break;
    case MUSA_ACT_SIGMOID:
    case MUSA_ACT_SILU:
#pragma unroll
      for (int i = 0; i < kN; i += 2) {
        const float2 z = make_float2(v[i], v[i + 1]);
        float2 p = SigmoidOf(z);
        if (act == MUSA_ACT_SILU) p = Mul2(p, z);
        v[i] = p.x;
        v[i + 1] = p.y;
      }
      break;
    case MUSA_ACT_GELU:
#pragma unroll
      for (int i = 0; i < kN; i += 2) {
        float2 bell;
        const float2 tail = NormalTail(make_float2(v[i], v[i + 1]), &bell);
        v[i] = GeluOf(v[i], tail.x);
        v[i + 1] = GeluOf(v[i + 1], tail.y);
      }
      break;
    default:
      break;
  }
}

// act'(z) in place of z.
template <int kN>
__device__ __forceinline__ void Slopes(float2 (&z)[kN], int act) {
  const float2 one = make_float2(1.0f, 1.0f);
  switch (act) {
    case MUSA_ACT_RELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        z[i] = make_float2(z[i].x > 0.0f ? 1.0f : 0.0f, z[i].y > 0.0f ? 1.0f : 0.0f);
      }
      break;
    case MUSA_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float2 p = SigmoidOf(z[i]);
        z[i] = Mul2(p, Add2(one, Neg2(p)));
      }
      break;
    case MUSA_ACT_SILU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float2 p = SigmoidOf(z[i]);
        z[i] = Mul2(p, Fma2(z[i], Add2(one, Neg2(p)), one));
      }
      break;
    case MUSA_ACT_GELU:
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        float2 bell;
        const float2 tail = NormalTail(z[i], &bell);
        const float2 phi = make_float2(z[i].x < 0.0f ? tail.x : 1.0f - tail.x,
                                       z[i].y < 0.0f ? tail.y : 1.0f - tail.y);
        z[i] = Fma2(Mul2(z[i], make_float2(0.39894228f, 0.39894228f)), bell, phi);
      }
      break;
    default:
#pragma unroll
      for (int i = 0; i < kN; ++i) z[i] = one;
      break;
  }
}

// -------------------------------------------------------- products, any size --

// Tiles of 128 columns of the product (lanes of tensor memory) x `rows_tile` rows of it
// (columns of tensor memory).  The product is computed transposed: what is stored for one
// row of it by the 32 lanes of a warp is contiguous whatever n, alignment and pitch, and
// a product of few rows (decoding) asks for no more than it has: the weights are the
// instruction's 128-row side, the rows its 16 .. 256-column side.  A reduction is
// split over the CTAs of a cluster when the tiles alone do not fill the machine; their
// partial tiles meet in shared memory (each CTA adds, in rank order, and finishes its
// share of the rows), so there is no scratch, no second launch and no atomic.
constexpr int kDepthBytes = 128;    // of both factors per stage
constexpr int kSideBytes = 128 * kDepthBytes;
constexpr int kMaxStages = 12;
constexpr int kSplitThreads = 192;  // four warps for the epilogue, one for TMA, one for the MMA

struct SplitArgs {
  Epilogue e;
  int64_t m, n;
  int blocks;      // stages of depth in all
  int rows_tile;
  int stages;
  int stage_bytes;
  int splits;      // CTAs of the cluster
  uint32_t idesc;
  uint32_t tmem_columns;
  bool p_rows, q_rows;   // the factors' rows_contiguous
};

__device__ __forceinline__ float LoadClusterF32At(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// What the epilogue of rows row .. row + kN - 1 of column `col` reads: asked for ahead of the
// product, or of the chunk before.
template <typename T, int kN, bool kBytes>
struct ColumnInputs {
  float residual[kN], scale[kBytes ? kN : 1];
  __device__ __forceinline__ void Load(const SplitArgs& a, int64_t row, int rows, int64_t col) {
    const T* at = static_cast<const T*>(a.e.residual) + row * a.n + col;
    const bool add = a.e.residual != nullptr && col < a.n;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      residual[i] = add && i < rows ? ToF32(at[i * a.n]) : 0.0f;
      if constexpr (kBytes) scale[i] = i < rows ? a.e.a_scale[row + i] : 0.0f;
    }
  }
};

// The first `rows` of rows row .. row + kN - 1 of the product in column `col`: one value per
// lane and row.
template <typename T, int kN, bool kBytes>
__device__ __forceinline__ void FinishColumn(float (&v)[kN], const ColumnInputs<T, kN, kBytes>& in,
                                             int64_t row, int rows, int64_t col,
                                             const SplitArgs& a, float bias, float col_scale) {
  const Epilogue& e = a.e;
  const bool inside = col < a.n;
  T* y = static_cast<T*>(e.y) + row * a.n + col;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    // One scale after the other: the product of the two may leave fp32's range.
    if constexpr (kBytes) v[i] = v[i] * in.scale[i] * col_scale;
    v[i] += bias;
  }
  if (e.z != nullptr) {
    T* z = static_cast<T*>(e.z) + row * a.n + col;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      if (inside && i < rows) z[i * a.n] = FromF32<T>(v[i]);
    }
  }
  Activate(v, e.act);
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    if (inside && i < rows) y[i * a.n] = FromF32<T>(v[i] + in.residual[i]);
  }
}

// P: the factor of the product's columns (b), Q: that of its rows (a).
template <typename T, bool kBytes>
__global__ void __launch_bounds__(kSplitThreads)
    SplitProductKernel(const __grid_constant__ CUtensorMap p_map,
                       const __grid_constant__ CUtensorMap q_map,
                       const __grid_constant__ SplitArgs a) {
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
  __shared__ uint32_t tmem_at;
  __shared__ volatile int give_up;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t ring = (SmemAddr(dynamic) + 1023u) & ~1023u;
  const uint32_t rank = a.splits > 1 ? ClusterCtaRank() : 0;
  const int64_t col0 = static_cast<int64_t>(blockIdx.x) * 128;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * a.rows_tile;
  const int first = static_cast<int>(static_cast<int64_t>(a.blocks) * rank / a.splits);
  const int last = static_cast<int>(static_cast<int64_t>(a.blocks) * (rank + 1) / a.splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      BarInit(SmemAddr(&full[s]), 1);
      BarInit(SmemAddr(&empty[s]), 1);
    }
    BarInit(SmemAddr(&done), 1);
    give_up = 0;
    BarInitFence();
  }
  if (warp == 5) TmemAlloc<1>(SmemAddr(&tmem_at), a.tmem_columns);
  TmemFenceBefore();
  __syncthreads();
  TmemFenceAfter();
  const uint32_t tmem = tmem_at;
  bool ok = true;
  GridDepWait();
  GridDepLaunch();

  if (warp == 4) {
    constexpr int kDepth = kBytes ? kDepthBytes : kDepthBytes / 2;  // elements
    int s = 0, phase = 1;
    for (int i = first; i < last; ++i) {
      if (!BarWait(SmemAddr(&empty[s]), phase, &give_up, &g_status)) break;
      const uint32_t bar = SmemAddr(&full[s]);
      const uint32_t p = ring + s * a.stage_bytes, q = p + kSideBytes;
      const int depth = i * kDepth;
      if (ElectLane()) {
        BarExpect(bar, a.stage_bytes);
        if (a.p_rows) {
          for (int b = 0; b < 2; ++b) {
            TmaLoad<false>(p + b * kBlockBytes, &p_map, static_cast<int>(col0) + b * 64, depth,
                           bar);
          }
        } else {
          TmaLoad<false>(p, &p_map, depth, static_cast<int>(col0), bar);
        }
        if (a.q_rows) {
          for (int b = 0; b < a.rows_tile / 64; ++b) {
            TmaLoad<false>(q + b * kBlockBytes, &q_map, static_cast<int>(row0) + b * 64, depth,
                           bar);
          }
        } else {
          TmaLoad<false>(q, &q_map, depth, static_cast<int>(row0), bar);
        }
      }
      __syncwarp();
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 5 && last > first) {
    const uint32_t p_step = DepthStep(a.p_rows), q_step = DepthStep(a.q_rows);
    int s = 0, phase = 0;
    for (int i = first; i < last; ++i) {
      ok = BarWait(SmemAddr(&full[s]), phase, &give_up, &g_status);
      if (!ok) break;
      TmemFenceAfter();
      const uint32_t p = ring + s * a.stage_bytes;
      const uint64_t pd = OperandDesc(p, a.p_rows), qd = OperandDesc(p + kSideBytes, a.q_rows);
      if (ElectLane()) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Mma<1, kBytes>(tmem, pd + j * p_step, qd + j * q_step, a.idesc, i > first || j > 0);
        }
        MmaCommit<1>(SmemAddr(&empty[s]));
      }
      __syncwarp();
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (ok && ElectLane()) MmaCommit<1>(SmemAddr(&done));
  }
  __syncwarp();
  // This CTA's rows of the tile, in chunks: all of it, or its share of the cluster's.
  constexpr int kChunkRows = 16;
  const int share = a.rows_tile / a.splits;
  const int64_t my_row = row0 + rank * share;
  const int64_t left = a.m - my_row;
  const int rows = warp >= 4 || left <= 0 ? 0 : left < share ? static_cast<int>(left) : share;
  const int64_t col = col0 + warp * 32 + lane;
  float bias = 0.0f, col_scale = 1.0f;
  if (warp < 4 && col < a.n) {
    if (a.e.bias != nullptr) bias = ToF32(static_cast<const T*>(a.e.bias)[col]);
    if (kBytes) col_scale = a.e.b_scale[col];
  }
  ColumnInputs<T, kChunkRows, kBytes> in;
  in.Load(a, my_row, rows, col);
  if (warp < 4 && last > first) {
    ok = BarWait(SmemAddr(&done), 0, &give_up, &g_status);
    TmemFenceAfter();
  }
  const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  if (a.splits > 1) {
    // Partial tile [row][128 columns] over the ring: this CTA's copies and matrix
    // instructions are done.
    if (warp < 4 && ok) {
      for (int c = 0; c < a.rows_tile; c += 16) {
        float v[16];
        TmemLoad(lanes + c, v);
        TmemLoadWait(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(ring + ((c + i) * 128 + warp * 32 + lane) * 4),
                       "f"(v[i])
                       : "memory");
        }
      }
    }
    ClusterSync();
  }
  if (ok) {
    for (int c = 0; c < rows; c += kChunkRows) {
      float v[kChunkRows];
#pragma unroll
      for (int i = 0; i < kChunkRows; ++i) v[i] = 0.0f;
      if (a.splits > 1) {
        // In rank order.  Rows of the chunk behind the share are not asked for.
        const uint32_t mine =
            ring + ((static_cast<int>(rank) * share + c) * 128 + warp * 32 + lane) * 4;
#pragma unroll 2
        for (int s = 0; s < a.splits; ++s) {
          const uint32_t at = MapToCta(mine, s);
#pragma unroll
          for (int i = 0; i < kChunkRows; ++i) {
            if (c + i < rows) v[i] += LoadClusterF32At(at + i * 512);
          }
        }
      } else if (last > first) {
        TmemLoad(lanes + c, v);
        TmemLoadWait(v);
      }
      const ColumnInputs<T, kChunkRows, kBytes> now = in;
      const int next = c + kChunkRows;
      if (next < rows) in.Load(a, my_row + next, rows - next, col);
      FinishColumn<T>(v, now, my_row + c, rows - c, col, a, bias, col_scale);
    }
  }
  if (a.splits > 1) ClusterSync();
  TmemFenceBefore();
  __syncthreads();
  if (give_up != 0) LeaveInFlight();
  if (warp == 5) {
    TmemFenceAfter();
    TmemFree<1>(tmem, a.tmem_columns);
  }
}

// ------------------------------------------------------ products, large sizes --

// A pair of CTAs on two neighbouring SMs computes 256 x tile_n of the product: one matrix
// instruction covers both (each holds its 128 rows of a and half of b's tile in shared
// memory, and its 128 rows of the accumulator in tensor memory), so an operand byte is
// fetched half as often as by two single CTAs.  The pairs are persistent: TMA keeps a ring
// of six stages (32 KB per CTA) ahead, two accumulators alternate, and eight epilogue
// warps finish one tile while the next is multiplied.  Their two groups of four halve the
// columns and go 32 at a time: accumulator -> registers -> shared memory (the TMA's
// swizzled lines of 64 bytes) -> one TMA store; the residual comes the same way back.  Outputs that TMA cannot address
// (odd pitch or base) are moved element by element instead.
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * kSideBytes;
constexpr int kPairThreads = 384;    // TMA, MMA, tensor memory, idle; 4 .. 11 epilogue
constexpr int kChunk = 32;           // columns of the epilogue
constexpr int kStagingBytes = 128 * kChunk * 2;
constexpr int kPairSmem = kPairStages * kPairStageBytes + 4 * kStagingBytes + 1024;
constexpr int kBand = 8;             // tile rows walked together, for the L2

struct PairArgs {
  Epilogue e;
  int64_t m, n;
  int blocks;       // stages of depth
  int tile_n;       // 128 or 256
  int tiles_m, tiles_n;
  uint32_t idesc;
  bool a_rows, b_rows;
  bool direct;      // y, z and the residual without TMA
};

// Tile number -> tile row and column: bands of kBand tile rows, columns inside a band.
__device__ __forceinline__ void TileAt(int tile, const PairArgs& a, int* tm, int* tn) {
  const int per_band = kBand * a.tiles_n;
  const int band = tile / per_band, in = tile - band * per_band;
  const int height = min(kBand, a.tiles_m - band * kBand);
  *tn = in / height;
  *tm = band * kBand + in - *tn * height;
}

__device__ __forceinline__ void GroupBar(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
}

// 16-byte piece `piece` of line `line` of a tile of 64-byte lines with the 64-byte swizzle.
__device__ __forceinline__ uint32_t Swizzled(uint32_t base, int line, int piece) {
  return base + line * 64 + ((piece ^ ((line >> 1) & 3)) << 4);
}
__device__ __forceinline__ uint4 LoadShared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
__device__ __forceinline__ void StoreShared16(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}

// Eight fp32 values to a 16-byte piece.
template <typename T>
__device__ __forceinline__ void StorePiece(uint32_t at, const float* v) {
  Pack<T, 8> p;
  float2 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = make_float2(v[2 * i], v[2 * i + 1]);
  NarrowPack<8>(w, p);
  StoreShared16(at, *reinterpret_cast<const uint4*>(&p));
}

// A tile of up to 128 x kChunk elements between global memory and swizzled shared memory, by
// the 128 threads of a group: a warp a line, sixteen lines in flight (one after the other, the
// residual of a 333 x 2047 product took as long as the rest of it).
template <typename T, bool kToShared>
__device__ __forceinline__ void MoveTile(uint32_t tile, T* global, int64_t row0, int64_t col0,
                                         const PairArgs& a, int thread) {
  static_assert(kChunk == 32, "a lane per column");
  constexpr int kBatch = 16;
  const int c = thread % 32;
  const int64_t left = col0 + c < a.n ? a.m - row0 : 0;
  T* at = global + row0 * a.n + col0 + c;
  const auto Shared = [&](int line) { return Swizzled(tile, line, c >> 3) + (c & 7) * 2; };
  for (int first = thread / 32; first < 128; first += 4 * kBatch) {
    uint16_t v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int line = first + 4 * i;
      if constexpr (kToShared) {
        if (line < left) v[i] = *reinterpret_cast<const uint16_t*>(at + line * a.n);
      } else {
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v[i]) : "r"(Shared(line)) : "memory");
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int line = first + 4 * i;
      if (line < left) {
        if constexpr (kToShared) {
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(Shared(line)), "h"(v[i]) : "memory");
        } else {
          *reinterpret_cast<uint16_t*>(at + line * a.n) = v[i];
        }
      }
    }
  }
}

template <typename T, bool kBytes>
__global__ void __launch_bounds__(kPairThreads, 1)
    PairProductKernel(const __grid_constant__ CUtensorMap a_map,
                      const __grid_constant__ CUtensorMap b_map,
                      const __grid_constant__ CUtensorMap y_map,
                      const __grid_constant__ CUtensorMap z_map,
                      const __grid_constant__ CUtensorMap r_map,
                      const __grid_constant__ PairArgs a) {
  extern __shared__ uint8_t dynamic[];
  __shared__ uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2], loaded[2];
  __shared__ __align__(16) T bias_of[2][128];
  __shared__ __align__(16) float scale_of[2][kBytes ? 128 : 4];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int give_up;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const int rank = static_cast<int>(ClusterCtaRank());
  const uint32_t ring = (SmemAddr(dynamic) + 1023u) & ~1023u;
  const uint32_t staging = ring + kPairStages * kPairStageBytes;
  const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  const int tiles = a.tiles_m * a.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      BarInit(SmemAddr(&full[s]), 1);
      BarInit(SmemAddr(&empty[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      BarInit(SmemAddr(&acc_full[i]), 1);
      BarInit(SmemAddr(&acc_empty[i]), 16);  // the epilogue warps of both CTAs
      BarInit(SmemAddr(&loaded[i]), 1);
    }
    give_up = 0;
    BarInitFence();
  }
  if (warp == 2) TmemAlloc<2>(SmemAddr(&tmem_at), 512);
  TmemFenceBefore();
  __syncthreads();
  ClusterSync();  // the peer's barriers are initialised
  TmemFenceAfter();
  GridDepWait();
  GridDepLaunch();
  const uint32_t tmem = tmem_at;

  if (warp == 0) {
    constexpr int kDepth = kBytes ? kDepthBytes : kDepthBytes / 2;
    const int half_n = a.tile_n / 2;
    const uint32_t bytes = 2 * (kSideBytes + half_n * kDepthBytes);
    int s = 0, phase = 1, used = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      int tm, tn;
      TileAt(tile, a, &tm, &tn);
      const int row = tm * 256 + rank * 128, col = tn * a.tile_n + rank * half_n;
      for (int k = 0; k < a.blocks; ++k) {
        ok = BarWait(SmemAddr(&empty[s]), phase, &give_up, &g_status);
        if (!ok) break;
        const uint32_t at = ring + s * kPairStageBytes;
        const uint32_t bar = MapToCta(SmemAddr(&full[s]), 0);
        const int depth = k * kDepth;
        if (ElectLane()) {
          if (rank == 0) BarExpect(SmemAddr(&full[s]), bytes);
          if (a.a_rows) {
            for (int b = 0; b < 2; ++b) {
              TmaLoad<true>(at + b * kBlockBytes, &a_map, row + b * 64, depth, bar);
            }
          } else {
            TmaLoad<true>(at, &a_map, depth, row, bar);
          }
          if (a.b_rows) {
            for (int b = 0; b < half_n / 64; ++b) {
              TmaLoad<true>(at + kSideBytes + b * kBlockBytes, &b_map, col + b * 64, depth, bar);
            }
          } else {
            TmaLoad<true>(at + kSideBytes, &b_map, depth, col, bar);
          }
        }
        __syncwarp();
        used = min(used + 1, kPairStages);
        if (++s == kPairStages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
    // The last arrivals on this CTA's barriers, before it may leave.
    for (int i = 0; i < used && ok; ++i) {
      // The oldest of them first: stage s, or stage 0 where the ring was not filled.
      const int at = used == kPairStages ? (s + i) % kPairStages : i;
      const int turn = used == kPairStages && at >= s ? phase : phase ^ 1;
      ok = BarWait(SmemAddr(&empty[at]), turn, &give_up, &g_status);
    }
  } else if (warp == 1 && rank == 0) {
    const uint32_t a_step = DepthStep(a.a_rows), b_step = DepthStep(a.b_rows);
    int s = 0, phase = 0, turn = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs, ++turn) {
      const int buffer = turn & 1;
      ok = BarWait(SmemAddr(&acc_empty[buffer]), ((turn >> 1) & 1) ^ 1, &give_up, &g_status);
      if (!ok) break;
      TmemFenceAfter();
      const uint32_t acc = tmem + buffer * 256;
      for (int k = 0; k < a.blocks; ++k) {
        ok = BarWait(SmemAddr(&full[s]), phase, &give_up, &g_status);
        if (!ok) break;
        TmemFenceAfter();
        const uint32_t at = ring + s * kPairStageBytes;
        const uint64_t ad = OperandDesc(at, a.a_rows);
        const uint64_t bd = OperandDesc(at + kSideBytes, a.b_rows);
        if (ElectLane()) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            Mma<2, kBytes>(acc, ad + j * a_step, bd + j * b_step, a.idesc, k > 0 || j > 0);
          }
          MmaCommit<2>(SmemAddr(&empty[s]));
          if (k == a.blocks - 1) MmaCommit<2>(SmemAddr(&acc_full[buffer]));
        }
        __syncwarp();
        if (++s == kPairStages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp >= 4) {
    const Epilogue& e = a.e;
    const int group = (warp - 4) / 4, thread = threadIdx.x - 128 - group * 128;
    const int line = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    const bool keep = e.z != nullptr, add = e.residual != nullptr;
    int turn = 0, slot = 0, loads = 0;
    bool ok = true;
    // Threads of a group that gave up a wait go on (without stores): the others count on them
    // at the group's barriers, and every later wait ends at once.
    for (int tile = pair; tile < tiles; tile += pairs, ++turn) {
      int tm, tn;
      TileAt(tile, a, &tm, &tn);
      const int buffer = turn & 1;
      const int64_t row0 = static_cast<int64_t>(tm) * 256 + rank * 128;
      const float row_scale =
          kBytes && row0 + line < a.m ? e.a_scale[row0 + line] : 1.0f;
      const int columns = a.tile_n / 2;
      const int64_t first = static_cast<int64_t>(tn) * a.tile_n + group * columns;
      if (thread < columns) {
        const bool there = first + thread < a.n;
        bias_of[group][thread] =
            there && e.bias != nullptr ? static_cast<const T*>(e.bias)[first + thread]
                                       : FromF32<T>(0.0f);
        if (kBytes) scale_of[group][thread] = there ? e.b_scale[first + thread] : 1.0f;
      }
      ok = BarWait(SmemAddr(&acc_full[buffer]), (turn >> 1) & 1, &give_up, &g_status) && ok;
      __syncwarp();
      TmemFenceAfter();
      for (int c = 0; c < columns; c += kChunk) {
        const int64_t col0 = first + c;
        const bool inside = row0 < a.m && col0 < a.n;
        const uint32_t z_tile = staging + (group * 2 + (slot ^ 1)) * kStagingBytes;
        const uint32_t y_tile = staging + (group * 2 + slot) * kStagingBytes;
        if (!keep && inside) slot ^= 1;
        float v[kChunk];
        TmemLoad(lanes + buffer * 256 + group * columns + c, v);
        // The stores that last read these tiles are done with them.
        if (a.direct) {
          GroupBar(group);
          if (add && inside) {
            MoveTile<T, true>(y_tile, const_cast<T*>(static_cast<const T*>(e.residual)), row0,
                              col0, a, thread);
          }
        } else if (thread == 0) {
          if (keep) TmaStoreWaitRead<0>();
          else TmaStoreWaitRead<1>();
          if (add && inside) {
            BarExpect(SmemAddr(&loaded[group]), kStagingBytes);
            TmaLoad<false>(y_tile, &r_map, static_cast<int>(col0), static_cast<int>(row0),
                           SmemAddr(&loaded[group]));
          }
        }
        GroupBar(group);
        TmemLoadWait(v);
        if (c + kChunk >= columns) {
          // All of this warp's accumulator is in registers.
          TmemFenceBefore();
          __syncwarp();
          if (lane == 0) BarArriveCluster(MapToCta(SmemAddr(&acc_empty[buffer]), 0));
        }
#pragma unroll
        for (int i = 0; i < kChunk; i += 4) {
          float2 b[2];
          WidenPack<4>(*reinterpret_cast<const Pack<T, 4>*>(&bias_of[group][c + i]), b);
          if constexpr (kBytes) {
            const float4 w = *reinterpret_cast<const float4*>(&scale_of[group][c + i]);
            v[i] = v[i] * row_scale * w.x;
            v[i + 1] = v[i + 1] * row_scale * w.y;
            v[i + 2] = v[i + 2] * row_scale * w.z;
            v[i + 3] = v[i + 3] * row_scale * w.w;
          }
          v[i] += b[0].x;
          v[i + 1] += b[0].y;
          v[i + 2] += b[1].x;
          v[i + 3] += b[1].y;
        }
        if (keep) {
#pragma unroll
          for (int i = 0; i < kChunk / 8; ++i) {
            StorePiece<T>(Swizzled(z_tile, line, i), v + i * 8);
          }
        }
        Activate(v, e.act);
        if (add && inside && !a.direct) {
          ok = BarWait(SmemAddr(&loaded[group]), loads & 1, &give_up, &g_status) && ok;
          ++loads;
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
          const uint32_t at = Swizzled(y_tile, line, i);
          if (add) {
            const uint4 w = LoadShared16(at);
            float2 r[4];
            WidenPack<8>(*reinterpret_cast<const Pack<T, 8>*>(&w), r);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              v[i * 8 + 2 * q] += r[q].x;
              v[i * 8 + 2 * q + 1] += r[q].y;
            }
          }
          StorePiece<T>(at, v + i * 8);
        }
        if (a.direct) {
          GroupBar(group);
          if (inside) {
            if (keep) MoveTile<T, false>(z_tile, static_cast<T*>(e.z), row0, col0, a, thread);
            MoveTile<T, false>(y_tile, static_cast<T*>(e.y), row0, col0, a, thread);
          }
        } else {
          FenceAsyncShared();
          GroupBar(group);
          if (thread == 0 && inside && ok) {
            if (keep) TmaStore(&z_map, static_cast<int>(col0), static_cast<int>(row0), z_tile);
            TmaStore(&y_map, static_cast<int>(col0), static_cast<int>(row0), y_tile);
            TmaStoreCommit();
          }
        }
      }
      GroupBar(group);  // before the next tile's bias
    }
    if (thread == 0) TmaStoreWaitAll();
  }
  __syncwarp();
  TmemFenceBefore();
  __syncthreads();
  if (give_up != 0) LeaveInFlight();
  ClusterSync();  // nobody signals or reads a CTA that has left
  TmemFenceAfter();
  if (warp == 2) TmemFree<2>(tmem, 512);
}

// ---------------------------------------------------------------- factors --

// Lines of `columns` elements, `ld` apart, to lines `pitch` apart.
template <typename E>
__global__ void __launch_bounds__(256)
    RepitchKernel(const E* __restrict__ src, E* __restrict__ dst, int64_t lines, int64_t columns,
                  int64_t ld, int64_t pitch) {
  GridDepWait();
  GridDepLaunch();
  for (int64_t r = blockIdx.y; r < lines; r += gridDim.y) {
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c + i * 256 < columns) dst[r * pitch + c + i * 256] = src[r * ld + c + i * 256];
    }
  }
}

int64_t RoundUp(int64_t v, int64_t to) { return CeilDiv(v, to) * to; }

// A factor's lines in memory.
struct Lines {
  int64_t count, length;
};
Lines LinesOf(const Factor& f, int64_t rows, int64_t depth) {
  return f.rows_contiguous ? Lines{depth, rows} : Lines{rows, depth};
}

// TMA takes it as it lies: 16-byte aligned base and lines.
bool Addressable(const Factor& f, const Lines& l, int elem) {
  return Aligned16(f.p) && (l.count <= 1 || f.ld * elem % 16 == 0);
}

size_t RepitchBytes(const Factor& f, int64_t rows, int64_t depth, int elem) {
  const Lines l = LinesOf(f, rows, depth);
  // Lines of 8-bit factors have to run along the depth.
  if (l.count == 0 || l.length == 0 || Addressable(f, l, elem)) return 0;
  return static_cast<size_t>(RoundUp(l.length * elem, 16) * l.count + 16);
}

cudaError_t Repitch(Factor* f, int64_t rows, int64_t depth, int elem, uint8_t** workspace,
                    cudaStream_t stream) {
  const size_t bytes = RepitchBytes(*f, rows, depth, elem);
  if (bytes == 0) return cudaSuccess;
  const Lines l = LinesOf(*f, rows, depth);
  const int64_t pitch = RoundUp(l.length * elem, 16) / elem;
  const dim3 grid(static_cast<unsigned>(CeilDiv(l.length, 1024)),
                  static_cast<unsigned>(l.count < 32768 ? l.count : 32768));
  const cudaError_t rc =
      elem == 2 ? LaunchChained(true, RepitchKernel<uint16_t>, grid, dim3(256), 0, stream,
                                static_cast<const uint16_t*>(f->p),
                                reinterpret_cast<uint16_t*>(*workspace), l.count, l.length, f->ld,
                                pitch)
                : LaunchChained(true, RepitchKernel<uint8_t>, grid, dim3(256), 0, stream,
                                static_cast<const uint8_t*>(f->p), *workspace, l.count, l.length,
                                f->ld, pitch);
  f->p = *workspace;
  f->ld = pitch;
  *workspace += RoundUp(static_cast<int64_t>(bytes), 16);
  return rc;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn Encode() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return static_cast<EncodeFn>(nullptr);
    }
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A map over lines of memory with boxes of 128 (or 64) bytes x `box_lines`, swizzled over
// their width.
template <typename T>
constexpr CUtensorMapDataType kMapType = CU_TENSOR_MAP_DATA_TYPE_UINT8;
template <>
constexpr CUtensorMapDataType kMapType<__half> = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
template <>
constexpr CUtensorMapDataType kMapType<__nv_bfloat16> = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;

template <typename E>
bool MakeMap(CUtensorMap* map, const void* p, int64_t count, int64_t length, int64_t ld,
             int box_lines, int box_bytes = 128) {
  const EncodeFn encode = Encode();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(length), static_cast<cuuint64_t>(count)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(
      count > 1 ? ld * static_cast<int64_t>(sizeof(E)) : RoundUp(length * sizeof(E), 16))};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_bytes / sizeof(E)),
                             static_cast<cuuint32_t>(box_lines)};
  const cuuint32_t steps[2] = {1, 1};
  return encode(map, kMapType<E>, 2, const_cast<void*>(p), dims, strides, box, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE,
                box_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---------------------------------------------------------------- launches --

constexpr int kSplitSmem = 208 * 1024;  // for the stages of an SM's CTAs

int SplitCtasPerSm(int rows_tile) {
  return (kSideBytes + rows_tile * kDepthBytes) * 4 <= kSplitSmem / 2 ? 2 : 1;
}

template <typename T, bool kBytes>
int LaunchSplit(int64_t m, int64_t n, int64_t k, const Factor& fa, const Factor& fb,
                const Epilogue& e, int rows_tile, int splits, cudaStream_t stream) {
  using E = std::conditional_t<kBytes, uint8_t, T>;
  constexpr int kDepth = 128 / sizeof(E);
  SplitArgs a = {};
  a.e = e;
  a.m = m;
  a.n = n;
  a.blocks = static_cast<int>(CeilDiv(k, kDepth));
  a.p_rows = fb.rows_contiguous;
  a.q_rows = fa.rows_contiguous;
  a.rows_tile = rows_tile;
  a.splits = splits;
  a.stage_bytes = kSideBytes + a.rows_tile * kDepthBytes;
  // Copies in flight carry a CTA through its depth: all the shared memory where it has an SM
  // to itself, half where four stages fit that.  Clusters of eight that need eight whole SMs
  // each do not fill the machine (128 such CTAs took 20 us where 128 of half an SM took 12).
  const int64_t ctas = CeilDiv(n, 128) * CeilDiv(m, rows_tile) * splits;
  const bool whole = SplitCtasPerSm(rows_tile) == 1 || ctas <= SmCount() / (splits == 8 ? 2 : 1);
  const int budget = whole ? kSplitSmem : kSplitSmem / 2;
  a.stages = budget / a.stage_bytes;
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  a.tmem_columns = 32;
  while (a.tmem_columns < static_cast<uint32_t>(a.rows_tile)) a.tmem_columns *= 2;
  constexpr int kType = kBytes ? 0 : std::is_same_v<T, __nv_bfloat16> ? 1 : 0;
  a.idesc = InstructionDesc(kType, a.p_rows, a.q_rows, 128, a.rows_tile);
  CUtensorMap p_map, q_map;
  const Lines pl = LinesOf(fb, n, k), ql = LinesOf(fa, m, k);
  if (k > 0 && (!MakeMap<E>(&p_map, fb.p, pl.count, pl.length, fb.ld, a.p_rows ? 64 : 128) ||
                !MakeMap<E>(&q_map, fa.p, ql.count, ql.length, fa.ld,
                            a.q_rows ? 64 : a.rows_tile))) {
    return MUSA_KERNELS_EINVAL;
  }
  const int smem = a.stages * a.stage_bytes + 1024;
  static std::atomic<int> ready[kMaxDevices];
  PerDevice(ready, [] {
    return cudaFuncSetAttribute(SplitProductKernel<T, kBytes>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                210 * 1024) == cudaSuccess
               ? 1
               : 0;
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CeilDiv(n, 128)),
                     static_cast<unsigned>(CeilDiv(m, a.rows_tile)),
                     static_cast<unsigned>(a.splits));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = static_cast<unsigned>(a.splits);
  cfg.attrs = attr;
  cfg.numAttrs = a.splits > 1 ? 2 : 1;
  CountKernelLaunch();
  return static_cast<int>(
      cudaLaunchKernelEx(&cfg, SplitProductKernel<T, kBytes>, p_map, q_map, a));
}

template <typename T, bool kBytes>
int LaunchPair(int64_t m, int64_t n, int64_t k, const Factor& fa, const Factor& fb,
               const Epilogue& e, int tile_n, cudaStream_t stream) {
  using E = std::conditional_t<kBytes, uint8_t, T>;
  constexpr int kDepth = 128 / sizeof(E);
  PairArgs a = {};
  a.e = e;
  a.m = m;
  a.n = n;
  a.blocks = static_cast<int>(CeilDiv(k, kDepth));
  a.tile_n = tile_n;
  a.tiles_m = static_cast<int>(CeilDiv(m, 256));
  a.tiles_n = static_cast<int>(CeilDiv(n, tile_n));
  a.a_rows = fa.rows_contiguous;
  a.b_rows = fb.rows_contiguous;
  constexpr int kType = kBytes ? 0 : std::is_same_v<T, __nv_bfloat16> ? 1 : 0;
  a.idesc = InstructionDesc(kType, a.a_rows, a.b_rows, 256, tile_n);
  a.direct = n % 8 != 0 || !Aligned16(e.y) || !Aligned16(e.z) || !Aligned16(e.residual);
  CUtensorMap maps[5] = {};
  const Lines al = LinesOf(fa, m, k), bl = LinesOf(fb, n, k);
  bool ok = MakeMap<E>(&maps[0], fa.p, al.count, al.length, fa.ld, a.a_rows ? 64 : 128) &&
            MakeMap<E>(&maps[1], fb.p, bl.count, bl.length, fb.ld, a.b_rows ? 64 : tile_n / 2);
  if (!a.direct) {
    ok = ok && MakeMap<T>(&maps[2], e.y, m, n, n, 128, 2 * kChunk);
    if (e.z != nullptr) ok = ok && MakeMap<T>(&maps[3], e.z, m, n, n, 128, 2 * kChunk);
    if (e.residual != nullptr) ok = ok && MakeMap<T>(&maps[4], e.residual, m, n, n, 128, 2 * kChunk);
  }
  if (!ok) return MUSA_KERNELS_EINVAL;
  static std::atomic<int> ready[kMaxDevices];
  PerDevice(ready, [] {
    return cudaFuncSetAttribute(PairProductKernel<T, kBytes>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kPairSmem) == cudaSuccess
               ? 1
               : 0;
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(SmCount()));
  cfg.blockDim = dim3(kPairThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // The pairs that run at once (SMs of one processing cluster pair up).
  static std::atomic<int> resident[kMaxDevices];
  const int most = PerDevice(resident, [&cfg] {
    int clusters = 0;
    cfg.gridDim = dim3(static_cast<unsigned>(SmCount() / 2 * 2));
    if (cudaOccupancyMaxActiveClusters(&clusters, PairProductKernel<T, kBytes>, &cfg) !=
            cudaSuccess ||
        clusters < 1) {
      cudaGetLastError();
      clusters = SmCount() / 2;
    }
    return clusters;
  });
  const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < most ? tiles : most)));
  cfg.numAttrs = 2;
  CountKernelLaunch();
  return static_cast<int>(cudaLaunchKernelEx(&cfg, PairProductKernel<T, kBytes>, maps[0], maps[1],
                                             maps[2], maps[3], maps[4], a));
}

// The form of a product.
struct Plan {
  int tile_n;             // pairs with tiles of this many columns, or 0: the split form
  int rows_tile, splits;  // of the split form
};

// The form whose estimated time is least.  An estimate adds up what bounds a form, at rates
// taken from a sweep of every form over 160 sizes (1 .. 2000 rows, both factor types): the
// longest of the depth steps of the waves of CTAs one after the other, the factors' copies
// out of L2 and the reads of HBM; then the epilogues of the waves, which a split tile pays with
// the exchange of its partial sums.  Over that sweep the choice was 4% off the best form in
// the mean and 1.79 times at the worst (100 x 640, depth 1408: 12.3 us against 6.8; then
// 64 x 16384, depth 256: 8.2 against 6.2).  It holds sizes whose lines are whole 16 bytes; the
// other sizes go by the same rule, which does not know what their outputs cost the split form
// (16 sizes with all outputs, half of them odd: 6% and 1.27).  Fixed tiles of 256 rows were 35% off (1000 x 640, depth 1408: 19.2 us against 8.9;
// 256 x 1000, depth 520: 15.7 against 6.6; one row x 4096, depth 4096: 12.1 against 11.0).
constexpr double kMbPerUs = 1e-6;

// Near-equal bounds of one stretch add a little to the longest.
double Longest(double a, double b, double c, double d) {
  const auto Fourth = [](double v) { return v * v * v * v; };
  return sqrt(sqrt(Fourth(a) + Fourth(b) + Fourth(c) + Fourth(d)));
}

double SplitMicroseconds(int64_t m, int64_t n, int blocks, double hbm_bytes, int rows_tile,
                         int splits) {
  const int per_sm = SplitCtasPerSm(rows_tile);
  const int64_t ctas = CeilDiv(n, 128) * CeilDiv(m, rows_tile) * splits;
  // Clusters of eight fit the SMs' groups 14 times.
  const int64_t waves = CeilDiv(ctas, (splits == 8 ? 112 : SmCount()) * per_sm);
  const int64_t steps = CeilDiv(blocks, splits);
  const double copied = static_cast<double>(ctas) * steps * (kSideBytes + rows_tile * kDepthBytes);
  const double rows = rows_tile * (per_sm == 2 && ctas > SmCount() ? 2.0 : 1.0);
  double epilogue = 0.0704 * rows / splits;
  if (splits > 1) epilogue += 0.0142 * rows + 1.82 + 0.327 * splits;
  return 1.94 + Longest(waves * steps * 0.194, waves * steps * rows * 0.0014,
                        copied * kMbPerUs / 18.2, hbm_bytes * kMbPerUs / 6.47) +
         waves * epilogue;
}

double PairMicroseconds(int64_t m, int64_t n, int blocks, double hbm_bytes, int tile_n) {
  const int64_t tiles = CeilDiv(m, 256) * CeilDiv(n, tile_n);
  const int64_t rounds = CeilDiv(tiles, SmCount() / 2);
  const double copied = static_cast<double>(tiles) * blocks * (256 + tile_n) * kDepthBytes;
  // Outputs that TMA cannot address go element by element (333 x 2047 with all outputs: 21 us,
  // 333 x 2048 11).
  const double moves = n % 8 != 0 ? 3.0 * tile_n / 128 : 0.0;
  return 4.87 + Longest(rounds * blocks * (tile_n == 256 ? 0.311 : 0.201), 0.0,
                        copied * kMbPerUs / 18.0, hbm_bytes * kMbPerUs / 5.83) +
         rounds * ((tile_n == 256 ? 2.17 : 1.17) + moves);
}

// The choice does not depend on how the factors are stored: it decides the order of the sums.
Plan PlanProduct(int64_t m, int64_t n, int blocks, bool a_rows) {
  const int form = GetTuning(kTuneMatMulForm);
  const int64_t most = RoundUp(m, 16);
  const auto Tile = [most](int64_t rows) { return static_cast<int>(rows < most ? rows : most); };
  Plan best = {0, Tile(256), 1};
  if (form >= 16) {
    best.rows_tile = Tile(form & ~15);
    best.splits = form & 15;
    // Every CTA of a cluster multiplies: one without a block of depth would hand on what its
    // tensor memory held before.
    while (best.splits > 1 && best.splits > blocks) best.splits /= 2;
  } else if (blocks > 0 && (form == 2 || form == 3)) {
    best.tile_n = form == 2 ? 256 : 128;
  } else if (blocks > 0) {
    const double hbm_bytes = (static_cast<double>(m) + n) * blocks * kDepthBytes + 4.0 * m * n;
    double least = 1e300;
    for (int rows = 16; rows <= 256; rows *= 2) {
      for (int splits = 1; splits <= 8 && splits <= blocks; splits *= 2) {
        const double t = SplitMicroseconds(m, n, blocks, hbm_bytes, Tile(rows), splits);
        if (t < least) {
          least = t;
          best.rows_tile = Tile(rows);
          best.splits = splits;
        }
      }
      if (rows >= most) break;
    }
    for (int tile_n = 128; tile_n <= 256 && form == 0; tile_n *= 2) {
      const double t = PairMicroseconds(m, n, blocks, hbm_bytes, tile_n);
      if (t < least) {
        least = t;
        best.tile_n = tile_n;
      }
    }
  }
  // Blocks of 64 rows where they are contiguous.
  if (a_rows) best.rows_tile = static_cast<int>(RoundUp(best.rows_tile, 64));
  return best;
}

template <typename T, bool kBytes>
int Product(int64_t m, int64_t n, int64_t k, const Factor& fa, const Factor& fb,
            const Epilogue& e, cudaStream_t stream) {
  const int blocks = static_cast<int>(CeilDiv(k * static_cast<int64_t>(kBytes ? 1 : sizeof(T)), 128));
  const Plan p = PlanProduct(m, n, blocks, fa.rows_contiguous);
  return p.tile_n != 0
             ? LaunchPair<T, kBytes>(m, n, k, fa, fb, e, p.tile_n, stream)
             : LaunchSplit<T, kBytes>(m, n, k, fa, fb, e, p.rows_tile, p.splits, stream);
}

// ---------------------------------------------------------------- gradient --

// dz = dy * act'(z), rounded to the factors' type (what the tensor cores multiply), and the
// column sums of the unrounded dz: CTA (x, y) walks a range of rows of a block of columns and
// leaves one fp32 partial row; the partial rows are added in order.
constexpr int kSumRows = 8;      // row lanes of a CTA

struct SlopeArgs {
  const void* dy;
  const void* z;
  void* dz;          // null: not wanted (dy itself serves)
  float* partial;    // [gridDim.y][n]
  int64_t m, n, pitch;
  int64_t rows_per_cta;
  int act;
};

constexpr int kSumCtas = 2;      // per SM: one wave of them, 128 registers

template <typename T, int kVec>
__global__ void __launch_bounds__(32 * kSumRows, kSumCtas) SlopeKernel(SlopeArgs a) {
  using P = Pack<T, kVec>;
  constexpr int kUnroll = 4, kPairs = (kVec + 1) / 2;
  const auto Widen = [](const P& p, float2 (&v)[kPairs]) {
    if constexpr (kVec == 1) v[0] = make_float2(ToF32(p.v[0]), 0.0f);
    else WidenPack<kVec>(p, v);
  };
  const auto Narrow = [](const float2 (&v)[kPairs], P& p) {
    if constexpr (kVec == 1) p.v[0] = FromF32<T>(v[0].x);
    else NarrowPack<kVec>(v, p);
  };
  __shared__ float sums[kSumRows][32 * kVec + 1];
  GridDepWait();
  GridDepLaunch();
  const int lane = threadIdx.x % 32, row_lane = threadIdx.x / 32;
  const int64_t col = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * kVec;
  const int64_t begin = blockIdx.y * a.rows_per_cta;
  const int64_t end = begin + a.rows_per_cta < a.m ? begin + a.rows_per_cta : a.m;
  const bool bent = a.act != MUSA_ACT_IDENTITY;
  float2 sum[kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) sum[e] = make_float2(0.0f, 0.0f);
  if (col < a.n) {
    const T* dy = static_cast<const T*>(a.dy) + col;
    const T* z = static_cast<const T*>(a.z) + col;
    T* dz = static_cast<T*>(a.dz) + col;
    for (int64_t r = begin + row_lane; r < end; r += kSumRows * kUnroll) {
      P g[kUnroll], x[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t row = r + u * kSumRows;
        if (row < end) {
          g[u] = LoadStream(reinterpret_cast<const P*>(dy + row * a.n));
          if (bent) x[u] = LoadStream(reinterpret_cast<const P*>(z + row * a.n));
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t row = r + u * kSumRows;
        if (row >= end) break;
        float2 d[kPairs];
        Widen(g[u], d);
        if (bent) {
          float2 slope[kPairs];
          Widen(x[u], slope);
          Slopes(slope, a.act);
#pragma unroll
          for (int e = 0; e < kPairs; ++e) d[e] = Mul2(d[e], slope[e]);
          Narrow(d, g[u]);
        }
#pragma unroll
        for (int e = 0; e < kPairs; ++e) sum[e] = Add2(sum[e], d[e]);
        if (a.dz != nullptr) *reinterpret_cast<P*>(dz + row * a.pitch) = g[u];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    sums[row_lane][lane * kVec + e] = e % 2 == 0 ? sum[e / 2].x : sum[e / 2].y;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * kVec; c += 32 * kSumRows) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 * kVec + c;
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < kSumRows; ++r) t += sums[r][c];
    if (at < a.n) a.partial[blockIdx.y * a.n + at] = t;
  }
}

struct SumShape {
  int64_t rows_per_cta;
  int parts;
};
// One wave of CTAs over blocks of `width` columns and parts of at least 64 rows.
SumShape SumRows(int64_t m, int64_t n, int width) {
  const int64_t blocks = n > 0 ? CeilDiv(n, width) : 1;
  int64_t parts = static_cast<int64_t>(SmCount()) * kSumCtas / blocks;
  if (parts > CeilDiv(m, 64)) parts = CeilDiv(m, 64);
  if (parts < 1) parts = 1;
  const int64_t rows = CeilDiv(CeilDiv(m, parts), kSumRows) * kSumRows;
  return {rows < 1 ? 1 : rows, static_cast<int>(rows < 1 ? 1 : CeilDiv(m, rows))};
}

struct GradPlan {
  bool packed;         // whole 16-byte packs
  bool want_dz;        // dz goes to the workspace
  int64_t dz_pitch;
  SumShape sum;
  size_t dz_bytes, partial_bytes, a_bytes, b_bytes;
  size_t Total() const { return dz_bytes + partial_bytes + a_bytes + b_bytes + 64; }
};

GradPlan PlanGrad(const void* dy, const void* z, const Factor& a, const Factor& b, int64_t m,
                  int64_t n, int64_t k, int act) {
  GradPlan p = {};
  p.packed = n % 8 == 0 && Aligned16(dy) && Aligned16(z);
  const bool direct = act == MUSA_ACT_IDENTITY && Aligned16(dy) && n % 8 == 0;
  p.want_dz = !direct;
  p.dz_pitch = RoundUp(n, 8);
  p.sum = SumRows(m, n, p.packed ? 256 : 32);
  p.dz_bytes = p.want_dz ? static_cast<size_t>(RoundUp(p.dz_pitch * m * 2, 16)) : 0;
  p.partial_bytes = static_cast<size_t>(RoundUp(n * p.sum.parts * 4, 16));
  p.a_bytes = static_cast<size_t>(RoundUp(RepitchBytes(a, m, k, 2), 16));
  p.b_bytes = static_cast<size_t>(RoundUp(RepitchBytes(b, n, k, 2), 16));
  return p;
}

bool BadSizes(int64_t m, int64_t n, int64_t k) { return m < 0 || n < 0 || k < 0; }

// grid.y holds the tiles of 256 rows; in a gradient every size is the rows of a product.
bool TooLarge(int64_t m, int64_t n, int64_t k) {
  constexpr int64_t kMost = int64_t(65535) * 256;
  return m > kMost || n > kMost || k > kMost;
}

bool BadFactor(const Factor& f, int64_t rows, int64_t depth) {
  const Lines l = LinesOf(f, rows, depth);
  return l.count > 0 && l.length > 0 && (f.p == nullptr || (l.count > 1 && f.ld < l.length));
}

bool KnownAct(int act) {
  return act == MUSA_ACT_IDENTITY || act == MUSA_ACT_RELU || act == MUSA_ACT_SIGMOID ||
         act == MUSA_ACT_SILU || act == MUSA_ACT_GELU;
}

bool BadWorkspace(const void* workspace, size_t bytes, size_t need) {
  return need > 0 && (workspace == nullptr || bytes < need || !Aligned16(workspace));
}

template <typename T>
int Forward(Factor a, Factor b, const Epilogue& e, int64_t m, int64_t n, int64_t k,
            void* workspace, size_t bytes, cudaStream_t stream) {
  if (BadWorkspace(workspace, bytes, RepitchBytes(a, m, k, 2) + RepitchBytes(b, n, k, 2))) {
    return MUSA_KERNELS_EWORKSPACE;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaError_t rc = Repitch(&a, m, k, 2, &ws, stream);
  if (rc == cudaSuccess) rc = Repitch(&b, n, k, 2, &ws, stream);
  return rc != cudaSuccess ? static_cast<int>(rc)
                           : Product<T, false>(m, n, k, a, b, e, stream);
}

template <typename T>
int Backward(const void* dy, Factor a, Factor b, const void* z, void* da, void* db, void* dbias,
             int64_t m, int64_t n, int64_t k, int act, void* workspace, size_t bytes,
             cudaStream_t stream) {
  const GradPlan p = PlanGrad(dy, act == MUSA_ACT_IDENTITY ? nullptr : z, a, b, m, n, k, act);
  if (BadWorkspace(workspace, bytes, p.Total())) return MUSA_KERNELS_EWORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* partial = reinterpret_cast<float*>(ws);
  ws += p.partial_bytes;
  void* dz = p.want_dz ? ws : nullptr;
  ws += p.dz_bytes;
  cudaError_t rc = cudaSuccess;
  if (m > 0 && n > 0) {
    if (p.want_dz || dbias != nullptr) {
      SlopeArgs s = {dy, z, dz, partial, m, n, p.dz_pitch, p.sum.rows_per_cta, act};
      const dim3 grid(static_cast<unsigned>(CeilDiv(n, p.packed ? 256 : 32)),
                      static_cast<unsigned>(p.sum.parts));
      rc = LaunchChained(true, p.packed ? SlopeKernel<T, 8> : SlopeKernel<T, 1>, grid,
                         dim3(32 * kSumRows), 0, stream, s);
      if (rc != cudaSuccess) return static_cast<int>(rc);
      if (dbias != nullptr) {
        rc = LaunchAddPartialRows<T>(true, partial, p.sum.parts, n, dbias, stream);
        if (rc != cudaSuccess) return static_cast<int>(rc);
      }
    }
  } else if (dbias != nullptr && n > 0) {
    cudaMemsetAsync(dbias, 0, sizeof(T) * n, stream);
  }
  rc = cudaGetLastError();
  if (rc == cudaSuccess && db != nullptr && m > 0) rc = Repitch(&a, m, k, 2, &ws, stream);
  if (rc == cudaSuccess && da != nullptr && n > 0) rc = Repitch(&b, n, k, 2, &ws, stream);
  if (rc != cudaSuccess) return static_cast<int>(rc);
  const void* g = p.want_dz ? dz : dy;
  const int64_t ldg = p.want_dz ? p.dz_pitch : n;
  int code = MUSA_KERNELS_OK;
  Epilogue e = {};
  if (da != nullptr && m > 0 && k > 0) {
    e.y = da;
    // op(b) read along n.
    const Factor ob = {b.p, b.ld, !b.rows_contiguous};
    code = a.rows_contiguous
               ? Product<T, false>(k, m, n, ob, Factor{g, ldg, false}, e, stream)
               : Product<T, false>(m, k, n, Factor{g, ldg, false}, ob, e, stream);
    if (code != MUSA_KERNELS_OK) return code;
  }
  if (db != nullptr && n > 0 && k > 0) {
    e.y = db;
    const Factor oa = {a.p, a.ld, !a.rows_contiguous};
    code = b.rows_contiguous
               ? Product<T, false>(k, n, m, oa, Factor{g, ldg, true}, e, stream)
               : Product<T, false>(n, k, m, Factor{g, ldg, true}, oa, e, stream);
  }
  return code;
}

}  // namespace
}  // namespace musa_b200

using namespace musa_b200;

extern "C" {

int MusaMatMulStatus(void) {
  int v = 0;
  // The copy alone would not wait for streams that do not block with the default one.
  cudaError_t rc = cudaDeviceSynchronize();
  if (rc == cudaSuccess) rc = cudaMemcpyFromSymbol(&v, g_status, sizeof(v));
  return rc != cudaSuccess ? static_cast<int>(rc) : v == 0 ? MUSA_KERNELS_OK : MUSA_KERNELS_EGAVEUP;
}

size_t MatMulWorkspaceBytes(int elem_bytes, const void* a, int64_t lda, bool transpose_a,
                            const void* b, int64_t ldb, bool transpose_b, int64_t m, int64_t n,
                            int64_t k) {
  if (BadSizes(m, n, k) || (elem_bytes != 1 && elem_bytes != 2)) return 0;
  return RepitchBytes(Factor{a, lda, transpose_a}, m, k, elem_bytes) +
         RepitchBytes(Factor{b, ldb, !transpose_b}, n, k, elem_bytes);
}

int LaunchMatMulBiasAct(int dtype, const void* a, int64_t lda, bool transpose_a, const void* b,
                        int64_t ldb, bool transpose_b, const void* bias, const void* residual,
                        void* y, void* preactivation, int64_t m, int64_t n, int64_t k, int act,
                        void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (dtype != MUSA_DT_F16 && dtype != MUSA_DT_BF16) return MUSA_KERNELS_EUNSUPPORTED;
  if (!KnownAct(act)) return MUSA_KERNELS_EUNSUPPORTED;
  if (BadSizes(m, n, k)) return MUSA_KERNELS_EINVAL;
  if (TooLarge(m, n, k)) return MUSA_KERNELS_ETOOLARGE;
  const int outputs = 1 + (preactivation != nullptr) + (residual != nullptr);
  MUSA_TRACE("LaunchMatMulBiasAct", 2 * (m * k + k * n + outputs * m * n));
  if (m == 0 || n == 0) return MUSA_KERNELS_OK;
  const Factor fa = {a, lda, transpose_a}, fb = {b, ldb, !transpose_b};
  if (y == nullptr || BadFactor(fa, m, k) || BadFactor(fb, n, k)) return MUSA_KERNELS_EINVAL;
  const Epilogue e = {bias, residual, nullptr, nullptr, y, preactivation, act};
  return dtype == MUSA_DT_F16
             ? Forward<__half>(fa, fb, e, m, n, k, workspace, workspace_bytes, stream)
             : Forward<__nv_bfloat16>(fa, fb, e, m, n, k, workspace, workspace_bytes, stream);
}

size_t MatMulGradWorkspaceBytes(const void* dy, const void* a, int64_t lda, bool transpose_a,
                                const void* b, int64_t ldb, bool transpose_b,
                                const void* preactivation, int64_t m, int64_t n, int64_t k,
                                int act) {
  if (BadSizes(m, n, k)) return 0;
  return PlanGrad(dy, act == MUSA_ACT_IDENTITY ? nullptr : preactivation,
                  Factor{a, lda, transpose_a}, Factor{b, ldb, !transpose_b}, m, n, k, act)
      .Total();
}

int LaunchMatMulBiasActGrad(int dtype, const void* dy, const void* a, int64_t lda,
                            bool transpose_a, const void* b, int64_t ldb, bool transpose_b,
                            const void* preactivation, void* da, void* db, void* dbias, int64_t m,
                            int64_t n, int64_t k, int act, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream) {
  if (dtype != MUSA_DT_F16 && dtype != MUSA_DT_BF16) return MUSA_KERNELS_EUNSUPPORTED;
  if (!KnownAct(act)) return MUSA_KERNELS_EUNSUPPORTED;
  if (BadSizes(m, n, k)) return MUSA_KERNELS_EINVAL;
  if (TooLarge(m, n, k)) return MUSA_KERNELS_ETOOLARGE;
  MUSA_TRACE("LaunchMatMulBiasActGrad",
             2 * ((act == MUSA_ACT_IDENTITY ? 1 : 2) * m * n + 2 * m * k + 2 * k * n));
  const Factor fa = {a, lda, transpose_a}, fb = {b, ldb, !transpose_b};
  if (BadFactor(fa, m, k) || BadFactor(fb, n, k)) return MUSA_KERNELS_EINVAL;
  if (m > 0 && n > 0 &&
      (dy == nullptr || (act != MUSA_ACT_IDENTITY && preactivation == nullptr))) {
    return MUSA_KERNELS_EINVAL;
  }
  return dtype == MUSA_DT_F16
             ? Backward<__half>(dy, fa, fb, preactivation, da, db, dbias, m, n, k, act, workspace,
                                workspace_bytes, stream)
             : Backward<__nv_bfloat16>(dy, fa, fb, preactivation, da, db, dbias, m, n, k, act,
                                       workspace, workspace_bytes, stream);
}

int LaunchQuantizedMatMulBiasAct(int out_dtype, const void* a, int64_t lda, const float* a_scale,
                                 const void* b, int64_t ldb, const float* b_scale,
                                 const void* bias, const void* residual, void* y, int64_t m,
                                 int64_t n, int64_t k, int act, void* workspace,
                                 size_t workspace_bytes, cudaStream_t stream) {
  if (out_dtype != MUSA_DT_F16 && out_dtype != MUSA_DT_BF16) return MUSA_KERNELS_EUNSUPPORTED;
  if (!KnownAct(act)) return MUSA_KERNELS_EUNSUPPORTED;
  if (BadSizes(m, n, k)) return MUSA_KERNELS_EINVAL;
  if (TooLarge(m, n, k)) return MUSA_KERNELS_ETOOLARGE;
  MUSA_TRACE("LaunchQuantizedMatMulBiasAct",
             m * k + k * n + 2 * (residual != nullptr ? 2 : 1) * m * n);
  if (m == 0 || n == 0) return MUSA_KERNELS_OK;
  Factor fa = {a, lda, false}, fb = {b, ldb, false};
  if (y == nullptr || a_scale == nullptr || b_scale == nullptr || BadFactor(fa, m, k) ||
      BadFactor(fb, n, k)) {
    return MUSA_KERNELS_EINVAL;
  }
  if (BadWorkspace(workspace, workspace_bytes,
                   RepitchBytes(fa, m, k, 1) + RepitchBytes(fb, n, k, 1))) {
    return MUSA_KERNELS_EWORKSPACE;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaError_t rc = Repitch(&fa, m, k, 1, &ws, stream);
  if (rc == cudaSuccess) rc = Repitch(&fb, n, k, 1, &ws, stream);
  if (rc != cudaSuccess) return static_cast<int>(rc);
  const Epilogue e = {bias, residual, a_scale, b_scale, y, nullptr, act};
  return out_dtype == MUSA_DT_F16 ? Product<__half, true>(m, n, k, fa, fb, e, stream)
                                  : Product<__nv_bfloat16, true>(m, n, k, fa, fb, e, stream);
}

}  // extern "C"
