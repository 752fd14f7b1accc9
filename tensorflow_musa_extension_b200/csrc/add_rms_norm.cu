// The residual's addition with the RMS norm behind it, its gradient, and the same
// forward with an 8-bit output.
//
//   s = x + residual;  inv = rsqrt(mean(s^2) + eps);  y = s * inv * gamma
//   scale = max(max|y| / 448, 2^-126);  q = e4m3(y / scale)
//   g = dy * gamma;  h = s * inv;  dx = dsum + inv * (g - h * mean(g * h))
//   dgamma = sum over rows of dy * h
//
// Bound by memory: 4 * sizeof(T) per element forward (x, residual in; y, sum out) and
// backward (dy, dsum, sum in; dx out), 3 * sizeof(T) + 1 with the 8-bit output.  A row is
// read once: a group of threads holds it in registers as fp32 sums.  Tensors off a 16-byte
// boundary and rows of more than 2048 packs in 16 bits, 4096 in fp32, are read twice, element
// by element.  The row's sum of
// squares and largest |s * gamma| come from one round of reductions, the 8-bit scale from
// both, so the 16-bit y is never written.
#include <cuda_fp8.h>

#include "common.cuh"
#include "partial_rows.cuh"
#include "row_layout.h"
#include "trace.h"
#include "../../include/musa_plugin_kernels.h"

namespace musa_b200 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleMin = 1.17549435e-38f;  // 2^-126

struct AddNormArgs {
  const void* x;
  const void* residual;  // may be null with the 8-bit output
  const void* gamma;     // may be null with the 8-bit output (rows as they are)
  void* y;               // y of type T, or q
  void* sum;
  float* stat;           // inv_rms, or scale
  int64_t rows;
  int row_size;
  int group;             // threads of a row, a power of two
  float epsilon;
  float inv_size;        // 1 / row_size
};

// Sum of `v` and (kMax) largest of `w` over the group's threads (power of two, aligned runs).
template <bool kMax>
__device__ __forceinline__ void GroupSumMax(float& v, unsigned& w, int group, float* sums,
                                            unsigned* tops) {
  if (group >= 32) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (kMax) w = __reduce_max_sync(0xffffffffu, w);
  } else {
    for (int m = group / 2; m > 0; m >>= 1) {
      v += __shfl_xor_sync(0xffffffffu, v, m);
      if (kMax) w = max(w, __shfl_xor_sync(0xffffffffu, w, m));
    }
  }
  if (group > 32) {
    const int warp = threadIdx.x >> 5, warps = group >> 5;
    const int first = warp & ~(warps - 1);
    if ((threadIdx.x & 31) == 0) {
      sums[warp] = v;
      if (kMax) tops[warp] = w;
    }
    __syncthreads();
    // Each warp folds the warps' values (every lane reading all of them was a third of the
    // instructions of a row of 8192).
    const int from = first + (threadIdx.x & (warps - 1));
    v = sums[from];
    if (kMax) w = __reduce_max_sync(0xffffffffu, tops[from]);
    for (int m = warps / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  }
}

// |v| as bits that order like the values, NaN above all.
__device__ __forceinline__ unsigned MagnitudeBits(float v) {
  return __float_as_uint(v) & 0x7fffffffu;
}

__device__ __forceinline__ float QuantizeScale(float top) {
  const float t = top / kE4m3Max;
  return t < kScaleMin ? kScaleMin : t;  // NaN goes through
}

// The largest magnitude of `w` and the pair; NaN stays.
__device__ __forceinline__ float MaxMagnitude(float w, float2 v) {
  float out;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(out) : "f"(w), "f"(v.x), "f"(v.y));
  return out;
}

template <int kVec>
__device__ __forceinline__ Pack<uint8_t, kVec> ToE4m3(const float2 (&v)[kVec / 2]) {
  Pack<uint8_t, kVec> out;
  uint16_t* w = reinterpret_cast<uint16_t*>(&out);
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) {
    w[i] = __nv_cvt_float2_to_fp8x2(v[i], __NV_SATFINITE, __NV_E4M3);
  }
  return out;
}

// Per-thread asynchronous copies of 16 bytes, or of a pack's first `bytes` with zeros behind.
// A thread reads back only slots that it filled itself.
__device__ __forceinline__ void CopyPack(uint4* slot, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<unsigned>(__cvta_generic_to_shared(slot))),
               "l"(from)
               : "memory");
}
__device__ __forceinline__ void CopyPart(uint4* slot, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<unsigned>(__cvta_generic_to_shared(slot))),
               "l"(from), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void CopyCommit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kPending>
__device__ __forceinline__ void CopyWait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// A row's packs against the tensor: whole packs, or (kShifted) rows of any length, whose
// first and last pack may hold elements of the neighbouring rows.
template <typename T, bool kShifted>
struct RowView {
  static constexpr int kVec = VecWidth<T>::value;
  int64_t first;  // element of the row's first pack
  int64_t total;  // elements of the tensor
  int shift, packs, row_size;
  __device__ RowView(int64_t row, int64_t rows, int size) : row_size(size) {
    total = rows * size;
    if constexpr (kShifted) {
      shift = RowShift<kVec>(row, size);
      packs = ShiftedPacks<kVec>(size, shift);
      first = row * size - shift;
    } else {
      shift = 0;
      packs = size / kVec;
      first = row * size;
    }
  }
  __device__ bool Edge(int p) const { return kShifted && (p == 0 || p == packs - 1); }
  __device__ bool Inside(int p, int e) const {
    return static_cast<unsigned>(p * kVec + e - shift) < static_cast<unsigned>(row_size);
  }
  // Elements of other rows become zeros.
  __device__ void Mask(int p, float2 (&v)[kVec / 2]) const {
    if (Edge(p)) {
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) {
        if (!Inside(p, 2 * e)) v[e].x = 0.0f;
        if (!Inside(p, 2 * e + 1)) v[e].y = 0.0f;
      }
    }
  }
  // Starts the copy of pack p to a slot of shared memory; what lies behind the tensor is
  // not read and comes as zeros.
  __device__ void Copy(uint4* slot, const void* base, int p) const {
    const T* at = static_cast<const T*>(base) + first + p * kVec;
    const int64_t left = total - (first + static_cast<int64_t>(p) * kVec);
    if (kShifted && left < kVec) {
      CopyPart(slot, at, static_cast<int>(left * sizeof(T)));
    } else {
      CopyPack(slot, at);
    }
  }
  template <typename U>
  __device__ void Store(void* base, int p, const Pack<U, kVec>& v) const {
    U* at = static_cast<U*>(base) + first + p * kVec;
    if (Edge(p)) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (Inside(p, e)) at[e] = v.v[e];
      }
    } else {
      StoreStream(reinterpret_cast<Pack<U, kVec>*>(at), v);
    }
  }
  // A vector of row_size values (gamma) where pack p's elements are.
  __device__ Pack<T, kVec> Vector(const void* base, int p) const {
    const T* at = static_cast<const T*>(base) + p * kVec - shift;
    if constexpr (kShifted) {
      Pack<T, kVec> v;
#pragma unroll
      for (int e = 0; e < kVec; ++e) v.v[e] = Inside(p, e) ? at[e] : FromF32<T>(0.0f);
      return v;
    } else {
      return LoadKeep(reinterpret_cast<const Pack<T, kVec>*>(at));
    }
  }
};

// A CTA of 256 to 1024 threads holds blockDim / group rows and goes round the tensor.  The
// rows come through a ring of slots in shared memory that asynchronous copies fill: once a
// thread has added its packs of a row into registers it asks for those of the row kStages
// rounds on, so the copies run through the reduction and the stores.  A thread meets the
// same columns in each of its rows (shifted rows: they are a multiple of the pack width
// apart, the launch sees to it) and keeps their gamma in registers.
__host__ __device__ constexpr int ForwardStages(int packs) { return packs == 4 ? 1 : 3; }

template <typename T, int kPacks, bool kQuantize, bool kShifted>
__global__ void __launch_bounds__(1024) AddNormKernel(AddNormArgs a) {
  constexpr int kVec = VecWidth<T>::value;
  constexpr int kStages = ForwardStages(kPacks);
  using P = Pack<T, kVec>;
  __shared__ float sums[2][32];
  __shared__ unsigned tops[2][32];
  extern __shared__ uint4 ring[];  // [stage][input][pack][thread]
  GridDepWait();
  GridDepLaunch();
  const int t = threadIdx.x & (a.group - 1);
  const int lanes = blockDim.x / a.group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * lanes;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * lanes;
  const bool add = !kQuantize || a.residual != nullptr;
  const bool normed = !kQuantize || a.gamma != nullptr;
  int64_t row = base + threadIdx.x / a.group;
  RowView<T, kShifted> view(row, a.rows, a.row_size);
  const int64_t jump = step * a.row_size;
  const auto Widen = [](const char* slot, float2 (&v)[kVec / 2]) {
    const uint4 w = *reinterpret_cast<const uint4*>(slot);
    WidenPack<kVec>(*reinterpret_cast<const P*>(&w), v);
  };
  // Slots of this thread: pack j of input i of a stage lies (i * kPacks + j) * pitch behind it.
  const int pitch = blockDim.x * 16, stage_bytes = 2 * kPacks * pitch;
  char* slots = reinterpret_cast<char*>(ring + threadIdx.x);
  // Where the next row to ask for lies; its packs are `hop` elements apart.
  const int hop = a.group * kVec;
  const T* next_x = static_cast<const T*>(a.x) + view.first + t * kVec;
  const T* next_r = add ? static_cast<const T*>(a.residual) + view.first + t * kVec : nullptr;
  int64_t next_row = row;
  // What lies behind the tensor is not read and comes as zeros (rows shorter than a pack share
  // the last one).
  const int64_t first_tail_row = FirstTailRow<kVec>(a.rows, a.row_size);
  // One group of copies, maybe empty.
  const auto Ask = [&](char* stage) {
    if (next_row < a.rows) {
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        const int p = t + j * a.group;
        if (p < view.packs) {
          uint4* x_slot = reinterpret_cast<uint4*>(stage + j * pitch);
          uint4* r_slot = reinterpret_cast<uint4*>(stage + (kPacks + j) * pitch);
          const int inside = kShifted ? ElementsInside<kVec>(next_row, a.rows, first_tail_row,
                                                             a.row_size, view.shift, p, view.packs)
                                      : kVec;
          if (inside < kVec) {
            CopyPart(x_slot, next_x + j * hop, inside * static_cast<int>(sizeof(T)));
            if (add) CopyPart(r_slot, next_r + j * hop, inside * static_cast<int>(sizeof(T)));
          } else {
            CopyPack(x_slot, next_x + j * hop);
            if (add) CopyPack(r_slot, next_r + j * hop);
          }
        }
      }
    }
    CopyCommit();
    next_row += step;
    next_x += jump;
    next_r += jump;
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) Ask(slots + i * stage_bytes);
  P gamma[kPacks];
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const int p = t + j * a.group;
    if (normed && p < view.packs) gamma[j] = view.Vector(a.gamma, p);
  }
  // Whole CTAs go round: the reductions of wide groups are barriers.
  int stage = 0, parity = 0;
  for (int64_t at = base; at < a.rows; at += step) {
    const bool there = row < a.rows;
    CopyWait<kStages - 1>();
    char* slot = slots + stage * stage_bytes;
    // s, then s * gamma: `sum` is written before the reduction.
    float2 s[kPacks][kVec / 2];
    float2 squares = make_float2(0.0f, 0.0f);
    float largest = 0.0f;
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int p = t + j * a.group;
      if (there && p < view.packs) {
        Widen(slot + j * pitch, s[j]);
        if (add) {
          float2 r[kVec / 2];
          Widen(slot + (kPacks + j) * pitch, r);
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) s[j][e] = Add2(s[j][e], r[e]);
        }
        view.Mask(p, s[j]);
#pragma unroll
        for (int e = 0; e < kVec / 2; ++e) squares = Fma2(s[j][e], s[j][e], squares);
        if (!kQuantize || a.sum != nullptr) {
          P total;
          NarrowPack<kVec>(s[j], total);
          view.Store(a.sum, p, total);
        }
        if (normed) {
          float2 g[kVec / 2];
          WidenPack<kVec>(gamma[j], g);
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) s[j][e] = Mul2(s[j][e], g[e]);
        }
        if constexpr (kQuantize) {
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) largest = MaxMagnitude(largest, s[j][e]);
        }
      }
    }
    Ask(slot);
    if (++stage == kStages) stage = 0;
    float square = squares.x + squares.y;
    unsigned top = MagnitudeBits(largest);
    GroupSumMax<kQuantize>(square, top, a.group, sums[parity], tops[parity]);
    parity ^= 1;
    float inv = rsqrtf(fmaf(square, a.inv_size, a.epsilon));
    if (!normed) inv = 1.0f;
    float scale = 1.0f, factor = inv, second = 1.0f;
    if constexpr (kQuantize) {
      scale = QuantizeScale(__uint_as_float(top) * inv);
      // y / scale as one product: off by a few fp32 roundings, where y is off by as many.
      factor = inv / scale;
      // It passes the largest float in rows of values near zero: one after the other there.
      if (!(factor < 3.4e38f)) {
        factor = inv;
        second = 1.0f / scale;
      }
    }
    if (there && t == 0) a.stat[row] = kQuantize ? scale : inv;
    const float2 factors = make_float2(factor, factor), seconds = make_float2(second, second);
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int p = t + j * a.group;
      if (there && p < view.packs) {
        if (normed) {
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) s[j][e] = Mul2(s[j][e], factors);
          if (kQuantize && second != 1.0f) {
#pragma unroll
            for (int e = 0; e < kVec / 2; ++e) s[j][e] = Mul2(s[j][e], seconds);
          }
        } else {
          // Rows as they are take the rounded division: quotients of 16-bit values fall on
          // borders between two e4m3 values, where a last bit decides.  Behind a norm the
          // fp32 values are off by more than the product with the factor.
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) {
            s[j][e] = make_float2(s[j][e].x / scale, s[j][e].y / scale);
          }
        }
        if constexpr (kQuantize) {
          view.Store(a.y, p, ToE4m3<kVec>(s[j]));
        } else {
          P out;
          NarrowPack<kVec>(s[j], out);
          view.Store(a.y, p, out);
        }
      }
    }
    view.first += jump;
    row += step;
  }
}

// Rows of any length and alignment: a CTA walks its row twice, element by element.
constexpr int kLoopThreads = 512;

template <typename T, bool kQuantize>
__global__ void __launch_bounds__(kLoopThreads) AddNormLoopKernel(AddNormArgs a) {
  __shared__ float sums[32];
  __shared__ unsigned tops[32];
  GridDepWait();
  GridDepLaunch();
  const T* gamma = static_cast<const T*>(a.gamma);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.row_size;
    const T* r = a.residual != nullptr ? static_cast<const T*>(a.residual) + row * a.row_size
                                       : nullptr;
    const auto Sum = [&](int c) { return r != nullptr ? ToF32(x[c]) + ToF32(r[c]) : ToF32(x[c]); };
    float square = 0.0f;
    unsigned top = 0;
    for (int c = threadIdx.x; c < a.row_size; c += kLoopThreads) {
      const float s = Sum(c);
      square = fmaf(s, s, square);
      if (kQuantize) top = max(top, MagnitudeBits(gamma != nullptr ? s * ToF32(gamma[c]) : s));
    }
    GroupSumMax<kQuantize>(square, top, kLoopThreads, sums, tops);
    __syncthreads();  // before the next row's sums
    float inv = rsqrtf(fmaf(square, a.inv_size, a.epsilon));
    if (kQuantize && gamma == nullptr) inv = 1.0f;
    const float scale = kQuantize ? QuantizeScale(__uint_as_float(top) * inv) : 1.0f;
    const float unscale = 1.0f / scale;
    if (threadIdx.x == 0) a.stat[row] = kQuantize ? scale : inv;
    for (int c = threadIdx.x; c < a.row_size; c += kLoopThreads) {
      const float s = Sum(c);
      const int64_t at = row * a.row_size + c;
      if (a.sum != nullptr) static_cast<T*>(a.sum)[at] = FromF32<T>(s);
      const float y = s * inv * (gamma != nullptr ? ToF32(gamma[c]) : 1.0f);
      if constexpr (kQuantize) {
        static_cast<uint8_t*>(a.y)[at] =
            __nv_cvt_float_to_fp8(gamma != nullptr ? y * unscale : y / scale, __NV_SATFINITE,
                                  __NV_E4M3);
      } else {
        static_cast<T*>(a.y)[at] = FromF32<T>(y);
      }
    }
  }
}

// ---------------------------------------------------------------- gradient --

struct AddNormGradArgs {
  const void* dy;
  const void* dsum;   // may be null
  const void* sum;
  const float* inv;
  const void* gamma;
  void* dx;
  float* partial;     // [gridDim.x][row_size]
  int64_t rows;
  int row_size;
  int group;
  float inv_size;
};

// As the forward, with the dgamma of a thread's columns in registers too; a row's slots are
// read twice, before and after its reduction, and asked for again behind its stores.  At the
// end the row lanes of the CTA are added in order and the CTA leaves one partial row.
// Registers (85, 128 or 64) and shared memory (72, 96 or 192 KB) of the three shapes that the
// launch takes: two packs for 256 threads, four for 256 and 512, fp32 rows of more for 1024.
__host__ __device__ constexpr int GradStages(int packs, int threads) {
  return packs == 2 ? 3 : threads == 1024 ? 1 : 2;
}
__host__ __device__ constexpr int GradCtas(int packs, int threads) {
  return threads > 256 ? 1 : packs == 2 ? 3 : 2;
}

template <typename T, int kPacks, int kThreads, bool kShifted>
__global__ void __launch_bounds__(kThreads, GradCtas(kPacks, kThreads)) AddNormGradKernel(
    AddNormGradArgs a) {
  constexpr int kVec = VecWidth<T>::value;
  constexpr int kStages = GradStages(kPacks, kThreads);
  using P = Pack<T, kVec>;
  __shared__ float sums[2][32];
  extern __shared__ uint4 ring[];  // [stage][input][pack][thread]
  GridDepWait();
  GridDepLaunch();
  const int t = threadIdx.x & (a.group - 1);
  const int lane_row = threadIdx.x / a.group, lanes = blockDim.x / a.group;
  const int64_t step = static_cast<int64_t>(gridDim.x) * lanes;
  const int64_t jump = step * a.row_size;
  const int64_t first_row = static_cast<int64_t>(blockIdx.x) * lanes + lane_row;
  int64_t row = first_row;
  RowView<T, kShifted> view(first_row, a.rows, a.row_size);
  const auto Slot = [&](int stage, int input, int j) {
    return ring + ((stage * 3 + input) * kPacks + j) * blockDim.x + threadIdx.x;
  };
  const auto Ask = [&](int stage, int ahead) {
    if (row + ahead * step < a.rows) {
      RowView<T, kShifted> at = view;
      at.first += ahead * jump;
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        const int p = t + j * a.group;
        if (p < view.packs) {
          at.Copy(Slot(stage, 0, j), a.sum, p);
          at.Copy(Slot(stage, 1, j), a.dy, p);
          if (a.dsum != nullptr) at.Copy(Slot(stage, 2, j), a.dsum, p);
        }
      }
    }
    CopyCommit();
  };
  const auto Values = [&](int stage, int input, int j, int p, float2 (&v)[kVec / 2]) {
    const uint4 w = *Slot(stage, input, j);
    WidenPack<kVec>(*reinterpret_cast<const P*>(&w), v);
    view.Mask(p, v);
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) Ask(i, i);
  float inv_next = row < a.rows ? a.inv[row] : 0.0f;
  float2 acc[kPacks][kVec / 2];
  P gamma[kPacks];
#pragma unroll
  for (int j = 0; j < kPacks; ++j) {
    const int p = t + j * a.group;
    if (p < view.packs) gamma[j] = view.Vector(a.gamma, p);
#pragma unroll
    for (int e = 0; e < kVec / 2; ++e) acc[j][e] = make_float2(0.0f, 0.0f);
  }
  int stage = 0, parity = 0;
  // Whole CTAs go round: the reductions of wide groups are barriers.
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * lanes; at < a.rows; at += step) {
    const bool there = row < a.rows;
    const float inv = inv_next;
    if (row + step < a.rows) inv_next = a.inv[row + step];
    CopyWait<kStages - 1>();
    float2 dots = make_float2(0.0f, 0.0f);
    const float2 invs = make_float2(inv, inv);
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int p = t + j * a.group;
      if (there && p < view.packs) {
        float2 s[kVec / 2], dy[kVec / 2], g[kVec / 2];
        Values(stage, 0, j, p, s);
        Values(stage, 1, j, p, dy);
        WidenPack<kVec>(gamma[j], g);
#pragma unroll
        for (int e = 0; e < kVec / 2; ++e) {
          const float2 dh = Mul2(dy[e], Mul2(s[e], invs));
          acc[j][e] = Add2(acc[j][e], dh);
          dots = Fma2(dh, g[e], dots);
        }
      }
    }
    float dot = dots.x + dots.y;
    unsigned none = 0;
    GroupSumMax<false>(dot, none, a.group, sums[parity], nullptr);
    parity ^= 1;
    // dx = dsum + inv * (g - h * mean), h = s * inv.
    const float back = -inv * inv * (dot * a.inv_size);
    const float2 backs = make_float2(back, back);
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int p = t + j * a.group;
      if (there && p < view.packs) {
        float2 s[kVec / 2], dy[kVec / 2], g[kVec / 2];
        Values(stage, 0, j, p, s);
        Values(stage, 1, j, p, dy);
        WidenPack<kVec>(gamma[j], g);
#pragma unroll
        for (int e = 0; e < kVec / 2; ++e) {
          s[e] = Fma2(Mul2(dy[e], g[e]), invs, Mul2(s[e], backs));
        }
        if (a.dsum != nullptr) {
          Values(stage, 2, j, p, dy);
#pragma unroll
          for (int e = 0; e < kVec / 2; ++e) s[e] = Add2(s[e], dy[e]);
        }
        P out;
        NarrowPack<kVec>(s, out);
        view.Store(a.dx, p, out);
      }
    }
    Ask(stage, kStages);
    if (++stage == kStages) stage = 0;
    view.first += jump;
    row += step;
  }
  float* partial = a.partial + static_cast<int64_t>(blockIdx.x) * a.row_size;
  if (lanes == 1) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int p = t + j * a.group;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        if (p < view.packs && view.Inside(p, e)) {
          partial[p * kVec + e - view.shift] = e % 2 == 0 ? acc[j][e / 2].x : acc[j][e / 2].y;
        }
      }
    }
    return;
  }
  // Over the ring: every copy of this CTA has landed and been read.
  float* columns = reinterpret_cast<float*>(ring);
  CopyWait<0>();
  __syncthreads();
  for (int c = threadIdx.x; c < a.row_size; c += blockDim.x) columns[c] = 0.0f;
  __syncthreads();
  for (int l = 0; l < lanes; ++l) {
    if (l == lane_row && first_row < a.rows) {
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        const int p = t + j * a.group;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          if (p < view.packs && view.Inside(p, e)) {
            columns[p * kVec + e - view.shift] += e % 2 == 0 ? acc[j][e / 2].x : acc[j][e / 2].y;
          }
        }
      }
    }
    __syncthreads();
  }
  for (int c = threadIdx.x; c < a.row_size; c += blockDim.x) partial[c] = columns[c];
}

template <typename T>
__global__ void __launch_bounds__(kLoopThreads) AddNormGradLoopKernel(AddNormGradArgs a) {
  __shared__ float sums[2][32];
  GridDepWait();
  GridDepLaunch();
  const T* gamma = static_cast<const T*>(a.gamma);
  float* partial = a.partial + static_cast<int64_t>(blockIdx.x) * a.row_size;
  for (int c = threadIdx.x; c < a.row_size; c += kLoopThreads) partial[c] = 0.0f;
  int parity = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* s = static_cast<const T*>(a.sum) + row * a.row_size;
    const T* dy = static_cast<const T*>(a.dy) + row * a.row_size;
    const float inv = a.inv[row];
    float dot = 0.0f;
    for (int c = threadIdx.x; c < a.row_size; c += kLoopThreads) {
      const float dh = ToF32(dy[c]) * (ToF32(s[c]) * inv);
      partial[c] += dh;
      dot = fmaf(dh, ToF32(gamma[c]), dot);
    }
    unsigned none = 0;
    GroupSumMax<false>(dot, none, kLoopThreads, sums[parity], nullptr);
    parity ^= 1;
    const float mean = dot * a.inv_size;
    for (int c = threadIdx.x; c < a.row_size; c += kLoopThreads) {
      const int64_t at = row * a.row_size + c;
      float d = inv * (ToF32(dy[c]) * ToF32(gamma[c]) - ToF32(s[c]) * inv * mean);
      if (a.dsum != nullptr) d += ToF32(static_cast<const T*>(a.dsum)[at]);
      static_cast<T*>(a.dx)[at] = FromF32<T>(d);
    }
  }
}

// ---------------------------------------------------------------- launches --

inline bool BadRows(int64_t rows, int64_t row_size) {
  return rows < 0 || row_size < 0 || row_size > (int64_t(1) << 24);
}

int PowerOfTwoAtLeast(int64_t v, int low) {
  int p = low;
  while (p < v) p *= 2;
  return p;
}

// CTAs that go round `rows` rows, `lanes` at a time, at most `most`: as even as the rounds
// allow, and a multiple of `multiple` where a CTA has more than one round.
int EvenCtas(int64_t rows, int lanes, int64_t most, int multiple) {
  const int64_t blocks = CeilDiv(rows, lanes);
  if (blocks <= most) return static_cast<int>(blocks);
  const int64_t rounds = CeilDiv(blocks, most);
  const int64_t even = CeilDiv(CeilDiv(blocks, rounds), multiple) * multiple;
  return static_cast<int>(even <= most ? even : most / multiple * multiple);
}

// Function attributes are per device: raised once for each kernel.
template <typename K>
void AllowShared(std::atomic<int>* ready, K kernel) {
  PerDevice(ready, [kernel] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                200 * 1024) == cudaSuccess
               ? 1
               : 0;
  });
}

template <typename T, int kPacks, bool kQuantize, bool kShifted>
cudaError_t RunForward(const AddNormArgs& a, cudaStream_t stream) {
  const int threads = a.group > 256 ? a.group : 256;
  static std::atomic<int> ready[kMaxDevices];
  AllowShared(ready, AddNormKernel<T, kPacks, kQuantize, kShifted>);
  const int ctas = EvenCtas(a.rows, threads / a.group, SmCount() * (1024 / threads),
                            kShifted ? VecWidth<T>::value : 1);
  return LaunchChained(true, AddNormKernel<T, kPacks, kQuantize, kShifted>,
                       dim3(static_cast<unsigned>(ctas)), dim3(threads),
                       ForwardStages(kPacks) * 2 * kPacks * threads * 16, stream, a);
}

template <typename T, bool kQuantize>
int LaunchForward(AddNormArgs a, bool aligned, cudaStream_t stream) {
  constexpr int kVec = VecWidth<T>::value;
  // Four packs a thread where their sums fit 64 registers: fp32.
  constexpr int kMost = sizeof(T) == 4 ? 4 : 2;
  const bool shifted = a.row_size % kVec != 0;
  const int64_t packs = CeilDiv(a.row_size, kVec) + (shifted ? 1 : 0);
  a.inv_size = 1.0f / a.row_size;
  if (!aligned || packs > kMost * 1024) {
    const int64_t ctas = a.rows < SmCount() * 4 ? a.rows : SmCount() * 4;
    return static_cast<int>(LaunchChained(true, AddNormLoopKernel<T, kQuantize>,
                                          dim3(static_cast<unsigned>(ctas)), dim3(kLoopThreads),
                                          0, stream, a));
  }
  // Two packs a thread; one where rows are few (a call is all latency), four where a row
  // needs them.
  const int per_thread = packs > 2048 ? 4 : a.rows <= SmCount() && packs <= 1024 ? 1 : 2;
  a.group = PowerOfTwoAtLeast(CeilDiv(packs, per_thread), 8);
  cudaError_t rc;
  if (per_thread == 1) {
    rc = shifted ? RunForward<T, 1, kQuantize, true>(a, stream)
                 : RunForward<T, 1, kQuantize, false>(a, stream);
  } else if (per_thread == 2) {
    rc = shifted ? RunForward<T, 2, kQuantize, true>(a, stream)
                 : RunForward<T, 2, kQuantize, false>(a, stream);
  } else {
    rc = shifted ? RunForward<T, kMost, kQuantize, true>(a, stream)
                 : RunForward<T, kMost, kQuantize, false>(a, stream);
  }
  return static_cast<int>(rc);
}

// The most CTAs of a gradient, a multiple of eight: their partial rows stay below 64 MB (or
// at eight rows).
int MostGradCtas(int64_t row_size) {
  const int64_t by_size = (int64_t(16) << 20) / row_size;
  const int64_t most = by_size < SmCount() * 4 ? by_size : SmCount() * 4;
  return most < 8 ? 8 : static_cast<int>(most / 8 * 8);
}

template <typename T, int kPacks, int kThreads, bool kShifted>
cudaError_t RunGrad(const AddNormGradArgs& a, int most, int* ctas, cudaStream_t stream) {
  constexpr int threads = kThreads;
  static std::atomic<int> ready[kMaxDevices];
  AllowShared(ready, AddNormGradKernel<T, kPacks, kThreads, kShifted>);
  const int resident = SmCount() * GradCtas(kPacks, kThreads);
  *ctas = EvenCtas(a.rows, threads / a.group, resident < most ? resident : most,
                   kShifted ? VecWidth<T>::value : 1);
  return LaunchChained(true, AddNormGradKernel<T, kPacks, kThreads, kShifted>, dim3(*ctas),
                       dim3(threads), GradStages(kPacks, kThreads) * 3 * kPacks * threads * 16,
                       stream, a);
}

template <typename T>
int LaunchGrad(AddNormGradArgs a, bool aligned, void* dgamma, cudaStream_t stream) {
  constexpr int kVec = VecWidth<T>::value;
  // 1024 threads of four packs where their sums fit 64 registers: fp32.
  constexpr int kWidest = sizeof(T) == 4 ? 1024 : 512;
  const bool shifted = a.row_size % kVec != 0;
  const int64_t packs = CeilDiv(a.row_size, kVec) + (shifted ? 1 : 0);
  const int most = MostGradCtas(a.row_size);
  int ctas;
  cudaError_t rc;
  a.inv_size = 1.0f / a.row_size;
  if (!aligned || packs > 4 * kWidest) {
    ctas = static_cast<int>(a.rows < most ? a.rows : most);
    rc = LaunchChained(true, AddNormGradLoopKernel<T>, dim3(ctas), dim3(kLoopThreads), 0, stream,
                       a);
  } else {
    const int per_thread = packs > 512 ? 4 : 2;
    a.group = PowerOfTwoAtLeast(CeilDiv(packs, per_thread), 8);
#define MUSA_RUN(PACKS, THREADS)                                           \
  (shifted ? RunGrad<T, PACKS, THREADS, true>(a, most, &ctas, stream)      \
           : RunGrad<T, PACKS, THREADS, false>(a, most, &ctas, stream))
    rc = per_thread == 2  ? MUSA_RUN(2, 256)
         : a.group <= 256 ? MUSA_RUN(4, 256)
         : a.group <= 512 ? MUSA_RUN(4, 512)
                          : MUSA_RUN(4, kWidest);
#undef MUSA_RUN
  }
  if (rc != cudaSuccess) return static_cast<int>(rc);
  return static_cast<int>(
      LaunchAddPartialRows<T>(true, a.partial, ctas, a.row_size, dgamma, stream));
}

template <typename T>
int AddNorm(const void* x, const void* residual, const void* gamma, void* y, void* sum,
            float* inv_rms, int64_t rows, int64_t row_size, float epsilon, cudaStream_t stream) {
  if (BadRows(rows, row_size)) return MUSA_KERNELS_EINVAL;
  MUSA_TRACE("LaunchAddRmsNorm", 4 * sizeof(T) * rows * row_size);
  if (rows == 0 || row_size == 0) return MUSA_KERNELS_OK;
  if (x == nullptr || residual == nullptr || gamma == nullptr || y == nullptr || sum == nullptr ||
      inv_rms == nullptr) {
    return MUSA_KERNELS_EINVAL;
  }
  const bool aligned = Aligned16(x) && Aligned16(residual) && Aligned16(gamma) && Aligned16(y) &&
                       Aligned16(sum);
  return LaunchForward<T, false>({x, residual, gamma, y, sum, inv_rms, rows,
                                  static_cast<int>(row_size), 0, epsilon, 0.0f},
                                 aligned, stream);
}

template <typename T>
int AddNormQuantize(const void* x, const void* residual, const void* gamma, void* q, float* scale,
                    void* sum, int64_t rows, int64_t row_size, float epsilon,
                    cudaStream_t stream) {
  if (BadRows(rows, row_size)) return MUSA_KERNELS_EINVAL;
  MUSA_TRACE("LaunchAddRmsNormQuantize",
             ((residual != nullptr ? 3 : 1) * sizeof(T) + 1) * rows * row_size);
  if (rows == 0 || row_size == 0) return MUSA_KERNELS_OK;
  if (x == nullptr || q == nullptr || scale == nullptr ||
      (residual == nullptr) != (sum == nullptr) || (residual != nullptr && gamma == nullptr)) {
    return MUSA_KERNELS_EINVAL;
  }
  const bool aligned = Aligned16(x) && Aligned16(residual) && Aligned16(gamma) && Aligned16(q) &&
                       Aligned16(sum);
  return LaunchForward<T, true>({x, residual, gamma, q, sum, scale, rows,
                                 static_cast<int>(row_size), 0, epsilon, 0.0f},
                                aligned, stream);
}

template <typename T>
int AddNormGrad(const void* dy, const void* dsum, const void* sum, const float* inv_rms,
                const void* gamma, void* dx, void* dgamma, int64_t rows, int64_t row_size,
                void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (BadRows(rows, row_size)) return MUSA_KERNELS_EINVAL;
  MUSA_TRACE("LaunchAddRmsNormGrad",
             (dsum != nullptr ? 4 : 3) * sizeof(T) * rows * row_size);
  if (row_size == 0) return MUSA_KERNELS_OK;
  if (dgamma == nullptr) return MUSA_KERNELS_EINVAL;
  if (rows == 0) return static_cast<int>(cudaMemsetAsync(dgamma, 0, sizeof(T) * row_size, stream));
  if (dy == nullptr || sum == nullptr || inv_rms == nullptr || gamma == nullptr ||
      dx == nullptr) {
    return MUSA_KERNELS_EINVAL;
  }
  const size_t need = static_cast<size_t>(MostGradCtas(row_size)) * row_size * sizeof(float);
  if (workspace == nullptr || workspace_bytes < need || !Aligned16(workspace)) {
    return MUSA_KERNELS_EWORKSPACE;
  }
  const bool aligned = Aligned16(dy) && Aligned16(dsum) && Aligned16(sum) && Aligned16(gamma) &&
                       Aligned16(dx);
  return LaunchGrad<T>({dy, dsum, sum, inv_rms, gamma, dx, static_cast<float*>(workspace), rows,
                        static_cast<int>(row_size), 0, 0.0f},
                       aligned, dgamma, stream);
}

}  // namespace
}  // namespace musa_b200

using namespace musa_b200;

extern "C" {

size_t AddRmsNormGradWorkspaceBytes(int64_t rows, int64_t row_size) {
  if (BadRows(rows, row_size) || rows == 0 || row_size == 0) return 0;
  return static_cast<size_t>(MostGradCtas(row_size)) * row_size * sizeof(float);
}

#define MUSA_DEFINE_ADD_RMS_NORM(SUFFIX, TYPE)                                                   \
  int LaunchAddRmsNorm_##SUFFIX(const void* x, const void* residual, const void* gamma, void* y, \
                                void* sum, float* inv_rms, int64_t rows, int64_t row_size,       \
                                float epsilon, cudaStream_t stream) {                            \
    return AddNorm<TYPE>(x, residual, gamma, y, sum, inv_rms, rows, row_size, epsilon, stream);  \
  }                                                                                              \
  int LaunchAddRmsNormGrad_##SUFFIX(const void* dy, const void* dsum, const void* sum,           \
                                    const float* inv_rms, const void* gamma, void* dx,           \
                                    void* dgamma, int64_t rows, int64_t row_size,                \
                                    void* workspace, size_t workspace_bytes,                     \
                                    cudaStream_t stream) {                                       \
    return AddNormGrad<TYPE>(dy, dsum, sum, inv_rms, gamma, dx, dgamma, rows, row_size,          \
                             workspace, workspace_bytes, stream);                                \
  }                                                                                              \
  int LaunchAddRmsNormQuantize_##SUFFIX(const void* x, const void* residual, const void* gamma,  \
                                        void* q, float* scale, void* sum, int64_t rows,          \
                                        int64_t row_size, float epsilon, cudaStream_t stream) {  \
    return AddNormQuantize<TYPE>(x, residual, gamma, q, scale, sum, rows, row_size, epsilon,     \
                                 stream);                                                        \
  }
MUSA_DEFINE_ADD_RMS_NORM(F32, float)
MUSA_DEFINE_ADD_RMS_NORM(F16, __half)
MUSA_DEFINE_ADD_RMS_NORM(BF16, __nv_bfloat16)
#undef MUSA_DEFINE_ADD_RMS_NORM

}  // extern "C"
