// Root-mean-square norm over the last axis with the residual's addition in front of it and, if
// wanted, an output of 8 bits with one scale per row; its backward pass.
//
//   s = x + r,  y = s * rsqrt(mean(s^2) + eps) * w,
//   8 bits: scale = max(max|y| / most, 2^-126), q = round(y / scale), most = 448 (e4m3) or 127.
//
//   u = s * rstd, du = dy * w:  ds = rstd (du - u mean(du u)) + ds_out,  dw = sum over rows of dy u.
//
// The backward pass of 16-bit rows adds x and r again: the stored sum has been rounded to 16 bits,
// which would put 2^-9 of each term into the float32 dw.
//
// Bound by memory: every row is read once, kept in registers between the statistics and the output,
// and written once.
// Measured on a B200: 16384 x 4096 bf16 with a residual into e4m3 81 us (5.8 TB/s; with loads ahead in registers
// and two reductions 106 us); 16384 x 4095 210 us (element by element 274 us); one row of 4096 3.5 us; forward and backward of 4099 x 2560 bf16 43 us.
#pragma once

#include <algorithm>

#include "seq_common.cuh"

namespace xe {
namespace norm {

using namespace seq;

struct Params {
  const void* x;
  const void* residual;  // or null
  const void* weight;    // or null
  void* y;
  void* sum;     // or null
  float* scale;  // 8-bit outputs only
  int64_t x_row, r_row;  // row strides in elements; outputs are contiguous
  int64_t rows;
  int columns;
  float eps;
  int quantize;    // 0 none, XE_E4M3, XE_I8
  int weight_f32;  // weight is float32, else of x's type
};

// The widest block of a kernel that holds `groups` groups of eight elements per thread.
template <int kGroups>
constexpr int kMaxThreads = kGroups == 1 ? 1024 : kGroups == 8 ? 1024 : 512;
template <int kGroups>
constexpr int kMaxBackwardThreads = kGroups == 8 ? 1024 : 512;

// Sums over the threads of each row of the block (`wpr` warps per row, at most 32 warps in all), and maxima
// of values held as the bits of their sizes, among which a NaN is the largest: both with one barrier.
// `turn` alternates the buffer: a thread that writes a buffer again has passed the barrier of the
// reduction in between, which all readers of the buffer reach after reading.
struct RowBuffers {
  float sum[2][32];
  uint32_t most[2][32];  // or second sums
};

__device__ __forceinline__ float warp_sum(float v, int from = 16) {
  for (int o = from; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ int first_step(int wpr) { return wpr > 16 ? 16 : wpr > 8 ? 8 : wpr > 4 ? 4 : wpr > 2 ? 2 : 1; }

template <bool kMost>
__device__ __forceinline__ void row_reduce(float& v, uint32_t& most, int wpr, RowBuffers& smem, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (kMost) most = __reduce_max_sync(0xffffffffu, most);
  if (wpr == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    smem.sum[turn][warp] = v;
    if (kMost) smem.most[turn][warp] = most;
  }
  __syncthreads();
  const int at = warp / wpr * wpr + lane;
  v = lane < wpr ? smem.sum[turn][at] : 0.0f;
  if (kMost) most = __reduce_max_sync(0xffffffffu, lane < wpr ? smem.most[turn][at] : 0u);
  turn ^= 1;
  v = warp_sum(v, first_step(wpr));
}

// Two sums with one barrier.
__device__ __forceinline__ void row_sums(float& v, float& u, int wpr, RowBuffers& smem, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v += __shfl_xor_sync(0xffffffffu, v, o);
    u += __shfl_xor_sync(0xffffffffu, u, o);
  }
  if (wpr == 1) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    smem.sum[turn][warp] = v;
    smem.most[turn][warp] = __float_as_uint(u);
  }
  __syncthreads();
  const int at = warp / wpr * wpr + lane;
  v = lane < wpr ? smem.sum[turn][at] : 0.0f;
  u = lane < wpr ? __uint_as_float(smem.most[turn][at]) : 0.0f;
  turn ^= 1;
  v = warp_sum(v, first_step(wpr));
  u = warp_sum(u, first_step(wpr));
}

// Where a thread's element groups lie.  kVec: groups of 8 consecutive elements; otherwise the
// thread takes single elements a row's threads apart, so that a warp's accesses are contiguous.
template <bool kVec>
__device__ __forceinline__ int element(int group, int i, int lane, int lanes) {
  return kVec ? (group * lanes + lane) * 8 + i : (group * 8 + i) * lanes + lane;
}

// One group as it lies in memory.
template <typename T, bool kVec>
struct Group {
  Raw8<T> raw;

  __device__ __forceinline__ void load(const T* row, int g, int lane, int lanes, int columns) {
    if constexpr (kVec) {
      const int at = element<true>(g, 0, lane, lanes);
      raw = load8<T>(row + at, at < columns ? 8 : 0, true);
    } else {
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = element<false>(g, i, lane, lanes);
        e[i] = at < columns ? row[at] : from_f32<T>(0.0f);
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const { unpack8<T>(raw, v); }
};

// Rows on their way: kStages of them, a thread's groups of kTensors tensors in shared memory places of its
// own (so that no barrier is needed), filled by cp.async.  A place is 16 bytes per thread; consecutive
// threads' places are adjacent.  As many as fit for the widest block, at most four.
template <int kGroups>
constexpr bool kRing = kGroups <= 2;
constexpr int ring_stages(int threads, int bytes) { return std::min(4, 196608 / (threads * bytes)); }
template <typename T, typename R, int kGroups>
constexpr int kForwardBytes = kGroups * 8 * (sizeof(T) + sizeof(R));  // of a stage, per thread
template <typename T, typename R, int kGroups>
constexpr int kBackwardBytes = kGroups * 16 * (sizeof(T) + sizeof(R));
template <typename T, typename R, int kGroups>
constexpr int kForwardStages = kRing<kGroups> ? ring_stages(kMaxThreads<kGroups>, kForwardBytes<T, R, kGroups>) : 0;
template <typename T, typename R, int kGroups>
constexpr int kBackwardStages = kRing<kGroups> ? ring_stages(kMaxBackwardThreads<kGroups>, kBackwardBytes<T, R, kGroups>) : 0;

__device__ __forceinline__ uint32_t ring_place(uint32_t base, int index) {
  return base + (index * blockDim.x + threadIdx.x) * 16;
}
template <typename T>
__device__ __forceinline__ void ring_load(uint32_t base, int index, const T* row, int g, int lane, int lanes, int columns) {
  const int at = element<true>(g, 0, lane, lanes);
  if (at < columns) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
      cp_async16(ring_place(base, index + i), reinterpret_cast<const uint4*>(row + at) + i);
  }
}
template <typename T>
__device__ __forceinline__ void ring_get(uint32_t base, int index, bool in, float (&v)[8]) {
  Raw8<T> raw;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (in)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(ring_place(base, index + i)));
    raw.q[i] = q;
  }
  unpack8<T>(raw, v);
}

template <typename T, bool kVec>
__device__ __forceinline__ void load_group(const T* row, int g, int lane, int lanes, int columns, float (&v)[8]) {
  Group<T, kVec> q;
  q.load(row, g, lane, lanes, columns);
  q.get(v);
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_group(T* row, int g, int lane, int lanes, int columns, const float (&v)[8]) {
  if constexpr (kVec) {
    const int at = element<true>(g, 0, lane, lanes);
    if (at < columns) store8<T>(row + at, 8, true, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = element<false>(g, i, lane, lanes);
      if (at < columns) row[at] = from_f32<T>(v[i]);
    }
  }
}

// Weights are read by every row's threads: plain loads, which the L1 cache keeps.
template <typename T, bool kVec>
__device__ __forceinline__ void load_weight(const void* weight, int weight_f32, int columns, int g, int lane, int lanes,
                                            float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = element<kVec>(g, i, lane, lanes);
    w[i] = 1.0f;
    if (weight && at < columns)
      w[i] = weight_f32 ? static_cast<const float*>(weight)[at] : to_f32(static_cast<const T*>(weight)[at]);
  }
}

// Two codes in the low 16 bits.
__device__ __forceinline__ uint32_t codes8(float a, float b, int quantize) {
  if (quantize == XE_E4M3) return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const int i = max(-127, min(127, __float2int_rn(a))), j = max(-127, min(127, __float2int_rn(b)));
  return (uint32_t)(i & 255) | (uint32_t)(j & 255) << 8;
}

// How rows lie: every one on a vector's boundary; all tensors' rows off it by the same number of elements, the
// row's number times the columns (an odd number of columns), where groups begin on the boundaries and only a
// row's two ends go by elements; or anyhow.
enum Rows { kAnyhow, kAligned, kShifted };

template <typename T>
__device__ __forceinline__ void load_shifted(const T* row, int at, int columns, float (&v)[8]) {
  if (at >= 0 && at + 8 <= columns) {
    load8f<T>(row + at, 8, true, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = at + i >= 0 && at + i < columns ? to_f32(row[at + i]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_shifted(T* row, int at, int columns, const float (&v)[8]) {
  if (at >= 0 && at + 8 <= columns) {
    store8<T>(row + at, 8, true, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at + i >= 0 && at + i < columns) row[at + i] = from_f32<T>(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load_weight_at(const void* weight, int weight_f32, int columns, int at, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = 1.0f;
    if (weight && at + i >= 0 && at + i < columns)
      w[i] = weight_f32 ? static_cast<const float*>(weight)[at + i] : to_f32(static_cast<const T*>(weight)[at + i]);
  }
}

// `wpr` warps on each row, blockDim.x / 32 / wpr rows at a time, the blocks persistent over the rows; a
// thread holds kGroups groups of eight elements.  Rows to come are loaded ahead (aligned ones through the
// ring), since the reductions' barriers would otherwise leave the memory idle.
template <typename T, typename R, int kGroups, Rows kRows>
__global__ void __launch_bounds__(kMaxThreads<kGroups>, 1) rms_norm_kernel(const __grid_constant__ Params p, int wpr) {
  constexpr bool kVec = kRows == kAligned, kMoved = kRows == kShifted;
  constexpr bool kKeep = kGroups <= 2 && !kMoved;  // weights stay in registers
  constexpr bool kRinged = kVec && kRing<kGroups>;
  constexpr int kStages = std::max(1, kForwardStages<T, R, kGroups>);
  constexpr int kPlaces = kGroups * (sizeof(T) + sizeof(R)) / 2;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ RowBuffers smem;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t stage_bytes = kPlaces * blockDim.x * 16;
  int turn = 0;
  const int lanes = wpr * 32;
  const int lane = threadIdx.x % lanes;
  const int slots = blockDim.x / lanes;
  const int64_t stride = (int64_t)gridDim.x * slots;
  int64_t row = (int64_t)blockIdx.x * slots + threadIdx.x / lanes;
  auto issue = [&](int64_t at, int stage) {
    if (at < p.rows) {
      const T* x = static_cast<const T*>(p.x) + at * p.x_row;
      const R* r = static_cast<const R*>(p.residual) + at * p.r_row;
      const uint32_t base = ring_at + stage * stage_bytes;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        ring_load<T>(base, g * (sizeof(T) / 2), x, g, lane, lanes, p.columns);
        if (p.residual)
          ring_load<R>(base, kGroups * (sizeof(T) / 2) + g * (sizeof(R) / 2), r, g, lane, lanes, p.columns);
      }
    }
    cp_async_commit();
  };
  if (kRinged) {
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) issue(row + k * stride, k);
  }
  float w[kKeep ? kGroups : 1][8];
  if (kKeep) {
#pragma unroll
    for (int g = 0; g < (kKeep ? kGroups : 1); ++g)
      load_weight<T, kVec>(p.weight, p.weight_f32, p.columns, g, lane, lanes, w[g]);
  }
  int stage = 0;
  // all slots of a block take the same number of turns: the reductions are block-wide barriers
  for (int64_t base = (int64_t)blockIdx.x * slots; base < p.rows; base += stride, row += stride) {
    const int columns = row < p.rows ? p.columns : 0;
    const int64_t out = (columns ? row : 0) * p.columns;
    const int shift = kMoved ? (int)(out % 8) : 0;
    auto first = [&](int g) { return (g * lanes + lane) * 8 - shift; };  // kShifted: the group's first column
    float v[kGroups][8];
    float total = 0.0f;
    if (kRinged) {
      issue(row + (kStages - 1) * stride, (stage + kStages - 1) % kStages);
      cp_async_wait<kStages - 1>();
    }
    const uint32_t at = ring_at + stage * stage_bytes;
    stage = (stage + 1) % kStages;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const bool in = element<kVec>(g, 0, lane, lanes) < columns;
      if (kRinged)
        ring_get<T>(at, g * (sizeof(T) / 2), in, v[g]);
      else if (kMoved)
        load_shifted<T>(static_cast<const T*>(p.x) + (columns ? row : 0) * p.x_row, first(g), columns, v[g]);
      else
        load_group<T, kVec>(static_cast<const T*>(p.x) + (columns ? row : 0) * p.x_row, g, lane, lanes, columns, v[g]);
      if (p.residual) {
        float a[8];
        if (kRinged)
          ring_get<R>(at, kGroups * (sizeof(T) / 2) + g * (sizeof(R) / 2), in, a);
        else if (kMoved)
          load_shifted<R>(static_cast<const R*>(p.residual) + (columns ? row : 0) * p.r_row, first(g), columns, a);
        else
          load_group<R, kVec>(static_cast<const R*>(p.residual) + (columns ? row : 0) * p.r_row, g, lane, lanes, columns, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[g][i] += a[i];
        if (kMoved)
          store_shifted<R>(static_cast<R*>(p.sum) + out, first(g), columns, v[g]);
        else
          store_group<R, kVec>(static_cast<R*>(p.sum) + out, g, lane, lanes, columns, v[g]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) total = fmaf(v[g][i], v[g][i], total);
    }
    // max |y| = rstd max |s w|, so that one reduction serves both statistics
    uint32_t most = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (kMoved)
        load_weight_at<T>(p.weight, p.weight_f32, p.columns, first(g), w[0]);
      else if (!kKeep)
        load_weight<T, kVec>(p.weight, p.weight_f32, p.columns, g, lane, lanes, w[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[g][i] *= w[kKeep ? g : 0][i];
        most = max(most, __float_as_uint(fabsf(v[g][i])));
      }
    }
    if (p.quantize)
      row_reduce<true>(total, most, wpr, smem, turn);
    else
      row_reduce<false>(total, most, wpr, smem, turn);
    const float rstd = rsqrtf(total / (float)p.columns + p.eps);
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g][i] *= rstd;
    if (p.quantize == 0) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (kMoved)
          store_shifted<T>(static_cast<T*>(p.y) + out, first(g), columns, v[g]);
        else
          store_group<T, kVec>(static_cast<T*>(p.y) + out, g, lane, lanes, columns, v[g]);
      }
      continue;
    }
    float scale = __uint_as_float(most) * rstd / (p.quantize == XE_E4M3 ? 448.0f : 127.0f);
    if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;  // a NaN stays
    if (columns && lane == 0) p.scale[row] = scale;
    const float inverse = 1.0f / scale;
    uint8_t* q = static_cast<uint8_t*>(p.y) + out;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = codes8(v[g][2 * i] * inverse, v[g][2 * i + 1] * inverse, p.quantize);
      if constexpr (kMoved) {
        const int at = first(g);
        if (at >= 0 && at + 8 <= columns) {
          *reinterpret_cast<uint2*>(q + at) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (at + i >= 0 && at + i < columns) q[at + i] = (uint8_t)(c[i / 2] >> (8 * (i % 2)));
        }
      } else if constexpr (kVec) {
        const int at = element<true>(g, 0, lane, lanes);
        if (at < columns) *reinterpret_cast<uint2*>(q + at) = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = element<false>(g, i, lane, lanes);
          if (at < columns) q[at] = (uint8_t)(c[i / 2] >> (8 * (i % 2)));
        }
      }
    }
  }
}

struct BackwardParams {
  const void* sum;     // the normed values, of type R; or, with `addend`, the part of them of type R
  const void* addend;  // of type T, or null
  const void* weight;  // or null
  const void* dy;
  const void* dsum;  // or null
  void* dx;
  float* partial;  // (blocks, columns) sums of dy * u, or null
  int64_t s_row, a_row, dy_row, dsum_row;
  int64_t rows;
  int columns;
  float eps;
  int weight_f32;
};

// Rows whose dw adds up in registers: one running sum over all of a slot's rows would lose its last bits (16M rows of 32
// columns: 2.2e-6 of dw's norm, 2048 rows to a slot).
constexpr int kFold = 64;

// Persistent blocks over the rows as above; each slot keeps the dw sums of kFold rows in registers and adds them to a row of
// its own in memory, and sum_rows adds these in a fixed order.
template <typename T, typename R, int kGroups, bool kVec>
__global__ void __launch_bounds__(kMaxBackwardThreads<kGroups>, 1)
    rms_norm_backward_kernel(const __grid_constant__ BackwardParams p, int wpr) {
  constexpr bool kKeep = kGroups <= 2;
  constexpr bool kRinged = kVec && kRing<kGroups>;
  constexpr int kStages = std::max(1, kBackwardStages<T, R, kGroups>);
  constexpr int kR = sizeof(R) / 2, kT = sizeof(T) / 2;
  constexpr int kPlaces = kGroups * (2 * kR + 2 * kT);  // sum, dsum, dy, addend
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ RowBuffers smem;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t stage_bytes = kPlaces * blockDim.x * 16;
  int turn = 0;
  const int lanes = wpr * 32;
  const int lane = threadIdx.x % lanes;
  const int slots = blockDim.x / lanes;
  const int slot = threadIdx.x / lanes;
  const int64_t stride = (int64_t)gridDim.x * slots;
  int64_t row = (int64_t)blockIdx.x * slots + slot;
  auto issue = [&](int64_t at, int stage) {
    if (at < p.rows) {
      const uint32_t base = ring_at + stage * stage_bytes;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int place = g * (2 * kR + 2 * kT);
        ring_load<R>(base, place, static_cast<const R*>(p.sum) + at * p.s_row, g, lane, lanes, p.columns);
        if (p.dsum)
          ring_load<R>(base, place + kR, static_cast<const R*>(p.dsum) + at * p.dsum_row, g, lane, lanes, p.columns);
        ring_load<T>(base, place + 2 * kR, static_cast<const T*>(p.dy) + at * p.dy_row, g, lane, lanes, p.columns);
        if (p.addend)
          ring_load<T>(base, place + 2 * kR + kT, static_cast<const T*>(p.addend) + at * p.a_row, g, lane, lanes, p.columns);
      }
    }
    cp_async_commit();
  };
  if (kRinged) {
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) issue(row + k * stride, k);
  }
  float dw[kGroups][8], w[kKeep ? kGroups : 1][8];
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[g][i] = 0.0f;
  if (kKeep) {
#pragma unroll
    for (int g = 0; g < (kKeep ? kGroups : 1); ++g)
      load_weight<T, kVec>(p.weight, p.weight_f32, p.columns, g, lane, lanes, w[g]);
  }
  // each slot's sums as a row of their own
  float* partial = p.partial + ((int64_t)blockIdx.x * slots + slot) * p.columns;
  bool folded = false;
  auto fold = [&] {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (!folded) {
        store_group<float, kVec>(partial, g, lane, lanes, p.columns, dw[g]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = element<kVec>(g, i, lane, lanes);
          if (at < p.columns) partial[at] += dw[g][i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) dw[g][i] = 0.0f;
    }
    folded = true;
  };
  int stage = 0, turns = 0;
  for (int64_t base = (int64_t)blockIdx.x * slots; base < p.rows; base += stride, row += stride) {
    if (p.partial && turns == kFold) {
      fold();
      turns = 0;
    }
    ++turns;
    const int columns = row < p.rows ? p.columns : 0;
    const int64_t at = columns ? row : 0;
    float s[kGroups][8], du[kGroups][8];
    float square = 0.0f;
    if (kRinged) {
      issue(row + (kStages - 1) * stride, (stage + kStages - 1) % kStages);
      cp_async_wait<kStages - 1>();
    }
    const uint32_t ring_stage = ring_at + stage * stage_bytes;
    stage = (stage + 1) % kStages;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const bool in = element<kVec>(g, 0, lane, lanes) < columns;
      const int place = g * (2 * kR + 2 * kT);
      if (kRinged) {
        ring_get<R>(ring_stage, place, in, s[g]);
        ring_get<T>(ring_stage, place + 2 * kR, in, du[g]);
      } else {
        load_group<R, kVec>(static_cast<const R*>(p.sum) + at * p.s_row, g, lane, lanes, columns, s[g]);
        load_group<T, kVec>(static_cast<const T*>(p.dy) + at * p.dy_row, g, lane, lanes, columns, du[g]);
      }
      if (p.addend) {
        float a[8];
        if (kRinged)
          ring_get<T>(ring_stage, place + 2 * kR + kT, in, a);
        else
          load_group<T, kVec>(static_cast<const T*>(p.addend) + at * p.a_row, g, lane, lanes, columns, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[g][i] += a[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) square = fmaf(s[g][i], s[g][i], square);
    }
    // sum du u = rstd sum dy w s, so that one reduction serves both sums
    float dot = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (!kKeep) load_weight<T, kVec>(p.weight, p.weight_f32, p.columns, g, lane, lanes, w[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(du[g][i] * w[kKeep ? g : 0][i], s[g][i], dot);
    }
    row_sums(square, dot, wpr, smem, turn);
    const float rstd = rsqrtf(square / (float)p.columns + p.eps);
    dot = dot * rstd / (float)p.columns;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (!kKeep) load_weight<T, kVec>(p.weight, p.weight_f32, p.columns, g, lane, lanes, w[0]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[g][i] *= rstd;
        dw[g][i] = fmaf(du[g][i], s[g][i], dw[g][i]);
        du[g][i] *= w[kKeep ? g : 0][i];
      }
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = 0.0f;
      if (p.dsum) {
        if (kRinged)
          ring_get<R>(ring_stage, g * (2 * kR + 2 * kT) + kR, element<kVec>(g, 0, lane, lanes) < columns, o);
        else
          load_group<R, kVec>(static_cast<const R*>(p.dsum) + at * p.dsum_row, g, lane, lanes, columns, o);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(rstd, du[g][i] - s[g][i] * dot, o[i]);
      store_group<R, kVec>(static_cast<R*>(p.dx) + at * p.columns, g, lane, lanes, columns, o);
    }
  }
  if (p.partial) fold();
}

}  // namespace norm

namespace seq {

// out[j] = sum over i of partial[i, j]: 32 columns to a block, each of 32 threads adds every 32nd row, and
// then the threads' sums are added as a tree.
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* partial, int64_t rows, int64_t columns, float* out) {
  __shared__ float s[32][33];
  const int64_t j = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float acc = 0.0f;
  if (j < columns) {
#pragma unroll 4
    for (int64_t i = threadIdx.y; i < rows; i += 32) acc += partial[i * columns + j];
  }
  s[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  // warp y sums column y
  float t = s[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  const int64_t column = (int64_t)blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && column < columns) out[column] = t;
}

}  // namespace seq
}  // namespace xe
