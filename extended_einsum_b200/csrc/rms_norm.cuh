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
#pragma once

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
constexpr int kMaxThreads = kGroups == 1 ? 1024 : kGroups <= 4 ? 512 : 1024;

// Sums (or maxima) over the threads of each row of the block: `wpr` warps per row.
template <bool kMax>
__device__ __forceinline__ float row_reduce(float v, int wpr, float* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, v, o);
    // a NaN wins the maximum
    v = kMax ? ((other > v || other != other) ? other : v) : v + other;
  }
  if (wpr == 1) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) smem[warp] = v;
  __syncthreads();
  const int first = warp / wpr * wpr;
  float r = smem[first];
  for (int i = 1; i < wpr; ++i) {
    const float other = smem[first + i];
    r = kMax ? ((other > r || other != other) ? other : r) : r + other;
  }
  __syncthreads();
  return r;
}

// Where a thread's element groups lie.  kVec: groups of 8 consecutive elements; otherwise the
// thread takes single elements a row's threads apart, so that a warp's accesses are contiguous.
template <bool kVec>
__device__ __forceinline__ int element(int group, int i, int lane, int lanes) {
  return kVec ? (group * lanes + lane) * 8 + i : (group * 8 + i) * lanes + lane;
}

template <typename T, bool kVec>
__device__ __forceinline__ void load_group(const T* row, int g, int lane, int lanes, int columns, float (&v)[8]) {
  if constexpr (kVec) {
    const int at = element<true>(g, 0, lane, lanes);
    if (at < columns) {
      load8f<T>(row + at, 8, true, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = element<false>(g, i, lane, lanes);
      v[i] = at < columns ? to_f32(row[at]) : 0.0f;
    }
  }
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

template <typename T, bool kVec>
__device__ __forceinline__ void load_weight(const Params& p, int g, int lane, int lanes, float (&w)[8]) {
  if (!p.weight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.0f;
  } else if (p.weight_f32) {
    load_group<float, kVec>(static_cast<const float*>(p.weight), g, lane, lanes, p.columns, w);
  } else {
    load_group<T, kVec>(static_cast<const T*>(p.weight), g, lane, lanes, p.columns, w);
  }
}

__device__ __forceinline__ uint32_t code8(float v, int quantize) {
  if (quantize == XE_E4M3) return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  return (uint32_t)(uint8_t)(int8_t)max(-127, min(127, __float2int_rn(v)));
}

// A block handles blockDim.x / 32 / wpr rows, `wpr` warps on each; a thread holds kGroups groups of
// eight elements.
template <typename T, typename R, int kGroups, bool kVec>
__global__ void __launch_bounds__(kMaxThreads<kGroups>) rms_norm_kernel(Params p, int wpr) {
  __shared__ float smem[32];
  const int lanes = wpr * 32;
  const int lane = threadIdx.x % lanes;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes;
  const bool live = row < p.rows;
  const int columns = live ? p.columns : 0;
  const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.x_row;
  float v[kGroups][8];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) load_group<T, kVec>(x, g, lane, lanes, columns, v[g]);
  if (p.residual) {
    const R* r = static_cast<const R*>(p.residual) + (live ? row : 0) * p.r_row;
    R* sum = static_cast<R*>(p.sum) + (live ? row : 0) * p.columns;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float a[8];
      load_group<R, kVec>(r, g, lane, lanes, columns, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[g][i] += a[i];
      store_group<R, kVec>(sum, g, lane, lanes, columns, v[g]);
    }
  }
  float total = 0.0f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) total = fmaf(v[g][i], v[g][i], total);
  total = row_reduce<false>(total, wpr, smem);
  const float rstd = rsqrtf(total / (float)p.columns + p.eps);
  float most = 0.0f;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    float w[8];
    load_weight<T, kVec>(p, g, lane, lanes, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = element<kVec>(g, i, lane, lanes) < columns;
      v[g][i] = v[g][i] * rstd * w[i];
      const float m = fabsf(v[g][i]);
      if (in && (m > most || m != m)) most = m;
    }
  }
  if (p.quantize == 0) {
    T* y = static_cast<T*>(p.y) + (live ? row : 0) * p.columns;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) store_group<T, kVec>(y, g, lane, lanes, columns, v[g]);
    return;
  }
  most = row_reduce<true>(most, wpr, smem);
  const float limit = p.quantize == XE_E4M3 ? 448.0f : 127.0f;
  float scale = most / limit;
  if (scale < 1.17549435e-38f) scale = 1.17549435e-38f;  // a NaN stays
  if (live && lane == 0) p.scale[row] = scale;
  const float inverse = 1.0f / scale;
  uint8_t* q = static_cast<uint8_t*>(p.y) + (live ? row : 0) * p.columns;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = code8(v[g][i] * inverse, p.quantize);
    if constexpr (kVec) {
      const int at = element<true>(g, 0, lane, lanes);
      if (at < columns)
        *reinterpret_cast<uint2*>(q + at) = make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24,
                                                       c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = element<false>(g, i, lane, lanes);
        if (at < columns) q[at] = (uint8_t)c[i];
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

// Persistent blocks over rows; each block (wpr warps on a row at a time) keeps its dw sums in
// registers and writes them once, and rms_norm_dweight adds the blocks in a fixed order.
template <typename T, typename R, int kGroups, bool kVec>
__global__ void __launch_bounds__(kMaxThreads<kGroups>) rms_norm_backward_kernel(BackwardParams p, int wpr) {
  __shared__ float smem[32];
  const int lanes = wpr * 32;
  const int lane = threadIdx.x % lanes;
  const int slots = blockDim.x / lanes;
  const int slot = threadIdx.x / lanes;
  Params wp{};
  wp.weight = p.weight;
  wp.weight_f32 = p.weight_f32;
  wp.columns = p.columns;
  float dw[kGroups][8];
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[g][i] = 0.0f;
  // every slot of a block takes the same number of turns: the reductions are block-wide barriers
  const int64_t stride = (int64_t)gridDim.x * slots;
  for (int64_t base = (int64_t)blockIdx.x * slots; base < p.rows; base += stride) {
    const int64_t row = base + slot;
    const bool live = row < p.rows;
    const int columns = live ? p.columns : 0;
    const int64_t at = live ? row : 0;
    float s[kGroups][8], du[kGroups][8];
    float square = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      load_group<R, kVec>(static_cast<const R*>(p.sum) + at * p.s_row, g, lane, lanes, columns, s[g]);
      load_group<T, kVec>(static_cast<const T*>(p.dy) + at * p.dy_row, g, lane, lanes, columns, du[g]);
      if (p.addend) {
        float a[8];
        load_group<T, kVec>(static_cast<const T*>(p.addend) + at * p.a_row, g, lane, lanes, columns, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[g][i] += a[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) square = fmaf(s[g][i], s[g][i], square);
    }
    const float rstd = rsqrtf(row_reduce<false>(square, wpr, smem) / (float)p.columns + p.eps);
    float dot = 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float w[8];
      load_weight<T, kVec>(wp, g, lane, lanes, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[g][i] *= rstd;
        dw[g][i] = fmaf(du[g][i], s[g][i], dw[g][i]);
        du[g][i] *= w[i];
        dot = fmaf(du[g][i], s[g][i], dot);
      }
    }
    dot = row_reduce<false>(dot, wpr, smem) / (float)p.columns;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float o[8];
      if (p.dsum) {
        load_group<R, kVec>(static_cast<const R*>(p.dsum) + at * p.dsum_row, g, lane, lanes, columns, o);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(rstd, du[g][i] - s[g][i] * dot, o[i]);
      store_group<R, kVec>(static_cast<R*>(p.dx) + at * p.columns, g, lane, lanes, columns, o);
    }
  }
  if (!p.partial) return;
  // each slot's sums as a row of their own
  float* out = p.partial + ((int64_t)blockIdx.x * slots + slot) * p.columns;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) store_group<float, kVec>(out, g, lane, lanes, p.columns, dw[g]);
}

}  // namespace norm

namespace seq {

// out[j] = sum over i of partial[i, j], in the order of i within each of 8 interleaved threads and
// then of the threads: 32 columns to a block of 32 x 8 threads.
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* partial, int64_t rows, int64_t columns, float* out) {
  __shared__ float s[8][33];
  const int64_t j = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float acc = 0.0f;
  if (j < columns)
    for (int64_t i = threadIdx.y; i < rows; i += 8) acc += partial[i * columns + j];
  s[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y == 0 && j < columns) {
    float t = s[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += s[k][threadIdx.x];
    out[j] = t;
  }
}

}  // namespace seq
}  // namespace xe
