// Products with 4-bit weights: y[m, o] = xs[m] sum_k x[m, k] s[o, g(k)] (q[o, k] - z[o, g(k)]), for the
// few rows m of tokens being generated.  Codes lie two to a byte, the even k in the low nibble; a
// group of `group` consecutive k (a multiple of 32) shares a scale and a zero point (8 without them).
//
// Bound by reading the codes.  They stay 4 bits wide up to the registers: a nibble becomes a 16-bit
// float by two bit operations (the exponent of 128 for bf16, of 1024 for f16, with the nibble as the
// last bits of the significand), and subtracting 128 + z (1024 + z) leaves the exact integer q - z.  The
// tensor core sums these integers against the 16-bit activations exactly into float32 (the weights as
// the 16-row operand, the tokens as the 8 columns), and each group's sum is scaled in float32.
// Activations of 8 bits convert to bf16 exactly; float32 ones enter as three bf16 parts (8 + 8 + 8
// bits of significand, also exact) in columns of their own.
//
// The order of k inside a group of eight is free as long as both operands agree: a 32-bit word of
// codes gives the pairs (0, 4), (1, 5), (2, 6), (3, 7) by masking and shifting, so the activations
// are staged in that order.
#pragma once

#include "seq_common.cuh"

namespace xe {
namespace int4 {

using namespace seq;

constexpr int kStageK = 128;                       // k of one ring stage: 64 bytes of each row
constexpr int kRowPitch = 80;                      // bytes in the ring: 8 rows x 4 words in 32 banks
constexpr int kStageBytes = 16 * kRowPitch;
constexpr int kWarps = 8;

struct Params {
  const void* x;
  const float* x_scale;  // or null
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;  // or null
  void* y;
  int64_t x_row, packed_row;  // strides of a row: elements, bytes
  int rows, inputs, outputs, group;
  int scale_dtype, y_dtype;
  int pieces;   // columns of the product per token: 3 for float32 activations, else 1
  int tokens;   // tokens of one block
  int chunk;    // k staged at a time
  int pitch;    // of the staged activations, elements
  int warps_k;  // warps along k; the others along rows
};

template <bool kHalf>
struct Arithmetic;
template <>
struct Arithmetic<false> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128, 128
  static __device__ __forceinline__ uint32_t offset(float z) {
    const __nv_bfloat162 v = __float2bfloat162_rn(128.0f + z);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Arithmetic<true> {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024, 1024
  static __device__ __forceinline__ uint32_t offset(float z) {
    const __half2 v = __float2half2_rn(1024.0f + z);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Eight activations as 16-bit floats in the order 0 4 1 5 2 6 3 7; piece p of float32 ones.
template <typename X>
__device__ __forceinline__ uint4 staged8(const X* at, bool vec, int piece) {
  uint32_t v[8];
  if constexpr (sizeof(X) == 1) {
    uint2 q;
    if (vec) {
      q = *reinterpret_cast<const uint2*>(at);
    } else {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t) reinterpret_cast<const uint8_t*>(at)[i] << (8 * (i % 4));
      q = make_uint2(w[0], w[1]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint8_t code = (uint8_t)((i < 4 ? q.x : q.y) >> (8 * (i % 4)));
      float f;
      if constexpr (__is_same(X, __nv_fp8_e4m3)) {
        f = __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
      } else {
        f = (float)(int8_t)code;
      }
      v[i] = __bfloat16_as_ushort(__float2bfloat16_rn(f));  // exact
    }
  } else if constexpr (sizeof(X) == 2) {
    const Raw8<X> r = load8<X>(at, 8, vec);
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (w[i / 2] >> (16 * (i % 2))) & 0xffffu;
  } else {
    float f[8];
    load8f<X>(at, 8, vec, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // the leading bits by truncation, so that no part overflows; the rests are exact
      const bool finite = fabsf(f[i]) < __uint_as_float(0x7f800000u);
      uint32_t bits = f[i] != f[i] ? 0x7fc00000u : __float_as_uint(f[i]) & 0xffff0000u;
      if (piece > 0) {
        const float rest = f[i] - __uint_as_float(bits);
        bits = __float_as_uint(rest) & 0xffff0000u;
        if (piece > 1) bits = __float_as_uint(rest - __uint_as_float(bits));
        if (!finite) bits = 0;
      }
      v[i] = bits >> 16;
    }
  }
  return make_uint4(v[0] | v[4] << 16, v[1] | v[5] << 16, v[2] | v[6] << 16, v[3] | v[7] << 16);
}

__device__ __forceinline__ float load_scale(const void* p, int dtype, int64_t at) {
  if (dtype == XE_F32) return static_cast<const float*>(p)[at];
  if (dtype == XE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  return __half2float(static_cast<const __half*>(p)[at]);
}

__device__ __forceinline__ void store_as(void* y, int dtype, int64_t at, float v) {
  if (dtype == XE_F32)
    static_cast<float*>(y)[at] = v;
  else if (dtype == XE_BF16)
    static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(y)[at] = __float2half_rn(v);
}

// X: type of the activations; kTiles: columns / 8; kSplit: groups of 32 or 64 k, so
// that the four 32s of a stage differ in scale.
template <typename X, int kTiles, bool kSplit, int kStages>
__global__ void __launch_bounds__(kWarps * 32) int4_linear_kernel(Params p) {
  constexpr bool kHalf = __is_same(X, __half);
  using A = Arithmetic<kHalf>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int quad = lane % 4, row8 = lane / 4;
  const int warp_k = warp % p.warps_k, warp_m = warp / p.warps_k;
  const int rows_per_block = 16 * (kWarps / p.warps_k);
  const int o0 = blockIdx.x * rows_per_block + warp_m * 16;
  const int m0 = blockIdx.y * p.tokens;
  const int tokens = min(p.tokens, p.rows - m0);
  const int columns = tokens * p.pieces;
  uint8_t* ring = smem + warp * (kStages * kStageBytes);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  uint16_t* xs = reinterpret_cast<uint16_t*>(smem + kWarps * kStages * kStageBytes);
  const int groups = p.inputs / p.group;

  // the two rows of this lane's fragments and of its scales, the row of its copies; past the last
  // output all read the last one, and the results are dropped
  const int last_o = p.outputs - 1;
  const int oa = min(o0 + row8, last_o), ob = min(o0 + row8 + 8, last_o);
  const uint8_t* copy_from[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    copy_from[i] = p.packed + (int64_t)min(o0 + row8 + 8 * i, last_o) * p.packed_row + quad * 16;

  float acc[kTiles][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

  for (int k0 = 0; k0 < p.inputs; k0 += p.chunk) {
    const int kn = min(p.chunk, p.inputs - k0);
    const int stages = (kn + kStageK - 1) / kStageK;
    // this warp's stages of the chunk: warp_k, warp_k + warps_k, ...
    const int own = warp_k < stages ? (stages - warp_k + p.warps_k - 1) / p.warps_k : 0;
    float sa[kStages], sb[kStages], za[kStages], zb[kStages];
    auto issue = [&](int i, int slot) {
      if (i < own) {
        const int k = (warp_k + i * p.warps_k) * kStageK;  // inside the chunk
        if (k + quad * 32 < kn) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
            cp_async16(ring_at + slot * kStageBytes + (row8 + 8 * j) * kRowPitch + quad * 16, copy_from[j] + (k0 + k) / 2);
        }
        // kSplit: lane `quad` holds the scales of the stage's 32s number `quad`
        const int kk = k0 + k + (kSplit ? quad * 32 : 0);
        if (kk < p.inputs) {
          const int64_t ga = (int64_t)oa * groups + kk / p.group, gb = (int64_t)ob * groups + kk / p.group;
          sa[slot] = load_scale(p.scales, p.scale_dtype, ga);
          sb[slot] = load_scale(p.scales, p.scale_dtype, gb);
          za[slot] = p.zeros ? (float)p.zeros[ga] : 8.0f;
          zb[slot] = p.zeros ? (float)p.zeros[gb] : 8.0f;
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      sa[i] = sb[i] = za[i] = zb[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, i);
    // stage the activations: 8 k of one column at a time
    if (k0 > 0) __syncthreads();
    for (int i = threadIdx.x; i < kTiles * 8 * (kn / 8); i += kWarps * 32) {
      const int col = i / (kn / 8), k = (i % (kn / 8)) * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (col < columns) {
        const X* at = static_cast<const X*>(p.x) + (int64_t)(m0 + col / p.pieces) * p.x_row + k0 + k;
        v = staged8<X>(at, (reinterpret_cast<uintptr_t>(at) & 15) == 0 || (sizeof(X) == 1 && (reinterpret_cast<uintptr_t>(at) & 7) == 0),
                       col % p.pieces);
      }
      *reinterpret_cast<uint4*>(xs + (int64_t)col * p.pitch + k) = v;
    }
    __syncthreads();
    for (int i0 = 0; i0 < own; i0 += kStages) {
#pragma unroll
      for (int slot = 0; slot < kStages; ++slot) {
        const int i = i0 + slot;
        if (i < own) {
          issue(i + kStages - 1, (slot + kStages - 1) % kStages);
          cp_async_wait<kStages - 1>();
          __syncwarp();
          const int k = (warp_k + i * p.warps_k) * kStageK;
          const uint8_t* stage = ring + slot * kStageBytes;
          float part[kTiles][4];
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[n][j] = 0.0f;
          uint32_t offset_a = A::offset(za[slot]), offset_b = A::offset(zb[slot]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (k + j * 32 < kn) {
              float scale_a = sa[slot], scale_b = sb[slot];
              uint32_t off_a = offset_a, off_b = offset_b;
              if (kSplit) {
                scale_a = __shfl_sync(0xffffffffu, scale_a, j, 4);
                scale_b = __shfl_sync(0xffffffffu, scale_b, j, 4);
                off_a = __shfl_sync(0xffffffffu, off_a, j, 4);
                off_b = __shfl_sync(0xffffffffu, off_b, j, 4);
              }
              const uint32_t wa = *reinterpret_cast<const uint32_t*>(stage + row8 * kRowPitch + j * 16 + quad * 4);
              const uint32_t wb = *reinterpret_cast<const uint32_t*>(stage + (row8 + 8) * kRowPitch + j * 16 + quad * 4);
              uint32_t f[2][4];
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                const uint32_t qa = ((wa >> (4 * h)) & 0x000f000fu) | A::kMagic;
                const uint32_t qb = ((wb >> (4 * h)) & 0x000f000fu) | A::kMagic;
                f[h / 2][(h % 2) * 2] = A::sub(qa, off_a);
                f[h / 2][(h % 2) * 2 + 1] = A::sub(qb, off_b);
              }
#pragma unroll
              for (int n = 0; n < kTiles; ++n) {
                const uint4 b = *reinterpret_cast<const uint4*>(xs + (int64_t)(n * 8 + row8) * p.pitch + k + j * 32 + quad * 8);
                A::mma(part[n], f[0], b.x, b.y);
                A::mma(part[n], f[1], b.z, b.w);
              }
              if (kSplit || j == 3 || k + (j + 1) * 32 >= kn) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                  acc[n][0] = fmaf(scale_a, part[n][0], acc[n][0]);
                  acc[n][1] = fmaf(scale_a, part[n][1], acc[n][1]);
                  acc[n][2] = fmaf(scale_b, part[n][2], acc[n][2]);
                  acc[n][3] = fmaf(scale_b, part[n][3], acc[n][3]);
#pragma unroll
                  for (int q = 0; q < 4; ++q) part[n][q] = 0.0f;
                }
              }
            }
          }
          __syncwarp();  // the slot is free for the next copies
        }
      }
    }
    cp_async_wait<0>();
  }

  // sums over the warps of a row tile, in order; one part per warp_k, [warp][16 rows][columns + 1]
  __syncthreads();
  constexpr int kCols = kTiles * 8 + 1;
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      red[(warp * 16 + row8 + (i / 2) * 8) * kCols + n * 8 + quad * 2 + (i % 2)] = acc[n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < rows_per_block * tokens; i += kWarps * 32) {
    const int r = i % rows_per_block, m = i / rows_per_block;
    const int o = blockIdx.x * rows_per_block + r;
    if (o >= p.outputs) continue;
    float sum = 0.0f;
    for (int piece = p.pieces - 1; piece >= 0; --piece)
      for (int w = 0; w < p.warps_k; ++w)
        sum += red[(((r / 16) * p.warps_k + w) * 16 + r % 16) * kCols + m * p.pieces + piece];
    if (p.x_scale) sum *= p.x_scale[m0 + m];
    store_as(p.y, p.y_dtype, (int64_t)(m0 + m) * p.outputs + o, sum);
  }
}

}  // namespace int4
}  // namespace xe
