// Products with 4-bit weights: y[m, o] = xs[m] sum_k x[m, k] s[o, g(k)] (q[o, k] - z[o, g(k)]), for the
// few rows m of tokens being generated.  Codes lie two to a byte, the even k in the low nibble; a
// group of `group` consecutive k (a multiple of 32) shares a scale and a zero point (8 without them).
//
// Bound by reading the codes.  They stay 4 bits wide up to the registers: a nibble becomes a 16-bit
// float by two bit operations (the exponent of 128 for bf16, of 1024 for f16, with the nibble as the
// last bits of the significand), and subtracting 128 + z (1024 + z) leaves the exact integer q - z.  The
// tensor core sums these integers against the 16-bit activations exactly into float32 (the weights as
// the 16-row operand, the tokens as the 8 columns), and each group's sum is scaled in float32.
// Activations of 8 bits convert to f16 exactly; float32 ones enter as three bf16 parts (8 + 8 + 8
// bits of significand, also exact) in columns of their own.
//
// The order of k inside a group of eight is free as long as both operands agree: a 32-bit word of
// codes gives the pairs (0, 4), (1, 5), (2, 6), (3, 7) by masking and shifting, so the activations
// are staged in that order.
//
// A block holds a part of k of the activations in shared memory (the blocks of a cluster share the rows and
// split k between them, so that a part fits), its warps take row tiles of sixteen and every so many stages of
// 128 k, each with a ring of its own that cp.async fills.  Partial sums meet in shared memory, the warps' first
// and then the cluster's, in a fixed order.
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
  int x_vec;    // rows of x start on 16-byte boundaries (8 bytes for 8-bit types)
  int pieces;   // columns of the product per token: 3 for float32 activations, else 1
  int tokens;   // tokens of one block
  int part;     // k of one block of the cluster, a multiple of kStageK
  int chunk;    // k staged at a time, a multiple of kStageK
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

// Eight activations as they lie in memory, and as 16-bit floats in the order 0 4 1 5 2 6 3 7.
template <typename X>
struct Eight {
  uint32_t w[2 * sizeof(X)];

  __device__ __forceinline__ void load(const X* at, bool vec) {
    if (vec) {
      if constexpr (sizeof(X) == 1) {
        asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(at));
      } else {
#pragma unroll
        for (int i = 0; i < (int)sizeof(X) / 2; ++i)
          asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                       : "l"(reinterpret_cast<const uint4*>(at) + i));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(X); ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(X) == 1)
        w[i / 4] |= (uint32_t) reinterpret_cast<const uint8_t*>(at)[i] << (8 * (i % 4));
      else if constexpr (sizeof(X) == 2)
        w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(at)[i] << (16 * (i % 2));
      else
        w[i] = reinterpret_cast<const uint32_t*>(at)[i];
    }
  }

  __device__ __forceinline__ uint4 staged(int piece) const {
    uint32_t r[4];
    if constexpr (sizeof(X) == 1) {
      const uint32_t p[2] = {__byte_perm(w[0], w[1], 0x5140), __byte_perm(w[0], w[1], 0x7362)};  // 0 4 1 5, 2 6 3 7
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (__is_same(X, __nv_fp8_e4m3)) {
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(p[i / 2] >> (16 * (i % 2)) & 0xffffu), __NV_E4M3);
          r[i] = (uint32_t)h.x | (uint32_t)h.y << 16;
        } else {
          // 1024 + 128 + v by the bits of its significand, less 1152
          const uint32_t u = __byte_perm(p[i / 2] ^ 0x80808080u, 0x64646464u, i % 2 ? 0x4342 : 0x4140);
          r[i] = Arithmetic<true>::sub(u, 0x64806480u);
        }
      }
    } else if constexpr (sizeof(X) == 2) {
      r[0] = __byte_perm(w[0], w[2], 0x5410);
      r[1] = __byte_perm(w[0], w[2], 0x7632);
      r[2] = __byte_perm(w[1], w[3], 0x5410);
      r[3] = __byte_perm(w[1], w[3], 0x7632);
    } else {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // the leading bits by truncation, so that no part overflows; the rests are exact
        const float f = __uint_as_float(w[i]);
        const bool finite = fabsf(f) < __uint_as_float(0x7f800000u);
        uint32_t bits = f != f ? 0x7fc00000u : w[i] & 0xffff0000u;
        if (piece > 0) {
          const float rest = f - __uint_as_float(bits);
          bits = __float_as_uint(rest) & 0xffff0000u;
          if (piece > 1) bits = __float_as_uint(rest - __uint_as_float(bits));
          if (!finite) bits = 0;
        }
        v[i] = bits;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = __byte_perm(v[i], v[i + 4], 0x7632);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
};

// A scale is loaded as its bits and converted where it is used: a conversion would wait for the load.
__device__ __forceinline__ uint32_t load_scale(const void* p, int dtype, int64_t at) {
  return dtype == XE_F32 ? static_cast<const uint32_t*>(p)[at] : static_cast<const uint16_t*>(p)[at];
}
__device__ __forceinline__ float scale_value(uint32_t bits, int dtype) {
  return dtype == XE_F32   ? __uint_as_float(bits)
         : dtype == XE_BF16 ? __uint_as_float(bits << 16)
                            : __half2float(__ushort_as_half((unsigned short)bits));
}

// All threads of the cluster, with what they have written to shared memory.
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of block `rank`'s shared memory, at the place of `at` in this block's.
__device__ __forceinline__ float cluster_load(const float* at, int rank) {
  uint32_t remote;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ void store_as(void* y, int dtype, int64_t at, float v) {
  if (dtype == XE_F32)
    static_cast<float*>(y)[at] = v;
  else if (dtype == XE_BF16)
    static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(y)[at] = __float2half_rn(v);
}

// X: type of the activations; kTiles: columns / 8; kSplit: groups that are no multiple of 128, so that the
// four 32s of a stage may differ in scale.
template <typename X, int kTiles, bool kSplit, int kStages>
__global__ void __launch_bounds__(kWarps * 32) int4_linear_kernel(const __grid_constant__ Params p) {
  constexpr bool kHalf = __is_same(X, __half) || sizeof(X) == 1;
  using A = Arithmetic<kHalf>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int quad = lane % 4, row8 = lane / 4;
  const int warp_k = warp % p.warps_k, warp_m = warp / p.warps_k;
  const int rows_per_block = 16 * (kWarps / p.warps_k);
  const int o0 = blockIdx.y * rows_per_block + warp_m * 16;
  const int m0 = blockIdx.z * p.tokens;
  const int tokens = min(p.tokens, p.rows - m0);
  const int columns = tokens * p.pieces;
  uint8_t* ring = smem + warp * (kStages * kStageBytes);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  uint8_t* xs = smem + kWarps * kStages * kStageBytes;  // 16 zero bytes, then the activations
  const int groups = p.inputs / p.group;
  const int k_begin = blockIdx.x * p.part, k_end = min(k_begin + p.part, p.inputs);

  // the two rows of this lane's fragments, copies and scales; past the last output all read the last one, and
  // the results are dropped
  const int last_o = p.outputs - 1;
  const int oa = min(o0 + row8, last_o), ob = min(o0 + row8 + 8, last_o);
  const uint8_t* copy_a = p.packed + (int64_t)oa * p.packed_row + quad * 16;
  const uint8_t* copy_b = p.packed + (int64_t)ob * p.packed_row + quad * 16;
  const int64_t scales_a = (int64_t)oa * groups, scales_b = (int64_t)ob * groups;
  // this lane's column of each tile of eight; those past the last read the zero bytes at every k
  uint32_t column_at[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
    column_at[n] = n * 8 + row8 < columns ? 16 + ((n * 8 + row8) * p.pitch + quad * 8) * 2 : 0;
  if (threadIdx.x < 4) reinterpret_cast<uint32_t*>(xs)[threadIdx.x] = 0;

  float acc[kTiles][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

  for (int k0 = k_begin; k0 < k_end; k0 += p.chunk) {
    const int kn = min(p.chunk, k_end - k0);
    const int stages = (kn + kStageK - 1) / kStageK;
    // this warp's stages of the chunk: warp_k, warp_k + warps_k, ...
    const int own = warp_k < stages ? (stages - warp_k + p.warps_k - 1) / p.warps_k : 0;
    uint32_t sa[kStages], sb[kStages], za[kStages], zb[kStages];
    auto issue = [&](int i, int slot) {
      if (i < own) {
        const int k = k0 + (warp_k + i * p.warps_k) * kStageK;
        if (k + quad * 32 < k_end) {
          const uint32_t at = ring_at + slot * kStageBytes + row8 * kRowPitch + quad * 16;
          cp_async16(at, copy_a + k / 2);
          cp_async16(at + 8 * kRowPitch, copy_b + k / 2);
        }
        // kSplit: lane `quad` holds the scales of the stage's 32s number `quad`
        const int kk = k + (kSplit ? quad * 32 : 0);
        if (kk < k_end) {
          const int g = kk / p.group;
          sa[slot] = load_scale(p.scales, p.scale_dtype, scales_a + g);
          sb[slot] = load_scale(p.scales, p.scale_dtype, scales_b + g);
          if (p.zeros) {
            za[slot] = p.zeros[scales_a + g];
            zb[slot] = p.zeros[scales_b + g];
          }
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      sa[i] = sb[i] = 0;
      za[i] = zb[i] = 8;
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, i);
    // stage the activations, eight k at a time: the warps spread over the columns, and over k where there are
    // fewer columns than warps
    if (k0 > k_begin) __syncthreads();
    {
      const int across = columns > 4 ? 8 : columns > 2 ? 4 : columns > 1 ? 2 : 1;
      const int along = kWarps / across;
      for (int col = warp % across; col < columns; col += across) {
        const X* from = static_cast<const X*>(p.x) + (int64_t)(m0 + col / p.pieces) * p.x_row + k0;
        const int piece = p.pieces == 1 ? 0 : col % p.pieces;
        uint8_t* to = xs + 16 + (int64_t)col * p.pitch * 2;
        for (int k = (warp / across * 32 + lane) * 8; k < kn; k += along * 256 * 4) {
          Eight<X> e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + j * along * 256 < kn) e[j].load(from + k + j * along * 256, p.x_vec);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k + j * along * 256 < kn) *reinterpret_cast<uint4*>(to + (k + j * along * 256) * 2) = e[j].staged(piece);
        }
      }
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
          const int k = (warp_k + i * p.warps_k) * kStageK;  // inside the chunk
          const uint8_t* stage = ring + slot * kStageBytes + row8 * kRowPitch + quad * 4;
          float part[kTiles][4];
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[n][j] = 0.0f;
          const float first_a = scale_value(sa[slot], p.scale_dtype), first_b = scale_value(sb[slot], p.scale_dtype);
          const uint32_t offset_a = A::offset((float)za[slot]), offset_b = A::offset((float)zb[slot]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (k + j * 32 < kn) {
              float scale_a = first_a, scale_b = first_b;
              uint32_t off_a = offset_a, off_b = offset_b;
              if (kSplit) {
                scale_a = __shfl_sync(0xffffffffu, scale_a, j, 4);
                scale_b = __shfl_sync(0xffffffffu, scale_b, j, 4);
                off_a = __shfl_sync(0xffffffffu, off_a, j, 4);
                off_b = __shfl_sync(0xffffffffu, off_b, j, 4);
              }
              const uint32_t wa = *reinterpret_cast<const uint32_t*>(stage + j * 16);
              const uint32_t wb = *reinterpret_cast<const uint32_t*>(stage + 8 * kRowPitch + j * 16);
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
                const uint32_t at = column_at[n] ? column_at[n] + (k + j * 32) * 2 : 0;
                const uint4 b = *reinterpret_cast<const uint4*>(xs + at);
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
  }
  cp_async_wait<0>();

  // sums over the warps of a row tile and then over the blocks of the cluster, in order
  __syncthreads();
  constexpr int kCols = kTiles * 8 + 1;
  float* red = reinterpret_cast<float*>(smem);  // [warp][16 rows][columns + 1]
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      red[(warp * 16 + row8 + (i / 2) * 8) * kCols + n * 8 + quad * 2 + (i % 2)] = acc[n][i];
  const int parts = gridDim.x;
  __syncwarp();
  if (parts > 1)
    cluster_barrier();
  else
    __syncthreads();
  for (int i = threadIdx.x + blockIdx.x * (kWarps * 32); i < rows_per_block * tokens; i += parts * (kWarps * 32)) {
    const int r = i % rows_per_block, m = i / rows_per_block;
    const int o = blockIdx.y * rows_per_block + r;
    if (o >= p.outputs) continue;
    float sum = 0.0f;
    for (int piece = p.pieces - 1; piece >= 0; --piece) {
      for (int b = 0; b < parts; ++b) {
        for (int w = 0; w < p.warps_k; ++w) {
          const float* at = red + (((r / 16) * p.warps_k + w) * 16 + r % 16) * kCols + m * p.pieces + piece;
          sum += parts > 1 ? cluster_load(at, b) : *at;
        }
      }
    }
    if (p.x_scale) sum *= p.x_scale[m0 + m];
    store_as(p.y, p.y_dtype, (int64_t)(m0 + m) * p.outputs + o, sum);
  }
  if (parts > 1) {  // no block leaves while its sums are read
    __syncwarp();
    cluster_barrier();
  }
}

}  // namespace int4
}  // namespace xe
