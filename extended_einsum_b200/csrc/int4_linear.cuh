// Products with 4-bit weights: y[m, o] = xs[m] sum_k x[m, k] s[o, g(k)] (q[o, k] - z[o, g(k)]), for the
// few rows m of tokens being generated.  Codes lie two to a byte, the even k in the low nibble; a
// group of `group` consecutive k (a multiple of 32) shares a scale and a zero point (8 without them).
//
// Bound by reading the codes.  They stay 4 bits wide up to the registers: by a published technique a nibble becomes a
// 16-bit float by two bit operations (the exponent of 128 for bf16, of 1024 for f16, with the nibble as the
// last bits of the significand), and subtracting 128 + z (1024 + z) leaves the exact integer q - z.  The
// tensor core multiplies these integers by the 16-bit activations exactly and sums in float32 (the weights as
// the 16-row operand, the tokens as the 8 columns), and each group's sum is scaled in float32.
// Activations of 8 bits convert to f16 exactly; float32 ones enter as three bf16 parts (8 + 8 + 8
// bits of significand, also exact) in columns of their own.
//
// The order of k inside a group of eight is free as long as both operands agree: a 32-bit word of
// codes gives the pairs (0, 4), (1, 5), (2, 6), (3, 7) by masking and shifting, so the activations
// are staged in that order.
//
// Warps work alone: a unit of work is a tile of sixteen rows over a run of k, and a warp takes every so many
// units, its ring of stages (128 k of sixteen rows, filled by cp.async) running on from one unit to the next, so
// that the reads never pause for a barrier.  A block only shares the staged activations: all of k, or, where that
// does not fit, one part of it.  Where blocks hold all of k, a tile's runs go to neighbouring warps, whose sums
// meet in shared memory; sums of several parts go to a workspace and a second kernel adds them in order.
//
// Measured on a B200: a bf16 token against 8192 x 4096 10.3 us, against 28672 x 8192 61 us (2.0 TB/s);
// 16 e4m3 rows against 16384 x 8192 47 us.  Unpacking takes eleven integer and 16-bit instructions for eight
// codes (nine, and one for the zero point, in f16) beside one or two tensor instructions: its pipe is the busiest (42 %).
#pragma once

#include "seq_common.cuh"

namespace xe {
namespace int4 {

using namespace seq;

constexpr int kStageK = 128;                       // k of one ring stage: 64 bytes of each row
constexpr int kRowPitch = 80;                      // bytes in the ring: 8 rows x 4 words in 32 banks
constexpr int kStageBytes = 16 * kRowPitch;
constexpr int kStages = 4;
constexpr int kWarps = 8;
constexpr int kZeroBytes = 4 * kStageK / 2;

struct Params {
  const void* x;
  const float* x_scale;  // or null
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;  // or null
  void* y;
  float* sums;  // (parts * runs, columns of all tokens, outputs), or null where blocks hold all of k
  int64_t x_row, packed_row;  // strides of a row: elements, bytes
  int rows, inputs, outputs, group;
  uint32_t group_magic;  // floor(2^32 / (group / 32)) + 1, or 0 for groups of 32
  int scale_dtype, y_dtype;
  int x_vec;    // rows of x start on 16-byte boundaries (8 bytes for 8-bit types)
  int pieces;   // columns of the product per token: 3 for float32 activations, else 1
  int tokens;   // tokens of one block
  int parts;    // parts of k that blocks hold, blockIdx.x % parts
  int part;     // their stages
  int runs;     // runs of a part; 1, 2, 4 or 8 without `sums`
  int run;      // their stages
  int pitch;    // of the staged activations, elements
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
  // d = a b + c
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
  // The four pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word, less the offset.
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t offset, uint32_t (&f)[4]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) f[h] = sub(((w >> (4 * h)) & 0x000f000fu) | kMagic, offset);
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
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             float c0, float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
  // As above; the odd nibbles stay where they are and stand for sixteen times themselves, which a multiplication by
  // 1/16 takes back exactly (64 + q, less 64 + z): two shifts fewer.
  static __device__ __forceinline__ void expand(uint32_t w, uint32_t offset, uint32_t (&f)[4]) {
    const uint32_t v = w >> 8;
    const uint32_t offset16 = sub(0x63806380u, offset);  // 960 - (1024 + z) = -64 - z
    f[0] = sub((w & 0x000f000fu) | kMagic, offset);
    f[1] = fma16((w & 0x00f000f0u) | kMagic, offset16);
    f[2] = sub((v & 0x000f000fu) | kMagic, offset);
    f[3] = fma16((v & 0x00f000f0u) | kMagic, offset16);
  }
  // v / 16 + c
  static __device__ __forceinline__ uint32_t fma16(uint32_t v, uint32_t c) {
    const uint32_t k = 0x2c002c00u;  // 1/16
    const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&v), *reinterpret_cast<const __half2*>(&k), *reinterpret_cast<__half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
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

__device__ __forceinline__ uint32_t load_scale(const void* at, int dtype) {
  return dtype == XE_F32 ? *static_cast<const uint32_t*>(at) : *static_cast<const uint16_t*>(at);
}
__device__ __forceinline__ float scale_value(uint32_t bits, int dtype) {
  const float wide = __uint_as_float(dtype == XE_F32 ? bits : bits << 16);
  return dtype == XE_F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : wide;
}

// The group of k = 32 u.  The product's high word is the exact quotient as long as u * (group / 32) < 2^32.
__device__ __forceinline__ int group_of(const Params& p, int u) {
  return p.group_magic ? (int)__umulhi((uint32_t)u, p.group_magic) : u;
}

__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void lds64(uint32_t at, float& v, uint32_t& w) {
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=f"(v), "=r"(w) : "r"(at) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
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

// X: type of the activations; kTiles: columns / 8; kRun: how many 32s of a stage are sure to share a scale (1, 2
// or 4, the largest that divides group / 32).
template <typename X, int kTiles, int kRun>
__global__ void __launch_bounds__(kWarps * 32) int4_linear_kernel(const __grid_constant__ Params p) {
  constexpr bool kHalf = __is_same(X, __half) || sizeof(X) == 1;
  using A = Arithmetic<kHalf>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int quad = lane % 4, row8 = lane / 4;
  const int m0 = blockIdx.y * p.tokens;
  const int tokens = min(p.tokens, p.rows - m0);
  const int columns = tokens * p.pieces;
  const int part = blockIdx.x % p.parts;
  const int stage0 = part * p.part;                                               // of this block's part
  const int stage1 = min(stage0 + p.part, (p.inputs + kStageK - 1) / kStageK);
  uint8_t* xs = smem + kWarps * kStages * kStageBytes;  // zero bytes for a stage of a column, then the activations
  const uint32_t xs_at = (uint32_t)__cvta_generic_to_shared(xs);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(smem) + warp * (kStages * kStageBytes);
  const uint32_t copy_to = ring_at + row8 * kRowPitch + quad * 16;
  const uint32_t read_at = ring_at + row8 * kRowPitch + quad * 4;
  const int groups = p.inputs / p.group;
  const int last_o = p.outputs - 1;

  // this warp's units: (row tile, run of the part), every `stride`th
  const int units = (p.outputs + 15) / 16 * p.runs;
  const int stride = gridDim.x / p.parts * kWarps;
  const int first = blockIdx.x / p.parts * kWarps + warp;

  // the copying side: the next stage and where its rows and scales lie.  Rows past the last output read the last one.
  int copy_unit = first, copy_stage = 0, copy_end = 0;
  const uint8_t *from_a = nullptr, *from_b = nullptr;
  const uint8_t *scale_a = nullptr, *scale_b = nullptr, *zero_a = nullptr, *zero_b = nullptr;
  const int scale_shift = p.scale_dtype == XE_F32 ? 2 : 1;
  // The last part may have fewer stages than the others, and runs of none: they are passed over here, and
  // their sums are zeros.
  auto open_copy = [&] {
    for (; copy_unit < units; copy_unit += stride) {
      const int tile = copy_unit / p.runs, run = copy_unit - tile * p.runs;
      copy_stage = stage0 + run * p.run;
      copy_end = min(copy_stage + p.run, stage1);
      if (copy_stage >= copy_end) continue;
      const int oa = min(tile * 16 + row8, last_o), ob = min(tile * 16 + row8 + 8, last_o);
      from_a = p.packed + oa * p.packed_row + (int64_t)copy_stage * (kStageK / 2) + quad * 16;
      from_b = p.packed + ob * p.packed_row + (int64_t)copy_stage * (kStageK / 2) + quad * 16;
      scale_a = static_cast<const uint8_t*>(p.scales) + (((int64_t)oa * groups) << scale_shift);
      scale_b = static_cast<const uint8_t*>(p.scales) + (((int64_t)ob * groups) << scale_shift);
      zero_a = p.zeros + (int64_t)oa * groups;
      zero_b = p.zeros + (int64_t)ob * groups;
      return;
    }
  };
  // a stage's scales, loaded as bits: a conversion would wait for the load.  kRun < 4: lane `quad` holds those of
  // the stage's 32s number `quad`.
  uint32_t sa[kStages], sb[kStages], za[kStages], zb[kStages];
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    sa[i] = sb[i] = 0;
    za[i] = zb[i] = 8;
  }
  auto issue = [&](int slot) {
    if (copy_unit < units) {
      const int k32 = copy_stage * 4 + quad;
      if (k32 * 32 < p.inputs) {
        cp_async16(copy_to + slot * kStageBytes, from_a);
        cp_async16(copy_to + slot * kStageBytes + 8 * kRowPitch, from_b);
        const int g = group_of(p, kRun < 4 ? k32 : copy_stage * 4);
        sa[slot] = load_scale(scale_a + (g << scale_shift), p.scale_dtype);
        sb[slot] = load_scale(scale_b + (g << scale_shift), p.scale_dtype);
        if (p.zeros) {
          za[slot] = zero_a[g];
          zb[slot] = zero_b[g];
        }
      } else if (kRun < 4) {
        sa[slot] = sb[slot] = 0;  // not another stage's: it might not be finite
      }
      from_a += kStageK / 2;
      from_b += kStageK / 2;
      if (++copy_stage == copy_end) {
        copy_unit += stride;
        open_copy();
      }
    }
    cp_async_commit();
  };
  open_copy();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  // stage the activations of the part, eight k at a time: the warps spread over the columns, and over k where
  // there are fewer columns than warps
  if (threadIdx.x < kZeroBytes / 4) reinterpret_cast<uint32_t*>(xs)[threadIdx.x] = 0;
  {
    const int k0 = stage0 * kStageK, kn = min(stage1 * kStageK, p.inputs) - k0, ke = (stage1 - stage0) * kStageK;
    const int across = columns > 4 ? 8 : columns > 2 ? 4 : columns > 1 ? 2 : 1;
    const int along = kWarps / across;
    for (int col = warp % across; col < columns; col += across) {
      const X* from = static_cast<const X*>(p.x) + (int64_t)(m0 + col / p.pieces) * p.x_row + k0;
      const int piece = p.pieces == 1 ? 0 : col % p.pieces;
      uint8_t* to = xs + kZeroBytes + (int64_t)col * p.pitch * 2;
      for (int k = (warp / across * 32 + lane) * 8; k < ke; k += along * 256 * 4) {
        Eight<X> e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k + j * along * 256 < kn) e[j].load(from + k + j * along * 256, p.x_vec);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = k + j * along * 256;
          if (at < ke) *reinterpret_cast<uint4*>(to + at * 2) = at < kn ? e[j].staged(piece) : make_uint4(0, 0, 0, 0);
        }
      }
    }
  }
  __syncthreads();

  // this lane's activations by tile of eight columns; lanes past the last column stay on the zeros
  uint32_t x_base[kTiles], x_step[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const bool in = n * 8 + row8 < columns;
    x_base[n] = xs_at + (in ? kZeroBytes + ((n * 8 + row8) * p.pitch + quad * 8) * 2 : 0);
    x_step[n] = in ? kStageK * 2 : 0;
  }
  float acc[kTiles][4];
  int unit = first, stage = 0, end = 0, tile = 0, run = 0;
  uint32_t x_at[kTiles];
  constexpr int kCols = kTiles * 8 + 1;
  float* red = reinterpret_cast<float*>(xs + kZeroBytes + columns * p.pitch * 2);  // [warp][16 rows][columns + 1]
  auto close_unit = [&] {
    if (p.sums) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = n * 8 + quad * 2 + i % 2, o = tile * 16 + row8 + i / 2 * 8;
          if (col < columns && o <= last_o) {
            const int64_t all = (int64_t)p.rows * p.pieces;
            p.sums[((int64_t)(part * p.runs + run) * all + (int64_t)m0 * p.pieces + col) * p.outputs + o] = acc[n][i];
          }
        }
      }
      return;
    }
    // every warp of the block comes here once for each of the block's turns
    const uint32_t red_at = (uint32_t)__cvta_generic_to_shared(red + (warp * 16 + row8) * kCols + quad * 2);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(red_at + (i / 2 * 8 * kCols + n * 8 + i % 2) * 4), "f"(acc[n][i]) : "memory");
    }
    __syncthreads();
    const int rows = 16 * kWarps / p.runs;
    const int o0 = (unit - warp) / p.runs * 16;
    for (int i = threadIdx.x; i < rows * tokens; i += kWarps * 32) {
      const int r = i % rows, m = i / rows;
      if (o0 + r > last_o) continue;
      float v = 0.0f;
      for (int piece = p.pieces - 1; piece >= 0; --piece)
        for (int w = 0; w < p.runs; ++w) v += red[((r / 16 * p.runs + w) * 16 + r % 16) * kCols + m * p.pieces + piece];
      if (p.x_scale) v *= p.x_scale[m0 + m];
      store_as(p.y, p.y_dtype, (int64_t)(m0 + m) * p.outputs + o0 + r, v);
    }
    __syncthreads();
  };
  auto open_unit = [&] {
    for (; unit < units; unit += stride) {
      tile = unit / p.runs, run = unit - tile * p.runs;
      stage = stage0 + run * p.run;
      end = min(stage + p.run, stage1);
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        x_at[n] = x_base[n] + (stage - stage0) * x_step[n];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
      }
      if (stage < end) return;
      close_unit();
    }
  };
  auto work = [&](int slot) {
    float sum[kTiles][4];
    const float first_a = scale_value(sa[slot], p.scale_dtype), first_b = scale_value(sb[slot], p.scale_dtype);
    const uint32_t offset_a = A::offset((float)za[slot]), offset_b = A::offset((float)zb[slot]);
    float scale_a = first_a, scale_b = first_b;
    uint32_t off_a = offset_a, off_b = offset_b;
    auto group32 = [&](int j, bool start, bool last) {
      if (kRun < 4 && start) {
        scale_a = __shfl_sync(0xffffffffu, first_a, j, 4);
        scale_b = __shfl_sync(0xffffffffu, first_b, j, 4);
        if (p.zeros) {
          off_a = __shfl_sync(0xffffffffu, offset_a, j, 4);
          off_b = __shfl_sync(0xffffffffu, offset_b, j, 4);
        }
      }
      const uint32_t at = read_at + slot * kStageBytes + j * 16;
      uint32_t fa[4], fb[4];
      A::expand(lds32(at), off_a, fa);
      A::expand(lds32(at + 8 * kRowPitch), off_b, fb);
      const uint32_t f0[4] = {fa[0], fb[0], fa[1], fb[1]}, f1[4] = {fa[2], fb[2], fa[3], fb[3]};
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const uint4 b = lds128(x_at[n] + j * 64);
        if (start)
          A::mma(sum[n], f0, b.x, b.y, 0.0f, 0.0f, 0.0f, 0.0f);
        else
          A::mma(sum[n], f0, b.x, b.y, sum[n][0], sum[n][1], sum[n][2], sum[n][3]);
        A::mma(sum[n], f1, b.z, b.w, sum[n][0], sum[n][1], sum[n][2], sum[n][3]);
        if (last) {
          acc[n][0] = fmaf(scale_a, sum[n][0], acc[n][0]);
          acc[n][1] = fmaf(scale_a, sum[n][1], acc[n][1]);
          acc[n][2] = fmaf(scale_b, sum[n][2], acc[n][2]);
          acc[n][3] = fmaf(scale_b, sum[n][3], acc[n][3]);
        }
      }
    };
    // past the last k the activations are zeros, and the codes whatever the slot held
#pragma unroll
    for (int j = 0; j < 4; ++j) group32(j, j % kRun == 0, j % kRun == kRun - 1);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) x_at[n] += x_step[n];
  };
  open_unit();
  while (unit < units) {
#pragma unroll
    for (int slot = 0; slot < kStages; ++slot) {
      if (unit < units) {
        issue((slot + kStages - 1) % kStages);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        work(slot);
        __syncwarp();  // the slot is free for the next copies
        if (++stage == end) {
          close_unit();
          unit += stride;
          open_unit();
        }
      }
    }
  }
  cp_async_wait<0>();
  if (!p.sums) {
    // the last turn's units may end inside the block
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
    if (unit - warp < units) close_unit();
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// y from the runs' sums, in order; the parts of a float32 activation from the smallest on.
__global__ void __launch_bounds__(256) int4_sum_kernel(const __grid_constant__ Params p, int runs) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int o = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
  if (o >= p.outputs) return;
  const int64_t all = (int64_t)p.rows * p.pieces;
  float sum = 0.0f;
  for (int piece = p.pieces - 1; piece >= 0; --piece) {
    const float* at = p.sums + ((int64_t)m * p.pieces + piece) * p.outputs + o;
#pragma unroll 4
    for (int r = 0; r < runs; ++r) sum += at[r * all * p.outputs];
  }
  if (p.x_scale) sum *= p.x_scale[m];
  store_as(p.y, p.y_dtype, (int64_t)m * p.outputs + o, sum);
}

}  // namespace int4
}  // namespace xe
