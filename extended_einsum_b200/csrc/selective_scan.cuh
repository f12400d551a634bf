// Selective state space scan over the time axis, channel-last.  For channel d and state n
//
//   delta_t = softplus(raw_t + bias_d) (or raw_t + bias_d),   e_tn = exp(delta_t A_dn),
//   h_tn = e_tn h_{t-1,n} + delta_t x_t B_tn,   v_t = sum_n C_tn h_tn + D_d x_t,   y_t = v_t silu(z_t),
//
// with B and C shared by the channels of a group.  Bound by the special function unit: one
// exponential per token, channel and state at 16 results per clock and SM (plus three per token and
// channel for softplus and the gate); the 8 bytes of x, delta, z and y of a 16-bit type take a third of
// that time.
//
// Layout: one warp runs the recurrence of 8 kC channels; four lanes share kC channels and hold S states of each,
// 4 S >= states; states past the real ones have A = B = C = 0.  A second warp stages tiles of tokens in
// shared memory as float32 and puts out the tiles that are done, so that its chains of dependent instructions
// and its loads lie beside the recurrence's and not between its tiles: there are only one or two
// recurrences to a scheduler to hide them.  Two channels per thread because of the reads from shared
// memory: B and C for one channel alone take the whole 128 bytes per clock at the rate of the
// exponentials.  The packed instructions take two states at a time.
//
// Few channels: the length is split into segments.  A first pass runs each segment from a zero state
// and keeps its last state and sum of delta (the product of its e is exp(A sum delta)), a second
// joins them into every segment's first state, and the scan then runs all segments at once.
// Measured on a B200, 16 states, bf16: 4 x 4096 tokens of 4096 channels 529 us (the special function unit's
// floor is 274 us; 3.3 warps to a scheduler issue in about half of its slots); 2 x 2048 tokens of 2048 channels
// forward 122 us in four segments (140 us with the states stored for the backward pass), backward 262 us and 51 us for
// the segments' adjoints; one token of 64 x 4096 channels 12.5 to 13 us (36 MB, 2.8 TB/s).
#pragma once

#include "seq_common.cuh"

namespace xe {
namespace scan {

using namespace seq;

constexpr int kBackwardThreads = 64;
constexpr int kBackwardChannels = 32;

struct Params {
  const void *x, *delta, *z, *b, *c;
  void* y;
  const float *a, *d, *bias;  // (channels, states), (channels) or null, (channels) or null
  const float* state;         // (batch, channels, states) or null = zeros
  float* state_out;           // like state, or null
  float* checkpoints;         // (batch, ceil(length / kCheckpoint), channels, padded states), or null
  const void* lengths;
  int lengths64;
  int64_t x_sb, x_st, delta_sb, delta_st, z_sb, z_st, b_sb, b_st, b_sg, c_sb, c_st, c_sg;
  int batch, length, channels, states, groups;
  int softplus;
  int vec;  // bit 0: x, 1: delta, 2: z, 3: y, 4: b, 5: c, 6: dy
  int segments, segment_length;
  float* segment_state;  // (segments, batch, channels, states)
  float* segment_delta;  // (segments, batch, channels)
  // backward
  const void* dy;
  int64_t dy_sb, dy_st;
  const float* dstate_out;  // gradient of state_out, or null
  float* dstate;            // gradient of state, or null
  void *dx, *ddelta, *dz;   // contiguous (batch, length, channels); dz null without z
  float* dbc;               // (channel blocks, batch, length, 2, padded states)
  float* da;                // (segments * batch, channels, states)
  float* dd;                // (segments * batch, 2, channels): d(D), d(bias)
};

// Tokens between two stored states (training): the backward pass runs forward again from them.
constexpr int kCheckpoint = 8;

// A block's channels lie in one group: blocks [g * per_group, (g + 1) * per_group) are group g's.
struct Channels {
  int group, first, count;
};
__device__ __forceinline__ Channels block_channels(const Params& p, int per_block) {
  const int each = p.channels / p.groups;
  const int per_group = (each + per_block - 1) / per_block;
  const int group = blockIdx.x / per_group;
  const int at = (blockIdx.x % per_group) * per_block;
  return {group, group * each + at, min(per_block, each - at)};
}

// Sums v[k] over the kLanes lanes of a channel; lane l returns the sum of v[l].
template <int kLanes>
__device__ __forceinline__ float transpose_sum(float (&v)[kLanes], int lane) {
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) {
    const bool upper = lane & o;
#pragma unroll
    for (int k = 0; k < kLanes; k += 2 * o) {
      const float send = upper ? v[k] : v[k + o];
      const float keep = upper ? v[k + o] : v[k];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// kFull: the scan.  kStates: the last state of each segment from zero, no outputs.  kAdjoint: the
// same of the reversed recurrence of the backward pass, c_{t-1} = e_t (c_t + C_t dv_t).
enum Mode { kFull, kStates, kAdjoint };

template <typename T, int S, int kC, Mode kMode>
__global__ void __launch_bounds__(64) selective_scan_kernel(const __grid_constant__ Params p) {
  constexpr bool kStateOnly = kMode != kFull;
  constexpr int kLanes = 4;                     // lanes on a channel
  constexpr int kChannels = 32 / kLanes * kC;   // of the warp
  constexpr int kQuads = kChannels / 4;         // threads that stage a pair of tokens, four channels each
  constexpr int kPairs = 32 / kQuads;           // pairs of tokens in a tile
  constexpr int kTile = 2 * kPairs;
  constexpr int kRun = kTile < kCheckpoint ? kTile : kCheckpoint;
  constexpr int NP = kLanes * S;                // states, padded
  constexpr int kParts = kMode == kFull ? 2 : 1;               // B and C, or the one that is needed
  constexpr int kEach = kPairs * kParts * (NP / 4) / 32;       // their quads of states per thread
  static_assert(kPairs * kParts * (NP / 4) % 32 == 0 && kTile % kRun == 0 && kCheckpoint % kRun == 0, "whole turns");
  // two tiles: (delta, u) of each channel, u = delta x, or the adjoint's dv; B and C; v
  __shared__ __align__(16) float2 s_du[2][kTile][kChannels + 2];
  __shared__ __align__(16) float s_bc[2][kTile * kParts * NP];
  __shared__ __align__(16) float s_v[2][kStateOnly ? 1 : kTile][kChannels + 4];
  const Channels ch = block_channels(p, kChannels);
  // the first segment needs no adjoint from zero, the last one no state
  const int batch = blockIdx.y, segment = blockIdx.z + (kMode == kAdjoint ? 1 : 0);
  const int begin = segment * p.segment_length;
  const int end = min(begin + p.segment_length, p.length);
  const int live = min(end, sequence_length(p.lengths, p.lengths64, batch, p.length));
  const int tiles = (end - begin + kTile - 1) / kTile;
  const int step = kMode == kAdjoint ? -kTile : kTile;
  const int t_first = kMode == kAdjoint ? begin + (tiles - 1) * kTile : begin;
  // One warp runs the recurrence, the other one stages.  Which of the two is a matter of speed alone: a block's
  // warps go to neighbouring schedulers, and were it always the first, half of the schedulers would run all
  // the recurrences; so it changes with every second pair of warp slots.
  __shared__ int s_role;
  if (threadIdx.x == 0) {
    uint32_t slot;
    asm volatile("mov.u32 %0, %%warpid;" : "=r"(slot));
    s_role = slot >> 2 & 1;
  }
  __syncthreads();
  const bool runs = threadIdx.x / 32 == s_role;
  const int thread = threadIdx.x % 32;

  if (!runs) {
  // staging: this thread's pair of tokens and four channels; the places of the next loads move by a tile at a time
  const int row = thread / kQuads * 2;
  const int col = thread % kQuads * 4;
  const int count = max(0, min(4, ch.count - col));
  const int64_t x_st = kMode == kAdjoint ? p.dy_st : p.x_st;
  const T* x = kMode == kAdjoint ? static_cast<const T*>(p.dy) + batch * p.dy_sb : static_cast<const T*>(p.x) + batch * p.x_sb;
  x += ch.first + col + (t_first + row) * x_st;
  const T* delta = static_cast<const T*>(p.delta) + batch * p.delta_sb + ch.first + col + (t_first + row) * p.delta_st;
  const T* z = static_cast<const T*>(p.z) + batch * p.z_sb + ch.first + col + (t_first + row) * p.z_st;
  T* y = static_cast<T*>(p.y) + ((int64_t)batch * p.length + t_first + row) * p.channels + ch.first + col;
  const bool whole_x = (p.vec & (kMode == kAdjoint ? 64 : 1)) && count == 4, whole_d = (p.vec & 2) && count == 4;
  const bool whole_z = (p.vec & 4) && count == 4, whole_y = (p.vec & 8) && count == 4;
  const T* shared_at[kEach];  // B and C: pair of tokens, which of the two, four states
  int shared_t[kEach], shared_n[kEach];
  bool whole_s[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int i = k * 32 + thread;
    const int n0 = i % (NP / 4) * 4;
    const bool second = kMode == kAdjoint || (kParts == 2 && i / (NP / 4) % 2);
    shared_t[k] = i / (NP / 4 * kParts) * 2;
    shared_n[k] = max(0, min(4, p.states - n0));
    whole_s[k] = (p.vec & (second ? 32 : 16)) && (shared_n[k] == 4 || shared_n[k] == 0);
    shared_at[k] = second ? static_cast<const T*>(p.c) + batch * p.c_sb + ch.group * p.c_sg + n0 + (t_first + shared_t[k]) * p.c_st
                          : static_cast<const T*>(p.b) + batch * p.b_sb + ch.group * p.b_sg + n0 + (t_first + shared_t[k]) * p.b_st;
  }
  float bias[4], skip[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = p.bias && i < count ? p.bias[ch.first + col + i] : 0.0f;
    skip[i] = !kStateOnly && p.d && i < count ? p.d[ch.first + col + i] : 0.0f;
  }

  struct Loaded {
    Raw4<T> x, d, z;
  };
  Loaded next[2], staged[2], shown[2];  // of the tiles to come, on hand and to be put out
  Raw4<T> next_s[kEach][2];
  auto fetch = [&](int at) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const bool in = at + row + q < live;
      next[q].x = load4_if<T>(x + q * x_st, in, count, whole_x);
      next[q].d = load4_if<T>(delta + q * p.delta_st, in, count, whole_d);
      if (kMode != kStates && p.z) next[q].z = load4_if<T>(z + q * p.z_st, in, count, whole_z);
    }
    x += step * x_st;
    delta += step * p.delta_st;
    z += step * p.z_st;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const bool second = kMode == kAdjoint || (kParts == 2 && (k * 32 + thread) / (NP / 4) % 2);
      const int64_t st = second ? p.c_st : p.b_st;
#pragma unroll
      for (int q = 0; q < 2; ++q)
        next_s[k][q] = load4_if<T>(shared_at[k] + q * st, shared_n[k] > 0 && at + shared_t[k] + q < live, shared_n[k], whole_s[k]);
      shared_at[k] += step * st;
    }
  };
  auto stage = [&](int tile) {
    const int t0 = t_first + tile * step;
    const bool in[2] = {t0 + row < live, t0 + row + 1 < live};
    float2 du[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F2 xv = pack2(value4<T>(next[0].x, i), value4<T>(next[1].x, i));
      F2 d = add2(pack2(value4<T>(next[0].d, i), value4<T>(next[1].d, i)), both(bias[i]));
      if (p.softplus) d = softplus2(d);
      float2 dd = unpack2(d);
      if (!in[0]) dd.x = 0.0f;  // x, z, B and C have been read as zero
      if (!in[1]) dd.y = 0.0f;
      F2 u;
      if (kMode == kAdjoint)
        u = p.z ? gate2(xv, pack2(value4<T>(next[0].z, i), value4<T>(next[1].z, i))) : xv;
      else
        u = mul2(pack2(dd.x, dd.y), xv);
      const float2 uu = unpack2(u);
      du[0][i] = make_float2(dd.x, uu.x);
      du[1][i] = make_float2(dd.y, uu.y);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < 4; i += 2)
        *reinterpret_cast<float4*>(&s_du[tile & 1][row + q][col + i]) =
            make_float4(du[q][i].x, du[q][i].y, du[q][i + 1].x, du[q][i + 1].y);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = k * 32 + thread;  // pair of tokens, which of the two, four states
      float* at = s_bc[tile & 1] + ((i / (NP / 4 * kParts) * 2) * kParts + i / (NP / 4) % kParts) * NP + i % (NP / 4) * 4;
#pragma unroll
      for (int q = 0; q < 2; ++q)
        *reinterpret_cast<float4*>(at + q * kParts * NP) = make_float4(
            value4<T>(next_s[k][q], 0), value4<T>(next_s[k][q], 1), value4<T>(next_s[k][q], 2), value4<T>(next_s[k][q], 3));
    }
  };
  auto put_out = [&](int tile) {
    if (!kStateOnly) {
      const int t0 = t_first + tile * step;
      const bool in[2] = {t0 + row < live, t0 + row + 1 < live};
      float o[2][4];
      const float4 v0 = *reinterpret_cast<const float4*>(&s_v[tile & 1][row][col]);
      const float4 v1 = *reinterpret_cast<const float4*>(&s_v[tile & 1][row + 1][col]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        F2 v = fma2(both(skip[i]), pack2(value4<T>(shown[0].x, i), value4<T>(shown[1].x, i)), pack2((&v0.x)[i], (&v1.x)[i]));
        if (p.z) v = gate2(v, pack2(value4<T>(shown[0].z, i), value4<T>(shown[1].z, i)));
        const float2 f = unpack2(v);
        o[0][i] = f.x, o[1][i] = f.y;
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (t0 + row + q < end && count > 0) {
          if (!in[q]) o[q][0] = o[q][1] = o[q][2] = o[q][3] = 0.0f;
          store4<T>(y + q * (int64_t)p.channels, count, whole_y, o[q]);
        }
      }
      y += (int64_t)kTile * p.channels;
    }
  };
  if (tiles > 0) {
    fetch(t_first);
    stage(0);
  }
  for (int tile = 0; tile < tiles; ++tile) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      shown[q] = staged[q];
      staged[q] = next[q];
    }
    if (tile + 1 < tiles) fetch(t_first + (tile + 1) * step);
    __syncthreads();
    if (tile > 0) put_out(tile - 1);
    if (tile + 1 < tiles) stage(tile + 1);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2; ++q) shown[q] = staged[q];
  if (tiles > 0) put_out(tiles - 1);
  return;
  }

  // recurrence: this thread's kC channels and S states of each
  const int mine = thread / kLanes * kC, lane = thread % kLanes;
  F2 a[kC][S / 2], h[kC][S / 2];
  const int64_t state_at = ((int64_t)batch * p.channels + ch.first + mine) * p.states + lane * S;
#pragma unroll
  for (int j = 0; j < kC; ++j) {
    float a1[S], h1[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const bool in = mine + j < ch.count && lane * S + s < p.states;
      a1[s] = in ? decay_rate(p.a[(int64_t)(ch.first + mine + j) * p.states + lane * S + s]) : 0.0f;
      h1[s] = 0.0f;
      if (!kStateOnly && in) {
        if (p.segments > 1)
          h1[s] = p.segment_state[(int64_t)segment * p.batch * p.channels * p.states + state_at + j * p.states + s];
        else if (p.state)
          h1[s] = p.state[state_at + j * p.states + s];
      }
    }
#pragma unroll
    for (int s = 0; s < S / 2; ++s) {
      a[j][s] = pack2(a1[2 * s], a1[2 * s + 1]);
      h[j][s] = pack2(h1[2 * s], h1[2 * s + 1]);
    }
  }
  float delta_sum[kC] = {};
  const int64_t checkpoint_rows = (p.length + kCheckpoint - 1) / kCheckpoint;
  float* checkpoints = p.checkpoints + ((int64_t)batch * checkpoint_rows * p.channels + ch.first + mine) * NP + lane * S;

  for (int tile = 0; tile < tiles; ++tile) {
    __syncthreads();
    const int t0 = t_first + tile * step;
    if (t0 < live || (!kStateOnly && p.checkpoints)) {
#pragma unroll
      for (int t1 = 0; t1 < kTile; t1 += kRun) {
        if (!kStateOnly && p.checkpoints && (t0 + t1) % kCheckpoint == 0 && t0 + t1 < p.length) {
#pragma unroll
          for (int j = 0; j < kC; ++j) {
            float* at = checkpoints + ((int64_t)((t0 + t1) / kCheckpoint) * p.channels + j) * NP;
            if (mine + j < ch.count) {
#pragma unroll
              for (int s = 0; s < S / 2; s += 2)
                *reinterpret_cast<ulonglong2*>(at + 2 * s) = make_ulonglong2(h[j][s], h[j][s + 1]);
            }
          }
        }
#pragma unroll
        for (int t2 = 0; t2 < kRun; t2 += 4) {
          float v[kC][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int t = kMode == kAdjoint ? kTile - 1 - (t1 + t2 + k) : t1 + t2 + k;
            float2 du[kC];
            if constexpr (kC == 2)
              *reinterpret_cast<float4*>(du) = *reinterpret_cast<const float4*>(&s_du[tile & 1][t][mine]);
            else
              du[0] = s_du[tile & 1][t][mine];
            // B, or C in the adjoint recurrence
            const ulonglong2* bv = reinterpret_cast<const ulonglong2*>(s_bc[tile & 1] + t * kParts * NP + lane * S);
            const ulonglong2* cv = bv + NP / 4;
#pragma unroll
            for (int j = 0; j < kC; ++j) {
              const F2 d2 = both(du[j].x), u2 = both(du[j].y);
              F2 sum = 0;
              if (kStateOnly) delta_sum[j] += du[j].x;
#pragma unroll
              for (int s = 0; s < S / 2; ++s) {
                const F2 e = decay2(d2, a[j][s]), b2 = s % 2 ? bv[s / 2].y : bv[s / 2].x;
                if (kMode == kAdjoint)
                  h[j][s] = mul2(e, fma2(u2, b2, h[j][s]));
                else
                  h[j][s] = fma2(e, h[j][s], mul2(u2, b2));
                if (!kStateOnly) {
                  const F2 c2 = s % 2 ? cv[s / 2].y : cv[s / 2].x;
                  sum = s == 0 ? mul2(c2, h[j][s]) : fma2(c2, h[j][s], sum);
                }
              }
              if (!kStateOnly) {
                const float2 q = unpack2(sum);
                v[j][k] = q.x + q.y;
              }
            }
          }
          if (!kStateOnly) {
            float* at = &s_v[tile & 1][t1 + t2 + lane][mine];
            if constexpr (kC == 2)
              *reinterpret_cast<float2*>(at) = make_float2(transpose_sum<4>(v[0], lane), transpose_sum<4>(v[1], lane));
            else
              at[0] = transpose_sum<4>(v[0], lane);
          }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kC; ++j) {
    if (mine + j >= ch.count) continue;
    float* out = nullptr;
    if (kStateOnly)
      out = p.segment_state + (int64_t)segment * p.batch * p.channels * p.states + state_at + j * p.states;
    else if (p.state_out && segment == p.segments - 1)
      out = p.state_out + state_at + j * p.states;
    if (out) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const float2 q = unpack2(h[j][s / 2]);
        if (lane * S + s < p.states) out[s] = s % 2 ? q.y : q.x;
      }
    }
    if (kStateOnly && lane == 0)
      p.segment_delta[((int64_t)segment * p.batch + batch) * p.channels + ch.first + mine + j] = delta_sum[j];
  }
}

// The first states of all segments, in place over their last states from zero; or, kReverse, the
// adjoints that enter each segment from behind.
template <bool kReverse>
__global__ void __launch_bounds__(256) selective_scan_join_kernel(Params p) {
  const int64_t total = (int64_t)p.batch * p.channels * p.states;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int64_t bc = i / p.states;
  const float a = decay_rate(p.a[(bc % p.channels) * p.states + i % p.states]);
  const float* first = kReverse ? p.dstate_out : p.state;
  float h = first ? first[i] : 0.0f;
  for (int j = 0; j < p.segments; ++j) {
    const bool last = j == p.segments - 1;
    const int k = kReverse ? p.segments - 1 - j : j;
    const float own = last ? 0.0f : p.segment_state[k * total + i];
    const float sum = last ? 0.0f : p.segment_delta[k * (total / p.states) + bc];
    p.segment_state[k * total + i] = h;
    h = fmaf(decay(sum, a), h, own);
  }
}

// Sums v[0 .. 7] over the eight channels of a warp (lane bits 2 to 4); a lane returns the sum of
// v[(its channel)].
__device__ __forceinline__ float channel_sum(float (&v)[8], int lane_in_warp) {
#pragma unroll
  for (int o = 16, half = 4; half > 0; o >>= 1, half >>= 1) {
    const bool upper = lane_in_warp & o;
#pragma unroll
    for (int k = 0; k < half; ++k) {
      const float send = upper ? v[k] : v[k + half];
      const float keep = upper ? v[k + half] : v[k];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// Zeros for the gradients of tokens `from` to `end` of the block's channels (a call of its own: its registers are not
// the recurrence's).
template <typename T>
__device__ __noinline__ void clear_gradients(const Params& p, Channels ch, int batch, int from, int end, int padded) {
  float* dbc = p.dbc + (((int64_t)blockIdx.x * p.batch + batch) * p.length + from) * 2 * padded;
  for (int64_t i = threadIdx.x; i < (int64_t)(end - from) * 2 * padded; i += kBackwardThreads) dbc[i] = 0.0f;
  for (int t = from + threadIdx.x / kBackwardChannels; t < end; t += kBackwardThreads / kBackwardChannels) {
    const int c = threadIdx.x % kBackwardChannels;
    if (c < ch.count) {
      const int64_t at = ((int64_t)batch * p.length + t) * p.channels + ch.first + c;
      static_cast<T*>(p.dx)[at] = static_cast<T*>(p.ddelta)[at] = from_f32<T>(0.0f);
      if (p.z) static_cast<T*>(p.dz)[at] = from_f32<T>(0.0f);
    }
  }
}

// The backward pass.  With dv_t = dy_t silu(z_t) the adjoint of the state is
//
//   g_t = C_t dv_t + c_t,  c_{t-1} = e_t g_t  (c at the end: the gradient of the last state),
//   w_t = c_{t-1} h_{t-1} = g_t e_t h_{t-1}:
//   dx = D dv + delta sum_n g B,  ddelta = x sum_n g B + sum_n A w,  dA = sum_t delta w,
//   dB = sum_d g delta x,  dC = sum_d dv h,  dD = sum dv x,  dz = dy v silu'(z).
//
// Tiles of sixteen tokens are taken from the last to the first, in halves of kCheckpoint tokens: the states
// of a half are run again from its stored first state and stay in registers, with their e, for the
// way back.  A thread holds four states of two channels, so that their terms of dB and dC add up before any
// exchange; sixteen states at a time, and more take further turns over the staged tile.  Sums over the
// states of a channel and over the channels of a warp are transposed butterflies; the block's two warps'
// parts of dB and dC meet in shared memory, the blocks' in global memory, all in a fixed order.  The next tile is
// only called into the L2 cache: registers go to the states.
template <typename T, int kBlocks>
__global__ void __launch_bounds__(kBackwardThreads) selective_scan_backward_kernel(const __grid_constant__ Params p) {
  constexpr int kTile = 16, kHalf = kCheckpoint, kWarps = kBackwardThreads / 32, kChannels = kBackwardChannels;
  constexpr int NP = 16 * kBlocks;
  constexpr int kEach = 8 * 2 * (NP / 4) / kBackwardThreads;  // quads of B and C states per thread
  extern __shared__ __align__(16) float smem[];
  constexpr int kPitch = kChannels + 4;
  float2(*s_du)[kChannels + 2] = reinterpret_cast<float2(*)[kChannels + 2]>(smem);  // (delta, delta x)
  float* at_smem = smem + kTile * (kChannels + 2) * 2;
  float(*s_dv)[kPitch] = reinterpret_cast<float(*)[kPitch]>(at_smem);
  float(*s_v)[kPitch] = s_dv + kTile;   // sum C h
  float(*s_gb)[kPitch] = s_v + kTile;   // sum g B
  float(*s_ga)[kPitch] = s_gb + kTile;  // sum A w / ln 2
  float* s_bc = at_smem + 4 * kTile * kPitch;  // [kTile][2][NP]
  float* s_red = s_bc + kTile * 2 * NP;        // [kBlocks][kWarps][kTile][2][16]
  float* s_kept = s_red + kBlocks * kWarps * kTile * 32 + threadIdx.x;  // [8][threads], this thread's own

  const Channels ch = block_channels(p, kChannels);
  const int batch = blockIdx.y, segment = blockIdx.z;
  const int begin = segment * p.segment_length;
  const int end = min(begin + p.segment_length, p.length);
  const int live = min(end, sequence_length(p.lengths, p.lengths64, batch, p.length));

  // staging: this thread's pair of tokens and four channels
  const int row = threadIdx.x / (kChannels / 4) * 2;
  const int col = threadIdx.x % (kChannels / 4) * 4;
  const int count = max(0, min(4, ch.count - col));
  const bool whole = count == 4;
  float bias[4], skip[4], dd[4], dbias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bias[i] = p.bias && i < count ? p.bias[ch.first + col + i] : 0.0f;
    skip[i] = p.d && i < count ? p.d[ch.first + col + i] : 0.0f;
    dd[i] = dbias[i] = 0.0f;
    s_kept[i * kBackwardThreads] = s_kept[(4 + i) * kBackwardThreads] = 0.0f;
  }
  const T* x = static_cast<const T*>(p.x) + batch * p.x_sb + ch.first + col;
  const T* delta = static_cast<const T*>(p.delta) + batch * p.delta_sb + ch.first + col;
  const T* z = static_cast<const T*>(p.z) + batch * p.z_sb + ch.first + col;
  const T* dy = static_cast<const T*>(p.dy) + batch * p.dy_sb + ch.first + col;
  const int64_t out_at = (int64_t)batch * p.length * p.channels + ch.first + col;
  const T* b = static_cast<const T*>(p.b) + batch * p.b_sb + ch.group * p.b_sg;
  const T* c = static_cast<const T*>(p.c) + batch * p.c_sb + ch.group * p.c_sg;

  // recurrence: this thread's two channels and four states of each sixteen
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane % 4;
  const int mine = warp * 16 + lane / 4 * 2;
  const int64_t state_at = ((int64_t)batch * p.channels + ch.first + mine) * p.states;
  F2 a[kBlocks][2][2], carry[kBlocks][2][2], da[kBlocks][2][2];
  for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float a1[4], c1[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int n = nb * 16 + quad * 4 + s;
        const bool in = mine + j < ch.count && n < p.states;
        a1[s] = in ? decay_rate(p.a[(int64_t)(ch.first + mine + j) * p.states + n]) : 0.0f;
        c1[s] = 0.0f;
        if (in) {
          if (p.segments > 1)
            c1[s] = p.segment_state[(int64_t)segment * p.batch * p.channels * p.states + state_at + j * p.states + n];
          else if (p.dstate_out)
            c1[s] = p.dstate_out[state_at + j * p.states + n];
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        a[nb][j][s] = pack2(a1[2 * s], a1[2 * s + 1]);
        carry[nb][j][s] = pack2(c1[2 * s], c1[2 * s + 1]);
        da[nb][j][s] = 0;
      }
    }
  }
  const int64_t checkpoint_rows = (p.length + kCheckpoint - 1) / kCheckpoint;
  const float* checkpoints = p.checkpoints + ((int64_t)batch * checkpoint_rows * p.channels + ch.first + mine) * NP + quad * 4;

  const int tiles = (end - begin + kTile - 1) / kTile;
  int t0 = begin + (tiles - 1) * kTile;
  // Past the sequence's end all gradients are zero, and the adjoint stays as it is, be it finite or not.
  if (t0 >= begin && t0 >= live) {
    const int from = max(begin, (live - begin + kTile - 1) / kTile * kTile + begin);
    clear_gradients<T>(p, ch, batch, from, end, NP);
    t0 = from - kTile;
  }
  for (; t0 >= begin; t0 -= kTile) {
    struct {
      Raw4<T> x, d, g, z;
    } raw[2];
    const bool in[2] = {t0 + row < live, t0 + row + 1 < live};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t t = t0 + row + q;
      raw[q].x = load4_if<T>(x + t * p.x_st, in[q], count, whole && (p.vec & 1));
      raw[q].d = load4_if<T>(delta + t * p.delta_st, in[q], count, whole && (p.vec & 2));
      raw[q].g = load4_if<T>(dy + t * p.dy_st, in[q], count, whole && (p.vec & 64));
      if (p.z) raw[q].z = load4_if<T>(z + t * p.z_st, in[q], count, whole && (p.vec & 4));
      if (t0 > begin && count > 0) {
        prefetch_l2(x + (t - kTile) * p.x_st);
        prefetch_l2(delta + (t - kTile) * p.delta_st);
        prefetch_l2(dy + (t - kTile) * p.dy_st);
        if (p.z) prefetch_l2(z + (t - kTile) * p.z_st);
      }
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = k * kBackwardThreads + threadIdx.x;
      const int n0 = i % (NP / 4) * 4, which = i / (NP / 4) % 2, t = i / (NP / 4) / 2 * 2;
      const int n1 = max(0, min(4, p.states - n0));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const T* at = which ? c + (int64_t)(t0 + t + q) * p.c_st + n0 : b + (int64_t)(t0 + t + q) * p.b_st + n0;
        const Raw4<T> r = load4_if<T>(at, n1 > 0 && t0 + t + q < live, n1, n1 == 4 && (p.vec & (which ? 32 : 16)));
        *reinterpret_cast<float4*>(s_bc + ((t + q) * 2 + which) * NP + n0) =
            make_float4(value4<T>(r, 0), value4<T>(r, 1), value4<T>(r, 2), value4<T>(r, 3));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      F2 d = add2(pack2(value4<T>(raw[0].d, i), value4<T>(raw[1].d, i)), both(bias[i]));
      if (p.softplus) d = softplus2(d);
      const F2 g = pack2(value4<T>(raw[0].g, i), value4<T>(raw[1].g, i));
      const float2 dv = unpack2(p.z ? gate2(g, pack2(value4<T>(raw[0].z, i), value4<T>(raw[1].z, i))) : g);
      const float2 dl = unpack2(d);
      // past a sequence's end delta is a constant zero, though the adjoint still passes through; x, z, dy, B and C
      // have been read as zero
      const float d0 = in[0] ? dl.x : 0.0f, d1 = in[1] ? dl.y : 0.0f;
      s_du[row][col + i] = make_float2(d0, d0 * value4<T>(raw[0].x, i));
      s_du[row + 1][col + i] = make_float2(d1, d1 * value4<T>(raw[1].x, i));
      s_dv[row][col + i] = dv.x;
      s_dv[row + 1][col + i] = dv.y;
    }
    __syncthreads();
#pragma unroll 1
    for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll 1
      for (int half = kTile / kHalf - 1; half >= 0; --half) {
        const int u0 = half * kHalf;
        F2 h0[2][2], h[kHalf][2][2], e[kHalf][2][2], da_half[2][2] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          ulonglong2 q = make_ulonglong2(0, 0);
          if (mine + j < ch.count && t0 + u0 < p.length)
            q = *reinterpret_cast<const ulonglong2*>(
                checkpoints + ((int64_t)((t0 + u0) / kCheckpoint) * p.channels + j) * NP + nb * 16);
          h0[j][0] = q.x, h0[j][1] = q.y;
        }
#pragma unroll
        for (int t4 = 0; t4 < kHalf; t4 += 4) {
          float v[2][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int t = t4 + k;
            const float4 du = *reinterpret_cast<const float4*>(&s_du[u0 + t][mine]);
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(s_bc + (u0 + t) * 2 * NP + nb * 16 + quad * 4);
            const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(s_bc + ((u0 + t) * 2 + 1) * NP + nb * 16 + quad * 4);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const F2 d2 = both(j ? du.z : du.x), u2 = both(j ? du.w : du.y);
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                e[t][j][s] = decay2(d2, a[nb][j][s]);
                h[t][j][s] = fma2(e[t][j][s], t == 0 ? h0[j][s] : h[t > 0 ? t - 1 : 0][j][s], mul2(u2, s ? bv.y : bv.x));
              }
              const float2 q = unpack2(fma2(cv.y, h[t][j][1], mul2(cv.x, h[t][j][0])));
              v[j][k] = q.x + q.y;
            }
          }
          if (p.z) {  // only the gate's gradient asks for it
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float sum = transpose_sum<4>(v[j], quad);
              float& out = s_v[u0 + t4 + quad][mine + j];
              out = nb == 0 ? sum : out + sum;
            }
          }
        }
#pragma unroll
        for (int t4 = kHalf - 4; t4 >= 0; t4 -= 4) {
          float gb[2][4], ga[2][4];
#pragma unroll
          for (int k = 3; k >= 0; --k) {
            const int t = t4 + k;
            const float4 du = *reinterpret_cast<const float4*>(&s_du[u0 + t][mine]);
            const float2 dv = *reinterpret_cast<const float2*>(&s_dv[u0 + t][mine]);
            const ulonglong2 bv = *reinterpret_cast<const ulonglong2*>(s_bc + (u0 + t) * 2 * NP + nb * 16 + quad * 4);
            const ulonglong2 cv = *reinterpret_cast<const ulonglong2*>(s_bc + ((u0 + t) * 2 + 1) * NP + nb * 16 + quad * 4);
            F2 db[2], dc[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const F2 d2 = both(j ? du.z : du.x), u2 = both(j ? du.w : du.y), dv2 = both(j ? dv.y : dv.x);
              F2 gb2 = 0, ga2 = 0;
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                const F2 g = fma2(s ? cv.y : cv.x, dv2, carry[nb][j][s]);
                db[s] = j == 0 ? mul2(g, u2) : fma2(g, u2, db[s]);
                dc[s] = j == 0 ? mul2(dv2, h[t][j][s]) : fma2(dv2, h[t][j][s], dc[s]);
                gb2 = s == 0 ? mul2(g, bv.x) : fma2(g, bv.y, gb2);
                carry[nb][j][s] = mul2(g, e[t][j][s]);
                const F2 w = mul2(carry[nb][j][s], t == 0 ? h0[j][s] : h[t > 0 ? t - 1 : 0][j][s]);
                ga2 = s == 0 ? mul2(a[nb][j][s], w) : fma2(a[nb][j][s], w, ga2);
                da_half[j][s] = fma2(d2, w, da_half[j][s]);
              }
              const float2 q = unpack2(gb2), r = unpack2(ga2);
              gb[j][k] = q.x + q.y;
              ga[j][k] = r.x + r.y;
            }
            const float2 q0 = unpack2(db[0]), q1 = unpack2(db[1]), r0 = unpack2(dc[0]), r1 = unpack2(dc[1]);
            float both_sums[8] = {q0.x, q0.y, q1.x, q1.y, r0.x, r0.y, r1.x, r1.y};
            const float sum = channel_sum(both_sums, lane);
            const int index = lane >> 2;  // dB or dC, state of the quad
            s_red[((nb * kWarps + warp) * kTile + u0 + t) * 32 + (index >> 2) * 16 + quad * 4 + (index & 3)] = sum;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float sb = transpose_sum<4>(gb[j], quad), sa = transpose_sum<4>(ga[j], quad);
            float& ob = s_gb[u0 + t4 + quad][mine + j];
            float& oa = s_ga[u0 + t4 + quad][mine + j];
            ob = nb == 0 ? sb : ob + sb;
            oa = nb == 0 ? sa : oa + sa;
          }
        }
        // sums of sums: one running sum over thousands of tokens would lose its last bits
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int s = 0; s < 2; ++s) da[nb][j][s] = add2(da[nb][j][s], da_half[j][s]);
      }
    }
    __syncthreads();
    // the warps' parts of dB and dC
    for (int i = threadIdx.x; i < kBlocks * kTile * 32; i += kBackwardThreads) {
      const int nb = i / (kTile * 32), t = i / 32 % kTile;
      if (t0 + t < end) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) sum += s_red[((nb * kWarps + k) * kTile) * 32 + i % (kTile * 32)];
        p.dbc[(((int64_t)blockIdx.x * p.batch + batch) * p.length + t0 + t) * 2 * NP + (i / 16 % 2) * NP + nb * 16 + i % 16] = t0 + t < live ? sum : 0.0f;
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (t0 + row + q < end && count > 0) {
        float o_x[4], o_d[4], o_z[4];
        const float4 gb = *reinterpret_cast<const float4*>(&s_gb[row + q][col]);
        const float4 ga = *reinterpret_cast<const float4*>(&s_ga[row + q][col]);
        const float4 v4 = *reinterpret_cast<const float4*>(&s_v[row + q][col]);
        const float4 dv4 = *reinterpret_cast<const float4*>(&s_dv[row + q][col]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float xv = value4<T>(raw[q].x, i), gbi = (&gb.x)[i], dv = (&dv4.x)[i];
          o_x[i] = fmaf(dv, skip[i], s_du[row + q][col + i].x * gbi);
          o_d[i] = fmaf(xv, gbi, kLn2 * (&ga.x)[i]);
          if (p.softplus) o_d[i] *= sigmoid(value4<T>(raw[q].d, i) + bias[i]);
          if (!in[q]) o_x[i] = o_d[i] = 0.0f;
          if (p.z) {
            const float zv = value4<T>(raw[q].z, i), sg = sigmoid(zv);
            o_z[i] = value4<T>(raw[q].g, i) * sg * (1.0f + zv * (1.0f - sg)) * fmaf(skip[i], xv, (&v4.x)[i]);
            if (!in[q]) o_z[i] = 0.0f;
          }
          dd[i] = fmaf(dv, xv, dd[i]);
          dbias[i] += o_d[i];
        }
        const int64_t at = out_at + (int64_t)(t0 + row + q) * p.channels;
        store4<T>(static_cast<T*>(p.dx) + at, count, whole && (p.vec & 8), o_x);
        store4<T>(static_cast<T*>(p.ddelta) + at, count, whole && (p.vec & 8), o_d);
        if (p.z) store4<T>(static_cast<T*>(p.dz) + at, count, whole && (p.vec & 8), o_z);
      }
    }
    // sums of sums here too (65536 tokens: errors of dD and d(bias) 1.6e-6 and 2.2e-6 in one running sum)
    if ((t0 - begin) / kTile % 32 == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s_kept[i * kBackwardThreads] += dd[i];
        s_kept[(4 + i) * kBackwardThreads] += dbias[i];
        dd[i] = dbias[i] = 0.0f;
      }
    }
    __syncthreads();
  }
  const int64_t part = (int64_t)segment * p.batch + batch;
  for (int nb = 0; nb < kBlocks; ++nb) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int n = nb * 16 + quad * 4 + s;
        if (mine + j < ch.count && n < p.states) {
          const float2 q = unpack2(da[nb][j][s / 2]), r = unpack2(carry[nb][j][s / 2]);
          p.da[(part * p.channels + ch.first + mine + j) * p.states + n] = s % 2 ? q.y : q.x;
          if (p.dstate && segment == 0) p.dstate[state_at + j * p.states + n] = s % 2 ? r.y : r.x;
        }
      }
    }
  }
  // d(D) and d(bias): the eight pairs' threads of each channel, in a fixed order
  float* s_sum = smem;  // [8][2][kChannels]
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_sum[(row / 2 * 2 + 0) * kChannels + col + i] = s_kept[i * kBackwardThreads];
    s_sum[(row / 2 * 2 + 1) * kChannels + col + i] = s_kept[(4 + i) * kBackwardThreads];
  }
  __syncthreads();
  {
    const int which = threadIdx.x / kChannels, k = threadIdx.x % kChannels;
    float sum = 0.0f;
    for (int t = 0; t < kTile / 2; ++t) sum += s_sum[(t * 2 + which) * kChannels + k];
    if (k < ch.count) p.dd[(part * 2 + which) * p.channels + ch.first + k] = sum;
  }
}

template <int kBlocks>
constexpr int backward_smem_bytes() {
  return (16 * (32 + 2) * 2 + 4 * 16 * 36 + 16 * 2 * 16 * kBlocks + kBlocks * 2 * 16 * 32 +
          8 * kBackwardThreads) * 4;
}

// dB and dC from the channel blocks' parts, in the order of the blocks.
template <typename T>
__global__ void __launch_bounds__(256) selective_scan_dbc_kernel(const float* parts, T* db, T* dc, int64_t tokens, int groups,
                                                                 int per_group, int states, int padded) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t total = tokens * groups * 2 * padded;
  if (i >= total) return;
  const int n = (int)(i % padded);
  const int which = (int)(i / padded % 2);
  const int64_t token = i / (2 * padded) / groups;
  const int group = (int)(i / (2 * padded) % groups);
  if (n >= states) return;
  float sum = 0.0f;
  for (int k = 0; k < per_group; ++k)
    sum += parts[((int64_t)(group * per_group + k) * tokens + token) * 2 * padded + which * padded + n];
  (which ? dc : db)[(token * groups + group) * states + n] = from_f32<T>(sum);
}

// One token: every state is read and written once, four lanes on a channel with four states at a time.  The
// first four states' loads and those of everything else go out together; `four`: states, A, B and C come
// in aligned groups of four.
template <typename T>
__global__ void __launch_bounds__(128) selective_scan_step_kernel(const __grid_constant__ Params p, int four) {
  constexpr int kLanes = 4;
  const int64_t at = (int64_t)blockIdx.x * (128 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const bool in = at < (int64_t)p.batch * p.channels;
  const int b = in ? (int)(at / p.channels) : 0;
  const int c = in ? (int)(at - (int64_t)b * p.channels) : 0;
  const int group = p.groups == 1 ? 0 : c / (p.channels / p.groups);
  const T* bv = static_cast<const T*>(p.b) + b * p.b_sb + group * p.b_sg;
  const T* cv = static_cast<const T*>(p.c) + b * p.c_sb + group * p.c_sg;
  float* state = p.state_out + at * p.states;
  const float* a = p.a + (int64_t)c * p.states;
  float4 h4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), a4 = h4;
  Raw4<T> b4, c4;
  const bool first = in && four && lane * 4 < p.states;
  if (first) {
    h4 = *reinterpret_cast<const float4*>(state + lane * 4);
    a4 = *reinterpret_cast<const float4*>(a + lane * 4);
  }
  b4 = load4_if<T>(bv + lane * 4, first, 4, true);
  c4 = load4_if<T>(cv + lane * 4, first, 4, true);
  const float x = to_f32(static_cast<const T*>(p.x)[b * p.x_sb + c]);
  float delta = to_f32(static_cast<const T*>(p.delta)[b * p.delta_sb + c]) + (p.bias ? p.bias[c] : 0.0f);
  const float zv = p.z ? to_f32(static_cast<const T*>(p.z)[b * p.z_sb + c]) : 0.0f;
  const float skip = p.d ? p.d[c] : 0.0f;
  if (p.softplus) delta = softplus(delta);
  const float u = delta * x, d2 = delta * kLog2e;
  float v = 0.0f;
  auto quad = [&](int n) {
    h4.x = fmaf(decay(d2, a4.x), h4.x, u * value4<T>(b4, 0));
    h4.y = fmaf(decay(d2, a4.y), h4.y, u * value4<T>(b4, 1));
    h4.z = fmaf(decay(d2, a4.z), h4.z, u * value4<T>(b4, 2));
    h4.w = fmaf(decay(d2, a4.w), h4.w, u * value4<T>(b4, 3));
    *reinterpret_cast<float4*>(state + n) = h4;
    v = fmaf(value4<T>(c4, 0), h4.x, v);
    v = fmaf(value4<T>(c4, 1), h4.y, v);
    v = fmaf(value4<T>(c4, 2), h4.z, v);
    v = fmaf(value4<T>(c4, 3), h4.w, v);
  };
  if (first) {
    quad(lane * 4);
    for (int n = (lane + kLanes) * 4; n < p.states; n += kLanes * 4) {
      h4 = *reinterpret_cast<const float4*>(state + n);
      a4 = *reinterpret_cast<const float4*>(a + n);
      b4 = load4_if<T>(bv + n, true, 4, true);
      c4 = load4_if<T>(cv + n, true, 4, true);
      quad(n);
    }
  } else if (in && !four) {
    for (int n = lane; n < p.states; n += kLanes) {
      const float h = fmaf(decay(d2, a[n]), state[n], u * to_f32(bv[n]));
      v = fmaf(to_f32(cv[n]), h, v);
      state[n] = h;
    }
  }
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (in && lane == 0) {
    v = fmaf(skip, x, v);
    if (p.z) v *= zv * sigmoid(zv);
    static_cast<T*>(p.y)[at] = from_f32<T>(v);
  }
}

}  // namespace scan
}  // namespace xe
