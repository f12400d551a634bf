// Short causal convolution over the time axis, one filter per channel, channel-last:
//
//   pre[t, c] = bias[c] + sum_j w[c, j] v[t - W + 1 + j, c],  y = pre or silu(pre),
//
// with v = x from t = 0 on and the state (the W - 1 inputs before) at negative t.  The new state is
// the last W - 1 entries of the sequence [state, x[:length]].
//
//   dpre = dy * silu'(pre),  dv[t] = sum_j w_j dpre[t + W - 1 - j],  dw_j = sum_t dpre[t] v[t - W + 1 + j].
//
// Bound by memory: a thread owns eight channels (16 bytes of a 16-bit type) and walks a chunk of
// tokens with the window in registers, so that x is read once and W - 1 rows again per chunk.
#pragma once

#include "seq_common.cuh"

namespace xe {
namespace conv {

using namespace seq;

struct Params {
  const void* x;
  const float* weight;  // (channels, width) contiguous
  const float* bias;    // or null
  const void* state;    // (batch, width - 1, channels) contiguous, or null = zeros
  void* y;              // (batch, length, channels) contiguous
  void* state_out;      // like state, or null
  const void* lengths;
  int lengths64;
  int64_t x_sb, x_st;
  int batch, length, channels, chunk;
  int silu;
  int vec;  // bit 0: x, 1: state, 2: y and state_out, 3: dy, 4: dstate
  // backward
  const void* dy;
  int64_t dy_sb, dy_st;
  const void* dstate_out;  // gradient of the new state, contiguous, or null
  void* dx;
  void* dstate;    // gradient of the state, contiguous, or null
  float* partial;  // (batch * chunks, channels, width + 1)
};

template <typename T, int W>
__device__ __forceinline__ void load_filter(const Params& p, int c0, int count, float (&w)[W][8], float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    b[i] = p.bias && i < count ? p.bias[c0 + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) w[j][i] = i < count ? p.weight[(int64_t)(c0 + i) * W + j] : 0.0f;
  }
}

// v[t] of the sequence with the state in front: t in [-(W - 1), length).
template <typename T, int W>
__device__ __forceinline__ Raw8<T> value_at(const Params& p, int b, int t, int c0, int count) {
  if (t >= 0)
    return load8<T>(static_cast<const T*>(p.x) + b * p.x_sb + t * p.x_st + c0, count, p.vec & 1);
  if (p.state)
    return load8<T>(static_cast<const T*>(p.state) + ((int64_t)b * (W - 1) + (t + W - 1)) * p.channels + c0, count,
                    p.vec & 2);
  Raw8<T> z;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) z.q[i] = make_uint4(0, 0, 0, 0);
  return z;
}

template <typename T>
__device__ __forceinline__ void store_raw(T* p, int count, bool vec, const Raw8<T>& r) {
  float v[8];
  unpack8<T>(r, v);
  store8<T>(p, count, vec, v);
}

template <typename T, int W>
__global__ void __launch_bounds__(128) causal_conv_kernel(Params p) {
  const int c0 = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (c0 >= p.channels) return;
  const int count = min(8, p.channels - c0);
  const int b = blockIdx.z;
  const int first = blockIdx.y * p.chunk;
  const int last = min(first + p.chunk, p.length);
  const int length = sequence_length(p.lengths, p.lengths64, b, p.length);
  T* y = static_cast<T*>(p.y) + (int64_t)b * p.length * p.channels + c0;
  if (p.state_out && blockIdx.y == 0) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      store_raw<T>(static_cast<T*>(p.state_out) + ((int64_t)b * (W - 1) + j) * p.channels + c0, count, p.vec & 4,
                   value_at<T, W>(p, b, length - (W - 1) + j, c0, count));
  }
  float w[W][8], bias[8];
  load_filter<T, W>(p, c0, count, w, bias);
  float window[W][8];  // v[t - W + 1 .. t]
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = first - (W - 1) + j;
    if (t < length) {
      unpack8<T>(value_at<T, W>(p, b, t, c0, count), window[j + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) window[j + 1][i] = 0.0f;
    }
  }
  const int live = min(last, length);
  constexpr int kAhead = 4;
  int t = first;
  for (; t < live; t += kAhead) {
    Raw8<T> raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (t + k < live) raw[k] = value_at<T, W>(p, b, t + k, c0, count);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (t + k < live) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) window[j][i] = window[j + 1][i];
        unpack8<T>(raw[k], window[W - 1]);
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i] = bias[i];
#pragma unroll
          for (int j = 0; j < W; ++j) o[i] = fmaf(w[j][i], window[j][i], o[i]);
          if (p.silu) o[i] *= sigmoid(o[i]);
        }
        store8<T>(y + (int64_t)(t + k) * p.channels, count, p.vec & 4, o);
      }
    }
  }
  const float zero[8] = {};
  for (t = max(first, live); t < last; ++t) store8<T>(y + (int64_t)t * p.channels, count, p.vec & 4, zero);
}

// One token: the state is shifted in place.
template <typename T, int W>
__global__ void __launch_bounds__(128) causal_conv_step_kernel(Params p) {
  const int vectors = (p.channels + 7) / 8;
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= (int64_t)p.batch * vectors) return;
  const int b = (int)(at / vectors);
  const int c0 = (int)(at % vectors) * 8;
  const int count = min(8, p.channels - c0);
  T* state = static_cast<T*>(p.state_out) + (int64_t)b * (W - 1) * p.channels + c0;
  Raw8<T> window[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    // plain loads: the same thread writes these places below
    float v[8];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) window[j].q[i] = make_uint4(0, 0, 0, 0);
    if ((p.vec & 2) && count == 8) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        window[j].q[i] = reinterpret_cast<const uint4*>(state + (int64_t)j * p.channels)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < count) reinterpret_cast<T*>(&window[j])[i] = state[(int64_t)j * p.channels + i];
    }
    (void)v;
  }
  window[W - 1] = load8<T>(static_cast<const T*>(p.x) + b * p.x_sb + c0, count, p.vec & 1);
  float w[W][8], o[8];
  load_filter<T, W>(p, c0, count, w, o);
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float v[8];
    unpack8<T>(window[j], v);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf(w[j][i], v[i], o[i]);
    if (j > 0) store8<T>(state + (int64_t)(j - 1) * p.channels, count, p.vec & 2, v);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (p.silu) o[i] *= sigmoid(o[i]);
  store8<T>(static_cast<T*>(p.y) + (int64_t)b * p.channels + c0, count, p.vec & 4, o);
}

// Backward of a chunk of tokens: a thread walks t over [first, last + W - 1), keeps the W newest
// v and the W newest dpre, and completes dx[t - W + 1] at t.  dw and dbias count dpre of the
// chunk's own tokens only.
template <typename T, int W>
__global__ void __launch_bounds__(128) causal_conv_backward_kernel(Params p) {
  const int c0 = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
  if (c0 >= p.channels) return;
  const int count = min(8, p.channels - c0);
  const int b = blockIdx.z;
  const int first = blockIdx.y * p.chunk;
  const int last = min(first + p.chunk, p.length);
  const int length = sequence_length(p.lengths, p.lengths64, b, p.length);
  float w[W][8], bias[8];
  load_filter<T, W>(p, c0, count, w, bias);
  float window[W][8], dpre[W][8], dw[W][8], db[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    db[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) dw[j][i] = dpre[j][i] = window[j][i] = 0.0f;
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    const int t = first - (W - 1) + j;
    if (t < length) unpack8<T>(value_at<T, W>(p, b, t, c0, count), window[j + 1]);
  }
  const T* dy = static_cast<const T*>(p.dy) + b * p.dy_sb + c0;
  T* dx = static_cast<T*>(p.dx) + (int64_t)b * p.length * p.channels + c0;
  const T* ds = p.dstate_out ? static_cast<const T*>(p.dstate_out) + (int64_t)b * (W - 1) * p.channels + c0 : nullptr;
  // the first chunk also completes the gradients of the state, at negative t
  T* dstate = p.dstate ? static_cast<T*>(p.dstate) + (int64_t)b * (W - 1) * p.channels + c0 : nullptr;
  for (int t = first; t < last + W - 1; ++t) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        window[j][i] = window[j + 1][i];
        dpre[j][i] = dpre[j + 1][i];
      }
#pragma unroll
    for (int i = 0; i < 8; ++i) dpre[W - 1][i] = 0.0f;
    if (t < length) {
      float g[8];
      unpack8<T>(value_at<T, W>(p, b, t, c0, count), window[W - 1]);
      load8f<T>(dy + t * p.dy_st, count, p.vec & 8, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (p.silu) {
          float pre = bias[i];
#pragma unroll
          for (int j = 0; j < W; ++j) pre = fmaf(w[j][i], window[j][i], pre);
          const float s = sigmoid(pre);
          g[i] *= s * (1.0f + pre * (1.0f - s));
        }
        dpre[W - 1][i] = g[i];
        if (t < last) {
          db[i] += g[i];
#pragma unroll
          for (int j = 0; j < W; ++j) dw[j][i] = fmaf(g[i], window[j][i], dw[j][i]);
        }
      }
    }
    const int at = t - (W - 1);  // complete: dpre holds [at, at + W - 1]
    if (at < first && !(first == 0 && dstate)) continue;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < W; ++j) o[i] = fmaf(w[W - 1 - j][i], dpre[j][i], o[i]);
    }
    // entry `at` of [state, x[:length]] is also entry at - (length - W + 1) of the new state
    const int kept = at - (length - (W - 1));
    if (ds && kept >= 0 && kept < W - 1) {
      float e[8];
      load8f<T>(ds + (int64_t)kept * p.channels, count, p.vec & 16, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] += e[i];
    }
    if (at < 0)
      store8<T>(dstate + (int64_t)(at + W - 1) * p.channels, count, p.vec & 16, o);
    else
      store8<T>(dx + (int64_t)at * p.channels, count, p.vec & 4, o);
  }
  float* out = p.partial + (((int64_t)b * gridDim.y + blockIdx.y) * p.channels + c0) * (W + 1);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i < count) {
#pragma unroll
      for (int j = 0; j < W; ++j) out[i * (W + 1) + j] = dw[j][i];
      out[i * (W + 1) + W] = db[i];
    }
  }
}

}  // namespace conv
}  // namespace xe
