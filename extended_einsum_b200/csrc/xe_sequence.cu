// C ABI of the sequence operators (declared in include/xe_b200.h): the causal convolution, the
// selective scan, the root-mean-square norm and the products with 4-bit weights.  Their kernels have
// no device-side waits, so this translation unit has no use of the device status word.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>

#include "../../include/xe_b200.h"
#include "causal_conv.cuh"
#include "host_status.h"
#include "int4_linear.cuh"
#include "rms_norm.cuh"
#include "selective_scan.cuh"

namespace {

using xe::fail;

xe_status launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? XE_OK : fail(XE_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }
inline bool is_float(int32_t dtype) { return dtype == XE_F32 || dtype == XE_BF16 || dtype == XE_F16; }
inline int64_t size_of(int32_t dtype) { return dtype == XE_F32 ? 4 : dtype == XE_BF16 || dtype == XE_F16 ? 2 : 1; }

// Whether every row starts on a multiple of `bytes`.
bool aligned(int64_t bytes, const void* p, int32_t dtype, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  for (int64_t s : strides)
    if (s * size_of(dtype) % bytes) return false;
  return true;
}
bool vectors(const void* p, int32_t dtype, std::initializer_list<int64_t> strides) { return aligned(16, p, dtype, strides); }

// A workspace of at least `need` bytes, on a boundary that suits every vector stored to it.
xe_status check_workspace(const char* what, const void* workspace, size_t bytes, size_t need) {
  if (need == 0) return XE_OK;
  if (!workspace || bytes < need) return fail(XE_ERR_INVALID_ARGUMENT, "%s: workspace too small", what);
  if (reinterpret_cast<uintptr_t>(workspace) % 256)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: workspace must be 256-byte aligned", what);
  return XE_OK;
}

template <typename F>
void by_type(int32_t dtype, F f) {
  if (dtype == XE_F32)
    f(float{});
  else if (dtype == XE_BF16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

xe_status sum_rows(const float* partial, int64_t rows, int64_t columns, float* out, cudaStream_t stream) {
  xe::seq::sum_rows_kernel<<<(unsigned)ceil_div(columns, 32), dim3(32, 32), 0, stream>>>(partial, rows, columns, out);
  return launched("sum_rows");
}

// ------------------------------------------------------------------ convolution

xe_status check_conv(const char* what, const void* x, const void* weight, const void* y, int64_t batch, int64_t length,
                     int64_t channels, int64_t width, int32_t activation, int32_t dtype) {
  // an empty tensor may have no address
  if (batch * length * channels != 0 && (!x || !y)) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (batch * channels != 0 && !weight) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!is_float(dtype)) return fail(XE_ERR_NOT_SUPPORTED, "%s: element type %d", what, dtype);
  if (batch < 0 || length < 0 || channels < 0 || width < 1)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: negative size or width below 1", what);
  if (width > 4) return fail(XE_ERR_NOT_SUPPORTED, "%s: width %lld above 4", what, (long long)width);
  if (activation != 0 && activation != 1) return fail(XE_ERR_INVALID_ARGUMENT, "%s: activation %d", what, activation);
  if (batch > 65535 || length > INT_MAX / 2 || channels > INT_MAX / 2)
    return fail(XE_ERR_NOT_SUPPORTED, "%s: a size is above its limit", what);
  return XE_OK;
}

template <typename F>
void by_width(int64_t width, F f) {
  switch (width) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    default: f(std::integral_constant<int, 4>{});
  }
}

// Four channels per thread where every row allows it, else one.
bool fours(const void* p, int32_t dtype, std::initializer_list<int64_t> strides) {
  return aligned(4 * size_of(dtype), p, dtype, strides);
}
template <typename F>
void by_vector(int32_t dtype, bool vec, F f) {
  by_type(dtype, [&](auto t) {
    if (vec)
      f(t, std::integral_constant<int, 4>{});
    else
      f(t, std::integral_constant<int, 1>{});
  });
}

// How the length is cut into chunks.  A chunk reads width - 1 rows twice, so there are only as many
// as fill the device's resident threads (`resident` an SM at the kernel's registers) a whole number of times, of at
// most 256 tokens.  The backward pass is planned for vectors of four whatever the alignment, so that its
// workspace depends on the sizes alone.
struct ConvPlan {
  int64_t chunk, chunks;
};
constexpr int64_t kConvResident = 896, kConvBackwardResident = 512;
ConvPlan conv_plan(int64_t batch, int64_t length, int64_t vectors, int64_t resident) {
  if (length < 1) return {1, 1};
  const int64_t rows = std::max<int64_t>(1, batch * vectors), device = 148 * resident;
  const int64_t turns = std::max<int64_t>(1, ceil_div(rows * ceil_div(length, 256), device));
  int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(turns * device / rows, ceil_div(length, 8)));
  const int64_t chunk = ceil_div(length, chunks);
  return {chunk, ceil_div(length, chunk)};
}

template <typename F>
xe_status launch_conv(const char* what, const xe::conv::Params& p, int V, F kernel, cudaStream_t stream) {
  const int64_t blocks = ceil_div((int64_t)(p.channels / V) * p.chunks, xe::conv::kThreads);
  if (blocks > INT_MAX) return fail(XE_ERR_NOT_SUPPORTED, "%s: a size is above its limit", what);
  kernel<<<dim3((unsigned)blocks, (unsigned)p.batch), xe::conv::kThreads, 0, stream>>>(p);
  return launched(what);
}

}  // namespace

extern "C" {

xe_status xe_causal_conv1d(const void* x, int64_t x_sb, int64_t x_st, const float* weight, const float* bias,
                           const void* state, void* y, void* state_out, const void* lengths, int32_t lengths64,
                           int64_t batch, int64_t length, int64_t channels, int64_t width, int32_t activation,
                           int32_t dtype, void* stream) {
  const char* what = "xe_causal_conv1d";
  if (xe_status s = check_conv(what, x, weight, y, batch, length, channels, width, activation, dtype)) return s;
  if (batch == 0 || channels == 0) return XE_OK;
  xe::conv::Params p{};
  p.x = x, p.weight = weight, p.bias = bias, p.state = state, p.y = y, p.state_out = state_out;
  p.lengths = lengths, p.lengths64 = lengths64;
  p.x_sb = x_sb, p.x_st = x_st;
  p.batch = (int)batch, p.length = (int)length, p.channels = (int)channels;
  p.silu = activation;
  const bool vec = fours(x, dtype, {x_sb, x_st}) && fours(y, dtype, {channels}) && fours(state, dtype, {}) &&
                   fours(state_out, dtype, {});
  xe_status status = XE_OK;
  by_vector(dtype, vec, [&](auto t, auto v) {
    constexpr int V = decltype(v)::value;
    const ConvPlan plan = conv_plan(batch, length, channels / V, kConvResident);
    p.chunk = (int)plan.chunk, p.chunks = (int)plan.chunks;
    by_width(width, [&](auto w) {
      status = launch_conv(what, p, V, xe::conv::causal_conv_kernel<decltype(t), decltype(w)::value, V>, as_stream(stream));
    });
  });
  return status;
}

xe_status xe_causal_conv1d_step(const void* x, int64_t x_sb, const float* weight, const float* bias, void* state, void* y,
                                int64_t batch, int64_t channels, int64_t width, int32_t activation, int32_t dtype,
                                void* stream) {
  const char* what = "xe_causal_conv1d_step";
  if (xe_status s = check_conv(what, x, weight, y, batch > 65535 ? 1 : batch, 1, channels, width, activation, dtype)) return s;
  if (width > 1 && batch * channels != 0 && !state) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null state", what);
  if (batch > INT_MAX / 2) return fail(XE_ERR_NOT_SUPPORTED, "%s: a size is above its limit", what);
  if (batch == 0 || channels == 0) return XE_OK;
  xe::conv::Params p{};
  p.x = x, p.weight = weight, p.bias = bias, p.y = y, p.state_out = state;
  p.x_sb = x_sb;
  p.batch = (int)batch, p.channels = (int)channels, p.silu = activation;
  const bool vec = fours(x, dtype, {x_sb}) && fours(y, dtype, {channels}) && fours(state, dtype, {});
  by_vector(dtype, vec, [&](auto t, auto v) {
    constexpr int V = decltype(v)::value;
    const unsigned grid = (unsigned)ceil_div(batch * (channels / V), xe::conv::kThreads);
    by_width(width, [&](auto w) {
      xe::conv::causal_conv_step_kernel<decltype(t), decltype(w)::value, V>
          <<<grid, xe::conv::kThreads, 0, as_stream(stream)>>>(p);
    });
  });
  return launched(what);
}

size_t xe_causal_conv1d_backward_workspace_size(int64_t batch, int64_t length, int64_t channels, int64_t width) {
  if (batch <= 0 || length < 0 || channels <= 0 || width < 1 || width > 4) return 0;
  return padded((size_t)(batch * conv_plan(batch, length, ceil_div(channels, 4), kConvBackwardResident).chunks * channels * (width + 1)) * 4);
}

xe_status xe_causal_conv1d_backward(const void* x, int64_t x_sb, int64_t x_st, const float* weight, const float* bias,
                                    const void* state, const void* dy, int64_t dy_sb, int64_t dy_st,
                                    const void* dstate_out, void* dx, void* dstate, float* dweight,
                                    const void* lengths, int32_t lengths64, int64_t batch, int64_t length,
                                    int64_t channels, int64_t width, int32_t activation, int32_t dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* what = "xe_causal_conv1d_backward";
  if (xe_status s = check_conv(what, x, weight, dx, batch, length, channels, width, activation, dtype)) return s;
  if (channels == 0) return XE_OK;
  if ((batch * length != 0 && !dy) || !dweight) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (batch == 0) return fail(XE_ERR_INVALID_ARGUMENT, "%s: an empty batch has no gradients", what);
  if (xe_status s = check_workspace(what, workspace, workspace_bytes,
                                    xe_causal_conv1d_backward_workspace_size(batch, length, channels, width)))
    return s;
  xe::conv::Params p{};
  p.x = x, p.weight = weight, p.bias = bias, p.state = state;
  p.dy = dy, p.dy_sb = dy_sb, p.dy_st = dy_st, p.dstate_out = dstate_out, p.dx = dx, p.dstate = dstate;
  p.partial = static_cast<float*>(workspace);
  p.lengths = lengths, p.lengths64 = lengths64;
  p.x_sb = x_sb, p.x_st = x_st;
  p.batch = (int)batch, p.length = (int)length, p.channels = (int)channels;
  p.silu = activation;
  const bool vec = fours(x, dtype, {x_sb, x_st}) && fours(dx, dtype, {channels}) && fours(state, dtype, {}) &&
                   fours(dy, dtype, {dy_sb, dy_st}) && fours(dstate_out, dtype, {}) && fours(dstate, dtype, {});
  const ConvPlan plan = conv_plan(batch, length, ceil_div(channels, 4), kConvBackwardResident);
  p.chunk = (int)plan.chunk, p.chunks = (int)plan.chunks;
  xe_status status = XE_OK;
  by_vector(dtype, vec, [&](auto t, auto v) {
    constexpr int V = decltype(v)::value;
    by_width(width, [&](auto w) {
      status = launch_conv(what, p, V, xe::conv::causal_conv_backward_kernel<decltype(t), decltype(w)::value, V>,
                           as_stream(stream));
    });
  });
  if (status != XE_OK) return status;
  return sum_rows(p.partial, batch * plan.chunks, channels * (width + 1), dweight, as_stream(stream));
}

}  // extern "C"

// ------------------------------------------------------------------ scan

namespace {

using ScanParams = xe::scan::Params;

int scan_blocks(int64_t states) { return states <= 16 ? 1 : states <= 32 ? 2 : 4; }

struct ScanPlan {
  int segments, segment_length;
  int64_t channel_blocks;  // of the backward kernel: 32 channels
};

// How many segments the length is split into.  A split costs a pass of its own over x, delta and B, so
// it is taken only where the whole sequences give the device too few blocks, and no segment is shorter than 64
// tokens (forward, 300 tokens of 2048 channels: 31 us in segments of at least 128, 25 of 64, 21 of 32; forward and
// backward, 512 tokens of 1024 channels: 101, 70, 63; 509 of 3 x 1000: 40, 35, 35).
ScanPlan scan_plan(int64_t batch, int64_t length, int64_t channels, int64_t groups) {
  ScanPlan plan;
  plan.channel_blocks = groups * ceil_div(channels / groups, 32);
  const int64_t blocks = plan.channel_blocks * batch;
  int64_t segments = 1;
  if (blocks < 296) segments = std::max<int64_t>(1, std::min<int64_t>(592 / blocks, length / 64));
  plan.segment_length = (int)std::max<int64_t>(32, ceil_div(ceil_div(length, segments), 32) * 32);
  plan.segments = (int)std::max<int64_t>(1, ceil_div(length, plan.segment_length));
  return plan;
}

size_t scan_segment_bytes(const ScanPlan& plan, int64_t batch, int64_t channels, int64_t states) {
  if (plan.segments == 1) return 0;
  return padded((size_t)(plan.segments * batch * channels * states) * 4) + padded((size_t)(plan.segments * batch * channels) * 4);
}

xe_status check_scan(const char* what, const xe_selective_scan_args* q, bool step) {
  if (!q) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
  // an empty tensor may have no address
  const int64_t tokens = q->batch * (step ? 1 : q->length);
  if ((tokens * q->channels != 0 && (!q->x || !q->delta || !q->b || !q->c || !q->a)) ||
      (q->batch * q->channels != 0 && !q->a))
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!is_float(q->dtype)) return fail(XE_ERR_NOT_SUPPORTED, "%s: element type %d", what, q->dtype);
  if (q->batch < 0 || q->length < 0 || q->channels < 0 || q->states < 1 || q->groups < 1)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: negative size, or no states or groups", what);
  if (q->channels % q->groups)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: %lld channels do not divide into %lld groups", what, (long long)q->channels,
                (long long)q->groups);
  if (reinterpret_cast<uintptr_t>(q->checkpoints) % 16)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: checkpoints must be 16-byte aligned", what);
  if (q->states > 64 && !step) return fail(XE_ERR_NOT_SUPPORTED, "%s: %lld states above 64", what, (long long)q->states);
  if ((!step && q->batch > 65535) || q->batch > INT_MAX / 2 || q->length > INT_MAX / 2 || q->channels > INT_MAX / 2 ||
      q->states > 65536)
    return fail(XE_ERR_NOT_SUPPORTED, "%s: a size is above its limit", what);
  return XE_OK;
}

ScanParams scan_params(const xe_selective_scan_args* q) {
  ScanParams p{};
  p.x = q->x, p.delta = q->delta, p.z = q->z, p.b = q->b, p.c = q->c, p.y = q->y;
  p.a = q->a, p.d = q->d, p.bias = q->delta_bias;
  p.state = q->state, p.state_out = q->state_out, p.checkpoints = q->checkpoints;
  p.lengths = q->lengths, p.lengths64 = q->lengths64;
  p.x_sb = q->x_sb, p.x_st = q->x_st, p.delta_sb = q->delta_sb, p.delta_st = q->delta_st;
  p.z_sb = q->z_sb, p.z_st = q->z_st;
  p.b_sb = q->b_sb, p.b_st = q->b_st, p.b_sg = q->b_sg;
  p.c_sb = q->c_sb, p.c_st = q->c_st, p.c_sg = q->c_sg;
  p.batch = (int)q->batch, p.length = (int)q->length, p.channels = (int)q->channels;
  p.states = (int)q->states, p.groups = (int)q->groups;
  p.softplus = q->softplus;
  const int64_t each = q->channels / q->groups;  // a group's first channel starts a vector
  p.vec = (fours(q->x, q->dtype, {q->x_sb, q->x_st, each}) ? 1 : 0) |
          (fours(q->delta, q->dtype, {q->delta_sb, q->delta_st, each}) ? 2 : 0) |
          (fours(q->z, q->dtype, {q->z_sb, q->z_st, each}) ? 4 : 0) |
          (fours(q->y, q->dtype, {q->channels, each}) ? 8 : 0) |
          (fours(q->b, q->dtype, {q->b_sb, q->b_st, q->b_sg}) ? 16 : 0) |
          (fours(q->c, q->dtype, {q->c_sb, q->c_st, q->c_sg}) ? 32 : 0);
  return p;
}

void scan_segments(ScanParams& p, const ScanPlan& plan, void* workspace) {
  p.segments = plan.segments, p.segment_length = plan.segment_length;
  if (plan.segments == 1) return;
  p.segment_state = static_cast<float*>(workspace);
  p.segment_delta = reinterpret_cast<float*>(
      static_cast<char*>(workspace) + padded((size_t)p.segments * p.batch * p.channels * p.states * 4));
}

template <xe::scan::Mode kMode>
xe_status launch_scan(const ScanParams& p, const ScanPlan& plan, int32_t dtype, cudaStream_t stream) {
  using namespace xe::scan;
  const int kC = p.states <= 32 ? 2 : 1;
  const int64_t blocks = (int64_t)p.groups * ceil_div(p.channels / p.groups, 8 * kC);
  const dim3 grid((unsigned)blocks, (unsigned)p.batch, (unsigned)(kMode == kFull ? p.segments : p.segments - 1));
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (p.states <= 16)
      selective_scan_kernel<T, 4, 2, kMode><<<grid, 64, 0, stream>>>(p);
    else if (p.states <= 32)
      selective_scan_kernel<T, 8, 2, kMode><<<grid, 64, 0, stream>>>(p);
    else
      selective_scan_kernel<T, 16, 1, kMode><<<grid, 64, 0, stream>>>(p);
  });
  return launched("selective scan");
}

template <bool kReverse>
xe_status join_scan(const ScanParams& p, cudaStream_t stream) {
  const int64_t total = (int64_t)p.batch * p.channels * p.states;
  xe::scan::selective_scan_join_kernel<kReverse><<<(unsigned)ceil_div(total, 256), 256, 0, stream>>>(p);
  return launched("selective scan join");
}

template <typename T, int kBlocks>
xe_status launch_scan_backward(const ScanParams& p, const ScanPlan& plan, cudaStream_t stream) {
  using namespace xe::scan;
  constexpr int kBytes = backward_smem_bytes<kBlocks>();
  static std::atomic<uint32_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(done.load() >> (dev & 31) & 1u)) {
    const cudaError_t e = cudaFuncSetAttribute(selective_scan_backward_kernel<T, kBlocks>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess) return fail(XE_ERR_CUDA, "selective scan backward: %s", cudaGetErrorString(e));
    done.fetch_or(1u << (dev & 31));
  }
  const dim3 grid((unsigned)plan.channel_blocks, (unsigned)p.batch, (unsigned)p.segments);
  selective_scan_backward_kernel<T, kBlocks><<<grid, kBackwardThreads, kBytes, stream>>>(p);
  return launched("selective scan backward");
}

}  // namespace

extern "C" {

size_t xe_selective_scan_workspace_size(int64_t batch, int64_t length, int64_t channels, int64_t states, int64_t groups) {
  if (batch <= 0 || length < 0 || channels <= 0 || states < 1 || groups < 1 || channels % groups) return 0;
  return scan_segment_bytes(scan_plan(batch, length, channels, groups), batch, channels, states);
}

size_t xe_selective_scan_checkpoint_size(int64_t batch, int64_t length, int64_t channels, int64_t states) {
  if (batch <= 0 || length <= 0 || channels <= 0 || states < 1 || states > 64) return 0;
  return (size_t)(batch * ceil_div(length, xe::scan::kCheckpoint) * channels * 16 * scan_blocks(states)) * 4;
}

xe_status xe_selective_scan(const xe_selective_scan_args* q, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "xe_selective_scan";
  if (xe_status s = check_scan(what, q, false)) return s;
  if (q->batch == 0 || q->channels == 0) return XE_OK;
  if (q->length > 0 && !q->y) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  const ScanPlan plan = scan_plan(q->batch, q->length, q->channels, q->groups);
  if (xe_status s = check_workspace(what, workspace, workspace_bytes, scan_segment_bytes(plan, q->batch, q->channels, q->states)))
    return s;
  ScanParams p = scan_params(q);
  scan_segments(p, plan, workspace);
  if (p.segments > 1) {
    if (xe_status s = launch_scan<xe::scan::kStates>(p, plan, q->dtype, as_stream(stream))) return s;
    if (xe_status s = join_scan<false>(p, as_stream(stream))) return s;
  }
  return launch_scan<xe::scan::kFull>(p, plan, q->dtype, as_stream(stream));
}

xe_status xe_selective_scan_step(const xe_selective_scan_args* q, void* stream) {
  const char* what = "xe_selective_scan_step";
  if (xe_status s = check_scan(what, q, true)) return s;
  if (q->batch == 0 || q->channels == 0) return XE_OK;
  if (!q->y || !q->state_out) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  ScanParams p = scan_params(q);
  // states, A, B and C in aligned groups of four
  const int four = q->states % 4 == 0 && reinterpret_cast<uintptr_t>(q->state_out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(q->a) % 16 == 0 && fours(q->b, q->dtype, {q->b_sb, q->b_sg}) &&
                   fours(q->c, q->dtype, {q->c_sb, q->c_sg});
  const int64_t blocks = ceil_div(q->batch * q->channels, 32);
  if (blocks > INT_MAX) return fail(XE_ERR_NOT_SUPPORTED, "%s: a size is above its limit", what);
  by_type(q->dtype, [&](auto t) {
    xe::scan::selective_scan_step_kernel<decltype(t)><<<(unsigned)blocks, 128, 0, as_stream(stream)>>>(p, four);
  });
  return launched(what);
}

size_t xe_selective_scan_backward_workspace_size(int64_t batch, int64_t length, int64_t channels, int64_t states,
                                                 int64_t groups) {
  if (batch <= 0 || length < 0 || channels <= 0 || states < 1 || states > 64 || groups < 1 || channels % groups) return 0;
  const ScanPlan plan = scan_plan(batch, length, channels, groups);
  return scan_segment_bytes(plan, batch, channels, states) +
         padded((size_t)(plan.channel_blocks * batch * length * 2 * 16 * scan_blocks(states)) * 4) +
         padded((size_t)(plan.segments * batch * channels * states) * 4) + padded((size_t)(plan.segments * batch * 2 * channels) * 4);
}

xe_status xe_selective_scan_backward(const xe_selective_scan_args* q, const xe_selective_scan_grads* g, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* what = "xe_selective_scan_backward";
  if (xe_status s = check_scan(what, q, false)) return s;
  if (!g) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null arguments", what);
  if (q->channels == 0) return XE_OK;
  if (!g->da || !g->dd || (q->batch * q->length > 0 && (!g->dy || !g->dx || !g->ddelta || !g->db || !g->dc ||
                                                        (q->z && !g->dz) || !q->checkpoints)))
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (q->batch == 0) return fail(XE_ERR_INVALID_ARGUMENT, "%s: an empty batch has no gradients", what);
  if (xe_status s = check_workspace(
          what, workspace, workspace_bytes,
          xe_selective_scan_backward_workspace_size(q->batch, q->length, q->channels, q->states, q->groups)))
    return s;
  const ScanPlan plan = scan_plan(q->batch, q->length, q->channels, q->groups);
  ScanParams p = scan_params(q);
  scan_segments(p, plan, workspace);
  p.dy = g->dy, p.dy_sb = g->dy_sb, p.dy_st = g->dy_st, p.dstate_out = g->dstate_out, p.dstate = g->dstate;
  p.dx = g->dx, p.ddelta = g->ddelta, p.dz = g->dz;
  const int64_t each = q->channels / q->groups;
  p.vec = (p.vec & ~8) | (fours(g->dy, q->dtype, {g->dy_sb, g->dy_st, each}) ? 64 : 0) |
          (fours(g->dx, q->dtype, {q->channels, each}) && fours(g->ddelta, q->dtype, {}) && fours(g->dz, q->dtype, {}) ? 8 : 0);
  const int blocks = scan_blocks(q->states);
  char* at = static_cast<char*>(workspace) + scan_segment_bytes(plan, q->batch, q->channels, q->states);
  p.dbc = reinterpret_cast<float*>(at);
  at += padded((size_t)(plan.channel_blocks * q->batch * q->length * 2 * 16 * blocks) * 4);
  p.da = reinterpret_cast<float*>(at);
  at += padded((size_t)(plan.segments * q->batch * q->channels * q->states) * 4);
  p.dd = reinterpret_cast<float*>(at);
  cudaStream_t st = as_stream(stream);
  if (p.segments > 1) {
    if (xe_status s = launch_scan<xe::scan::kAdjoint>(p, plan, q->dtype, st)) return s;
    if (xe_status s = join_scan<true>(p, st)) return s;
  }
  xe_status status = XE_OK;
  by_type(q->dtype, [&](auto t) {
    using T = decltype(t);
    status = blocks == 1   ? launch_scan_backward<T, 1>(p, plan, st)
             : blocks == 2 ? launch_scan_backward<T, 2>(p, plan, st)
                           : launch_scan_backward<T, 4>(p, plan, st);
    const int64_t tokens = q->batch * q->length;
    const int64_t total = tokens * q->groups * 2 * 16 * blocks;
    if (status == XE_OK && total > 0) {
      xe::scan::selective_scan_dbc_kernel<T><<<(unsigned)ceil_div(total, 256), 256, 0, st>>>(
          p.dbc, static_cast<T*>(g->db), static_cast<T*>(g->dc), tokens, (int)q->groups,
          (int)(plan.channel_blocks / q->groups), (int)q->states, 16 * blocks);
      status = launched(what);
    }
  });
  if (status != XE_OK) return status;
  const int64_t parts = plan.segments * q->batch;
  if (xe_status s = sum_rows(p.da, parts, q->channels * q->states, g->da, st)) return s;
  return sum_rows(p.dd, parts, 2 * q->channels, g->dd, st);
}

}  // extern "C"

// ------------------------------------------------------------------ norm

namespace {

struct NormShape {
  int groups, warps_per_row, threads, rows_per_block;
};

// Groups of eight elements per thread and warps per row.  One group needs the fewest registers, so that
// many rows are in flight; few rows want the most threads on each.
bool norm_shape(int64_t columns, bool backward, int64_t rows, NormShape& s) {
  const int64_t groups = ceil_div(columns, 8);
  const int64_t one = backward ? 512 : rows <= 148 ? 1024 : 256;
  if (groups <= one)
    s.groups = 1;
  else if (groups <= 1024)
    s.groups = 2;
  else if (groups <= 2048)
    s.groups = 4;
  else if (groups <= 8192)
    s.groups = 8;
  else
    return false;
  s.warps_per_row = (int)ceil_div(groups, 32 * s.groups);
  s.rows_per_block = std::max(1, 8 / s.warps_per_row);
  s.threads = s.warps_per_row * 32 * s.rows_per_block;
  return true;
}

// Prepares a persistent kernel and gives its number of blocks: what the device holds at once, or fewer.
// `Tag`: a type of its own for each kernel, since kernels of one signature share a pointer type.
template <typename Tag, typename K>
int64_t persistent_blocks(K kernel, int threads, int bytes, int64_t wanted) {
  static std::atomic<int> known[32][33];  // by device and warps
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& at = known[dev & 31][threads / 32];
  int each = at.load();
  if (each == 0) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, threads, bytes) != cudaSuccess || each < 1) each = 1;
    at.store(each);
  }
  return std::min<int64_t>(wanted, 148ll * each);
}

template <typename F>
void by_groups(int groups, F f) {
  switch (groups) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    default: f(std::integral_constant<int, 8>{});
  }
}

// The residual stream is of the input's type or float32.
template <typename F>
void by_types(int32_t dtype, int32_t residual_dtype, F f) {
  by_type(dtype, [&](auto t) {
    if (residual_dtype == XE_F32)
      f(t, float{});
    else
      f(t, t);
  });
}

xe_status check_norm(const char* what, int64_t rows, int64_t columns, int32_t dtype, int32_t residual_dtype,
                     int32_t weight_dtype) {
  if (!is_float(dtype)) return fail(XE_ERR_NOT_SUPPORTED, "%s: element type %d", what, dtype);
  if (residual_dtype != dtype && residual_dtype != XE_F32)
    return fail(XE_ERR_NOT_SUPPORTED, "%s: residual type %d with elements of type %d", what, residual_dtype, dtype);
  if (weight_dtype != dtype && weight_dtype != XE_F32)
    return fail(XE_ERR_NOT_SUPPORTED, "%s: weight type %d with elements of type %d", what, weight_dtype, dtype);
  if (rows < 0 || columns < 1) return fail(XE_ERR_INVALID_ARGUMENT, "%s: negative rows, or no columns", what);
  if (columns > 65536) return fail(XE_ERR_NOT_SUPPORTED, "%s: %lld columns above 65536", what, (long long)columns);
  return XE_OK;
}

// The most blocks of the backward kernel (the workspace is planned for them).
int64_t norm_backward_blocks(int64_t rows, const NormShape& s) {
  return std::min<int64_t>(ceil_div(rows, s.rows_per_block), 148ll * std::max(1, 1024 / s.threads));
}

}  // namespace

extern "C" {

xe_status xe_rms_norm(const void* x, int64_t x_row, const void* residual, int64_t residual_row, const void* weight, void* y,
                      void* sum, float* scale, int64_t rows, int64_t columns, float eps, int32_t dtype,
                      int32_t residual_dtype, int32_t weight_dtype, int32_t out_dtype, void* stream) {
  const char* what = "xe_rms_norm";
  if (xe_status s = check_norm(what, rows, columns, dtype, residual_dtype, weight_dtype)) return s;
  if (rows > 0 && (!x || !y || (residual && !sum))) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  const bool quantize = out_dtype == XE_E4M3 || out_dtype == XE_I8;
  if (!quantize && out_dtype != dtype) return fail(XE_ERR_NOT_SUPPORTED, "%s: output type %d", what, out_dtype);
  if (quantize && rows > 0 && !scale) return fail(XE_ERR_INVALID_ARGUMENT, "%s: 8-bit outputs need scales", what);
  if (rows == 0) return XE_OK;
  NormShape shape;
  if (!norm_shape(columns, false, rows, shape)) return fail(XE_ERR_NOT_SUPPORTED, "%s: too many columns", what);
  xe::norm::Params p{};
  p.x = x, p.residual = residual, p.weight = weight, p.y = y, p.sum = sum, p.scale = scale;
  p.x_row = x_row, p.r_row = residual_row, p.rows = rows, p.columns = (int)columns, p.eps = eps;
  p.quantize = quantize ? out_dtype : 0;
  p.weight_f32 = weight_dtype == XE_F32;
  const bool vec = vectors(x, dtype, {x_row, columns}) && vectors(residual, residual_dtype, {residual_row}) &&
                   vectors(sum, residual_dtype, {columns}) && vectors(weight, weight_dtype, {}) && vectors(y, dtype, {}) &&
                   columns % 8 == 0;
  // every tensor's row r starts r * columns elements past a boundary, modulo a vector
  auto base = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 32 == 0; };
  const bool shifted = !vec && x_row % 8 == columns % 8 && (!residual || residual_row % 8 == columns % 8) && base(x) &&
                       base(residual) && base(sum) && base(y) && columns >= 64 && columns <= 65528;
  if (shifted && !norm_shape(columns + 7, false, rows, shape)) return fail(XE_ERR_NOT_SUPPORTED, "%s: too many columns", what);
  by_types(dtype, residual_dtype, [&](auto t, auto r) {
    by_groups(shape.groups, [&](auto g) {
      auto go = [&](auto v) {
        auto kernel = xe::norm::rms_norm_kernel<decltype(t), decltype(r), decltype(g)::value, decltype(v)::value>;
        struct Tag {};
        using T = decltype(t);
        using R = decltype(r);
        constexpr int kGroups = decltype(g)::value;
        const int bytes = decltype(v)::value == xe::norm::kAligned ? xe::norm::kForwardStages<T, R, kGroups> * shape.threads * xe::norm::kForwardBytes<T, R, kGroups> : 0;
        const int64_t blocks = persistent_blocks<Tag>(kernel, shape.threads, bytes, ceil_div(rows, shape.rows_per_block));
        kernel<<<(unsigned)blocks, shape.threads, bytes, as_stream(stream)>>>(p, shape.warps_per_row);
      };
      using xe::norm::Rows;
      if (vec)
        go(std::integral_constant<Rows, xe::norm::kAligned>{});
      else if (shifted)
        go(std::integral_constant<Rows, xe::norm::kShifted>{});
      else
        go(std::integral_constant<Rows, xe::norm::kAnyhow>{});
    });
  });
  return launched(what);
}

size_t xe_rms_norm_backward_workspace_size(int64_t rows, int64_t columns) {
  NormShape shape;
  if (rows <= 0 || columns < 1 || !norm_shape(columns, true, rows, shape)) return 0;
  return padded((size_t)(norm_backward_blocks(rows, shape) * shape.rows_per_block * columns) * 4);
}

xe_status xe_rms_norm_backward(const void* sum, int64_t sum_row, const void* addend, int64_t addend_row, const void* weight, const void* dy, int64_t dy_row,
                               const void* dsum, int64_t dsum_row, void* dx, float* dweight, int64_t rows,
                               int64_t columns, float eps, int32_t dtype, int32_t residual_dtype, int32_t weight_dtype,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "xe_rms_norm_backward";
  if (xe_status s = check_norm(what, rows, columns, dtype, residual_dtype, weight_dtype)) return s;
  if (!sum || !dy || !dx) return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (rows == 0) return fail(XE_ERR_INVALID_ARGUMENT, "%s: no rows, no gradients", what);
  if (xe_status s = check_workspace(what, workspace, workspace_bytes,
                                    dweight ? xe_rms_norm_backward_workspace_size(rows, columns) : 0))
    return s;
  NormShape shape;
  if (!norm_shape(columns, true, rows, shape)) return fail(XE_ERR_NOT_SUPPORTED, "%s: too many columns", what);
  int64_t blocks = norm_backward_blocks(rows, shape);
  xe::norm::BackwardParams p{};
  p.sum = sum, p.addend = addend, p.a_row = addend_row, p.weight = weight, p.dy = dy, p.dsum = dsum, p.dx = dx;
  p.partial = dweight ? static_cast<float*>(workspace) : nullptr;
  p.s_row = sum_row, p.dy_row = dy_row, p.dsum_row = dsum_row;
  p.rows = rows, p.columns = (int)columns, p.eps = eps, p.weight_f32 = weight_dtype == XE_F32;
  const bool vec = vectors(sum, residual_dtype, {sum_row, columns}) && vectors(addend, dtype, {addend_row}) && vectors(dy, dtype, {dy_row}) &&
                   vectors(dsum, residual_dtype, {dsum_row}) && vectors(weight, weight_dtype, {}) &&
                   vectors(dx, residual_dtype, {}) && columns % 8 == 0;
  by_types(dtype, residual_dtype, [&](auto t, auto r) {
    by_groups(shape.groups, [&](auto g) {
      auto go = [&](auto v) {
        auto kernel = xe::norm::rms_norm_backward_kernel<decltype(t), decltype(r), decltype(g)::value, decltype(v)::value>;
        struct Tag {};
        using T = decltype(t);
        using R = decltype(r);
        constexpr int kGroups = decltype(g)::value;
        const int bytes = decltype(v)::value ? xe::norm::kBackwardStages<T, R, kGroups> * shape.threads * xe::norm::kBackwardBytes<T, R, kGroups> : 0;
        blocks = persistent_blocks<Tag>(kernel, shape.threads, bytes, blocks);
        kernel<<<(unsigned)blocks, shape.threads, bytes, as_stream(stream)>>>(p, shape.warps_per_row);
      };
      if (vec)
        go(std::true_type{});
      else
        go(std::false_type{});
    });
  });
  if (xe_status s = launched(what)) return s;
  if (!dweight) return XE_OK;
  return sum_rows(p.partial, blocks * shape.rows_per_block, columns, dweight, as_stream(stream));
}

}  // extern "C"

// ------------------------------------------------------------------ 4-bit weights

namespace {

struct Int4Plan {
  int tokens, tiles;  // tokens of a block, and their columns in eights
  int parts, part, runs, run, pitch;
  int bytes, blocks;  // shared memory; blocks in x
  int each;           // blocks to a multiprocessor
};

// How the work is cut: k into the parts that fit a block's shared memory, and these into runs, so that the
// device's warps get equally many stages each.  A unit of work costs its stages and about two more for its
// start and its sums.
Int4Plan int4_plan(int64_t rows, int64_t inputs, int64_t outputs, int pieces) {
  using namespace xe::int4;
  Int4Plan q;
  q.tokens = (int)std::min<int64_t>(rows, 64 / pieces);
  const int columns = q.tokens * pieces;
  q.tiles = columns <= 8 ? 1 : columns <= 16 ? 2 : columns <= 32 ? 4 : 8;
  constexpr int kRing = kWarps * kStages * kStageBytes;
  const int64_t stages = ceil_div(inputs, kStageK), rows16 = ceil_div(outputs, 16);
  // three blocks to a multiprocessor, two, or one, as the columns (and with them the registers) grow; fewer too
  // where there is little work and their larger share of the memory holds all of k
  int each = q.tiles <= 2 ? 3 : q.tiles == 4 ? 2 : 1;
  const int sums = kWarps * 16 * (q.tiles * 8 + 1) * 4;
  auto fit = [&](int blocks, int beside) {
    const int budget = 225 * 1024 / blocks - 1024 - kRing - kZeroBytes - beside;
    return std::max<int64_t>(1, (budget / (columns * 2) - 32) / kStageK);
  };
  if (rows16 * stages <= 148 * kWarps * 4)
    while (each > 1 && fit(each, sums) < stages) --each;
  q.each = each;
  q.parts = fit(each, sums) >= stages ? 1 : (int)std::max<int64_t>(2, ceil_div(stages, fit(each, 0)));
  q.part = (int)ceil_div(stages, q.parts);
  q.parts = (int)ceil_div(stages, q.part);
  q.pitch = q.part * kStageK + 32;  // bytes: 64 past a multiple of 128, two columns' reads in different banks
  q.bytes = kRing + kZeroBytes + columns * q.pitch * 2 + (q.parts == 1 ? sums : 0);
  const int64_t blocks = ceil_div(rows, q.tokens);  // in y
  const int64_t workers = std::max<int64_t>(1, 148 * each / (q.parts * blocks));
  int64_t best = INT64_MAX;
  q.runs = 1, q.run = q.part;
  for (int64_t runs = 1; runs <= 16 && runs <= std::max(q.part, kWarps); ++runs) {
    const int64_t run = ceil_div(q.part, runs);
    if (q.parts == 1 ? (runs & (runs - 1)) != 0 || runs > kWarps : ceil_div(q.part, run) != runs) continue;
    const int64_t cost = ceil_div(rows16 * runs, workers * kWarps) * (run + 2);
    if (cost < best) best = cost, q.runs = (int)runs, q.run = (int)run;
  }
  q.blocks = (int)(q.parts * std::min<int64_t>(workers, ceil_div(rows16 * q.runs, kWarps)));
  return q;
}

size_t int4_sums(const Int4Plan& plan, int64_t rows, int64_t outputs, int pieces) {
  return plan.parts == 1 ? 0 : padded((size_t)((int64_t)plan.parts * plan.runs * rows * pieces * outputs) * 4);
}

// Rows of one launch.  Where k is cut into parts, their float32 sums are `parts * runs` times the result (6.4 GB for 16384
// bf16 rows of 8192 -> 16384); many rows go in slices one after another, whose sums share a workspace of at most
// kInt4Sums, and a slice's blocks fill the device a whole number of times (16384 bf16 rows of 4096 -> 8192: 3.2 GB and
// 4.95 ms at once, 4.65 ms in slices; in slices of half the size 5.3 ms).  A grid has at most 65535 rows.
constexpr int64_t kInt4Sums = 512 << 20;
int64_t int4_slice(int64_t rows, int64_t inputs, int64_t outputs, int pieces) {
  const int64_t tokens = 64 / pieces;
  int64_t slice = std::min(rows, 65535 / tokens * tokens);
  while (slice > tokens) {
    const Int4Plan plan = int4_plan(slice, inputs, outputs, pieces);
    const int64_t need = (int64_t)int4_sums(plan, slice, outputs, pieces);
    if (need <= kInt4Sums) break;
    int64_t blocks = std::max<int64_t>(1, (int64_t)((double)slice * kInt4Sums / need) / tokens);
    const int64_t turn = std::max(1, 148 * plan.each / plan.parts);
    if (blocks > turn) blocks = blocks / turn * turn;
    slice = std::min(blocks * tokens, slice - 1);
  }
  return slice;
}

template <typename X, int kTiles, int kRun>
xe_status launch_int4(const xe::int4::Params& p, const Int4Plan& plan, cudaStream_t stream) {
  using namespace xe::int4;
  static std::atomic<uint32_t> done{0};
  auto kernel = int4_linear_kernel<X, kTiles, kRun>;
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(done.load() >> (dev & 31) & 1u)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return fail(XE_ERR_CUDA, "xe_int4_linear: %s", cudaGetErrorString(e));
    done.fetch_or(1u << (dev & 31));
  }
  const dim3 grid((unsigned)plan.blocks, (unsigned)ceil_div(p.rows, p.tokens));
  kernel<<<grid, kWarps * 32, plan.bytes, stream>>>(p);
  if (xe_status s = launched("xe_int4_linear")) return s;
  if (!p.sums) return XE_OK;
  // the second kernel's blocks may start while the first one ends; they wait for its results themselves
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)ceil_div(p.outputs, 256), (unsigned)p.rows);
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &early;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, int4_sum_kernel, p, plan.parts * plan.runs);
  if (e != cudaSuccess) return fail(XE_ERR_CUDA, "xe_int4_linear: %s", cudaGetErrorString(e));
  return launched("xe_int4_linear");
}

template <typename X>
xe_status run_int4(const xe::int4::Params& p, const Int4Plan& plan, cudaStream_t stream) {
  const int units = p.group / 32;
  auto go = [&](auto tiles) {
    constexpr int n = decltype(tiles)::value;
    return units % 4 == 0   ? launch_int4<X, n, 4>(p, plan, stream)
           : units % 2 == 0 ? launch_int4<X, n, 2>(p, plan, stream)
                            : launch_int4<X, n, 1>(p, plan, stream);
  };
  switch (plan.tiles) {
    case 1: return go(std::integral_constant<int, 1>{});
    case 2: return go(std::integral_constant<int, 2>{});
    case 4: return go(std::integral_constant<int, 4>{});
    default: return go(std::integral_constant<int, 8>{});
  }
}

}  // namespace

extern "C" {

size_t xe_int4_linear_workspace_size(int64_t rows, int64_t inputs, int64_t outputs, int32_t x_dtype) {
  if (rows <= 0 || inputs < 1 || outputs <= 0 || inputs > 1 << 20) return 0;
  const int pieces = x_dtype == XE_F32 ? 3 : 1;
  const int64_t slice = int4_slice(rows, inputs, outputs, pieces), rest = rows % slice;
  const size_t need = int4_sums(int4_plan(slice, inputs, outputs, pieces), slice, outputs, pieces);
  return rest == 0 ? need : std::max(need, int4_sums(int4_plan(rest, inputs, outputs, pieces), rest, outputs, pieces));
}

xe_status xe_int4_linear(const void* x, int64_t x_row, const float* x_scale, const void* packed, int64_t packed_row,
                         const void* scales, const void* zeros, void* y, int64_t rows, int64_t inputs, int64_t outputs,
                         int64_t group, int32_t x_dtype, int32_t scale_dtype, int32_t y_dtype, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const char* what = "xe_int4_linear";
  if (rows * outputs != 0 && (!x || !packed || !scales || !y))
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!is_float(x_dtype) && x_dtype != XE_E4M3 && x_dtype != XE_I8)
    return fail(XE_ERR_NOT_SUPPORTED, "%s: activations of type %d", what, x_dtype);
  if (!is_float(scale_dtype) || !is_float(y_dtype))
    return fail(XE_ERR_NOT_SUPPORTED, "%s: scales of type %d, result of type %d", what, scale_dtype, y_dtype);
  if (rows < 0 || outputs < 0 || inputs < 1 || group < 1 || inputs % group)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: %lld inputs in groups of %lld", what, (long long)inputs, (long long)group);
  if (group % 32) return fail(XE_ERR_NOT_SUPPORTED, "%s: groups of %lld, not a multiple of 32", what, (long long)group);
  if (reinterpret_cast<uintptr_t>(packed) % 16 || packed_row % 16)
    return fail(XE_ERR_INVALID_ARGUMENT, "%s: rows of codes must start on 16-byte boundaries", what);
  if (rows > INT_MAX / 4 || inputs > 1 << 20 || outputs > INT_MAX / 64)
    return fail(XE_ERR_NOT_SUPPORTED, "%s: a size is above its limit", what);
  if (rows == 0 || outputs == 0) return XE_OK;
  xe::int4::Params p{};
  p.packed = static_cast<const uint8_t*>(packed), p.scales = scales, p.zeros = static_cast<const uint8_t*>(zeros);
  p.x_row = x_row, p.packed_row = packed_row;
  p.inputs = (int)inputs, p.outputs = (int)outputs, p.group = (int)group;
  p.scale_dtype = scale_dtype, p.y_dtype = y_dtype;
  p.pieces = x_dtype == XE_F32 ? 3 : 1;
  p.group_magic = group == 32 ? 0u : (uint32_t)((1ull << 32) / (uint64_t)(group / 32)) + 1u;
  p.x_vec = aligned(size_of(x_dtype) == 1 ? 8 : 16, x, x_dtype, {x_row});
  if (xe_status s = check_workspace(what, workspace, workspace_bytes, xe_int4_linear_workspace_size(rows, inputs, outputs, x_dtype)))
    return s;
  cudaStream_t st = as_stream(stream);
  const int64_t slice = int4_slice(rows, inputs, outputs, p.pieces);
  for (int64_t m = 0; m < rows; m += slice) {
    p.rows = (int)std::min(slice, rows - m);
    const Int4Plan plan = int4_plan(p.rows, inputs, outputs, p.pieces);
    p.x = static_cast<const char*>(x) + m * x_row * size_of(x_dtype);
    p.x_scale = x_scale ? x_scale + m : nullptr;
    p.y = static_cast<char*>(y) + m * outputs * size_of(y_dtype);
    p.sums = plan.parts > 1 ? static_cast<float*>(workspace) : nullptr;
    p.tokens = plan.tokens, p.parts = plan.parts, p.part = plan.part, p.runs = plan.runs, p.run = plan.run, p.pitch = plan.pitch;
    xe_status status = XE_OK;
    switch (x_dtype) {
      case XE_F32: status = run_int4<float>(p, plan, st); break;
      case XE_BF16: status = run_int4<__nv_bfloat16>(p, plan, st); break;
      case XE_F16: status = run_int4<__half>(p, plan, st); break;
      case XE_E4M3: status = run_int4<__nv_fp8_e4m3>(p, plan, st); break;
      default: status = run_int4<int8_t>(p, plan, st);
    }
    if (status != XE_OK) return status;
  }
  return XE_OK;
}

}  // extern "C"
