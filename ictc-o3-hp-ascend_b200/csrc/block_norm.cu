// Entry points of the block norms: argument checks, launch shapes, weight-gradient sums.
#include "block_norm.cuh"

namespace ictc {
namespace block_norm {
namespace {

// The status word of callers without one of their own, per device.  The library's memory and not an allocation: it is
// there, zeroed, before any stream captures, and graphs may keep its address.
__device__ int own_status;

// Weight gradients from the blocks' sums: one warp per (degree, channel) column.
__global__ void __launch_bounds__(256) weight_sum_kernel(const float* __restrict__ partial, int blocks, int columns,
                                                         const float* __restrict__ post,
                                                         const float* __restrict__ scale, float* grad_post,
                                                         float* grad_scale, float* grad_pre) {
  const int lane = threadIdx.x & 31, column = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (column >= columns) return;
  float w = 0.f, b = 0.f;
  for (int k = lane; k < blocks; k += 32) {
    w += partial[(int64_t)k * 2 * columns + column];
    b += partial[(int64_t)k * 2 * columns + columns + column];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    w += __shfl_xor_sync(0xffffffffu, w, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (lane == 0) {
    if (grad_post) grad_post[column] = w * (scale ? scale[column] : 1.f);
    if (grad_scale) grad_scale[column] = w * (post ? post[column] : 1.f);
    if (grad_pre) grad_pre[column] = b;
  }
}

// Lanes, warps, rows per tile, copy stages and groups per block that fit shared memory, and
// the places of the staged tensors (`there`: bit per slot).
bool shape_of(int C, int L, int mode, unsigned there, bool sums, int64_t rows, int sms, Shape* s, BlockArgs* a,
              int* shared_bytes) {
  const int N = L + 1, most_row = max_row_warps(mode, L);
  const int64_t W = (int64_t)C * N * N;
  if (W > (1 << 16)) return false;
  s->hold = C <= 32 * most_row;
  s->warps = 1;
  s->lanes = 1;
  if (C <= 32) {
    while (s->lanes < C) s->lanes *= 2;
  } else {
    s->warps = (C + 31) / 32 < most_row ? (C + 31) / 32 : most_row;
    s->lanes = 32 * s->warps;
  }
  const int beside = 32 * s->warps / s->lanes;
  s->per = beside * rows_per_lane(mode, L, s->hold);
  int64_t stage = 0;
  for (int k = 0; k < kSlots; ++k) {
    a->at[k] = -1;
    if (!(there >> k & 1u) || (!s->hold && (k == kGate || k == kGateDot))) continue;
    a->at[k] = (int)stage;
    const int64_t wd = k < kGate ? W : k < kR1 ? (int64_t)N * C : 4;
    stage += (s->per * wd + 3) & ~3ll;
  }
  const int64_t fixed = 2 * s->warps * kScratch + kBarrierFloats + (sums && !s->hold ? (2 * N * C + 3) & ~3 : 0);
  int most = max_warps(mode, L) / s->warps;
  if (s->warps > 1 && most > 15) most = 15;      // named barriers
  const int64_t tiles = (rows + s->per - 1) / s->per, wanted = (tiles + sms - 1) / sms;
  if (wanted < most) most = (int)(wanted > 0 ? wanted : 1);
  for (s->stages = 4; s->stages >= 1; --s->stages) {
    const int64_t bytes = 4 * (s->stages * stage + fixed);
    int64_t groups = (s->stages > 1 ? shared_budget(mode) : kSharedLimit) / bytes;
    if (groups > most) groups = most;
    // fewer stages where they make room for more groups, two where two fit
    if (groups < 1 || (groups < most && s->stages > 2)) {
      if (s->stages > 1) continue;
      return false;
    }
    s->groups = (int)groups;
    int64_t total = groups * bytes;
    if (sums && s->hold) {
      const int64_t end = 4 * groups * beside * 2 * N * C;      // the sums at the end lie over the stages
      if (end > kSharedLimit) return false;
      if (end > total) total = end;
    }
    *shared_bytes = (int)total;
    a->stage_floats = (int)stage;
    a->group_floats = (int)(s->stages * stage + fixed);
    return true;
  }
  return false;
}

std::atomic<uint64_t> wait_limit{kWaitNs};

int invalid(const char* what) {
  ictc_set_error(what, "");
  return ICTC_ERR_INVALID;
}

int checked(cudaError_t err) {
  if (err == cudaSuccess) return ICTC_OK;
  ictc_set_error("ictc_block: %s", cudaGetErrorString(err));
  return ICTC_ERR_CUDA;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int sm_count() {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return sms > 0 ? sms : 1;
}

// All rows through one mode; the blocks that left weight-gradient sums go to *blocks.
int run(int mode, BlockArgs& a, int lmax, int layout, bool branch, int* blocks, cudaStream_t stream) {
  const int C = a.channels, N = lmax + 1, sms = sm_count();
  unsigned there = 0;
  for (int k = 0; k < kSlots; ++k)
    if (a.in[k] || (k < 6 && a.out[k])) there |= 1u << k;
  // places that only the work itself needs: T behind p (or q), tau behind al
  if (mode != kForward && branch) there |= 1u << kP;
  if (mode == kSecond) there |= 1u << kAl;
  Shape s{};
  int bytes = 0;
  if (!shape_of(C, lmax, mode, there, a.partial != nullptr, a.rows, sms, &s, &a, &bytes)) {
    ictc_set_error("ictc_block: rows of this width do not fit shared memory%s", "");
    return ICTC_ERR_UNSUPPORTED;
  }
  a.wait_ns = wait_limit.load(std::memory_order_relaxed);
  a.wide = 0;
  a.row_bytes = 0;
  s.bulk = s.hold && s.stages > 1;
  for (int k = 0; k < kSlots; ++k) {
    const int64_t wd = k < kGate ? (int64_t)C * N * N : k < kR1 ? (int64_t)N * C : 4;
    if (a.in[k]) {
      a.row_bytes += (int)(4 * wd);
      if (wd % 4 || !aligned(a.in[k])) s.bulk = 0;
    }
    if (k < 6 && a.out[k] && (wd % 4 || !aligned(a.out[k]))) s.bulk = 0;
    if (s.per * wd % 4) continue;
    if (aligned(a.in[k])) a.wide |= 1u << k;
    if (k < 6 && aligned(a.out[k])) a.wide |= 1u << (16 + k);
  }
  for (int l = 0; l < N; ++l) a.inv[l] = (float)(1.0 / ((double)C * (2 * l + 1)));
  a.lanes = s.lanes;
  a.warps = s.warps;
  a.per = s.per;
  a.stages = s.stages;
  const int64_t tiles = (a.rows + s.per - 1) / s.per, want = (tiles + s.groups - 1) / s.groups;
  const int grid = (int)(want < sms ? want : sms);
  if (blocks) *blocks = grid;
  const cudaError_t err = mode == kForward    ? launch_forward(a, s, grid, bytes, lmax, layout, branch, stream)
                          : mode == kBackward ? launch_backward(a, s, grid, bytes, lmax, layout, branch, stream)
                                              : launch_second(a, s, grid, bytes, lmax, layout, branch, stream);
  return checked(err);
}

int weight_sums(const BlockArgs& a, int lmax, int blocks, float* grad_post, float* grad_scale, float* grad_pre,
                cudaStream_t stream) {
  const int columns = (lmax + 1) * a.channels;
  weight_sum_kernel<<<(columns + 7) / 8, 256, 0, stream>>>(a.partial, blocks, columns, a.post, a.scale, grad_post,
                                                           grad_scale, grad_pre);
  return checked(cudaGetLastError());
}

bool bad_shape(int64_t rows, int channels, int lmax, int layout, float eps) {
  return rows < 0 || channels < 1 || lmax < 0 || lmax > kMaxL || (layout != kIrMul && layout != kMulIr) ||
         !(eps > 0.f);
}

}  // namespace
}  // namespace block_norm
}  // namespace ictc

using namespace ictc;
using namespace ictc::block_norm;

extern "C" int ictc_block_status_word(int** word) {
  if (!word) return invalid("ictc_block_status_word: invalid argument%s");
  return checked(cudaGetSymbolAddress(reinterpret_cast<void**>(word), own_status));
}

extern "C" int ictc_block_status(int reset, int* value, void* stream) {
  if (!value) return invalid("ictc_block_status: invalid argument%s");
  int* word = nullptr;
  if (int rc = ictc_block_status_word(&word)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (int rc = checked(cudaMemcpyAsync(value, word, sizeof(int), cudaMemcpyDeviceToHost, s))) return rc;
  if (reset)
    if (int rc = checked(cudaMemsetAsync(word, 0, sizeof(int), s))) return rc;
  return checked(cudaStreamSynchronize(s));
}

extern "C" int ictc_block_wait_limit(uint64_t nanoseconds) {
  if (nanoseconds > kWaitNs) return invalid("ictc_block_wait_limit: at most two seconds%s");
  wait_limit.store(nanoseconds, std::memory_order_relaxed);
  return ICTC_OK;
}

extern "C" int64_t ictc_block_partial_floats(int channels, int lmax) {
  if (channels < 1 || lmax < 0 || lmax > kMaxL) return -1;
  return (int64_t)sm_count() * 2 * (lmax + 1) * channels;
}

extern "C" int ictc_block_supported(int channels, int lmax) {
  Shape s{};
  BlockArgs a{};
  int bytes = 0;
  return channels >= 1 && lmax >= 0 && lmax <= kMaxL &&
         shape_of(channels, lmax, kSecond, (1u << kSlots) - 1, true, 1, 1, &s, &a, &bytes);
}

extern "C" int ictc_block_forward(const float* stream_in, const float* branch, const float* gate, const float* post,
                                  const float* scale, const float* pre, int norm, int64_t rows, int channels,
                                  int lmax, int layout, float eps, float* stream_out, float* normed, float* r1,
                                  float* r2, int* status, void* stream) {
  if (bad_shape(rows, channels, lmax, layout, eps) ||
      (rows > 0 && (!stream_in || (branch ? !stream_out : !norm) || (norm && !normed) || !status)))
    return invalid("ictc_block_forward: invalid argument%s");
  if (rows == 0) return ICTC_OK;
  BlockArgs a{};
  a.status = status;
  a.in[kY] = branch;
  a.in[kH] = stream_in;
  a.out[kY] = norm ? normed : nullptr;      // u leaves from y's place
  a.out[kH] = branch ? stream_out : nullptr;
  a.in[kGate] = branch ? gate : nullptr;
  a.post = post;
  a.scale = scale;
  a.pre = pre;
  a.r1_out = branch ? r1 : nullptr;
  a.r2_out = r2;
  a.rows = rows;
  a.channels = channels;
  a.norm = norm;
  a.eps = eps;
  return run(kForward, a, lmax, layout, branch != nullptr, nullptr, (cudaStream_t)stream);
}

extern "C" int ictc_block_backward(const float* stream_out, const float* branch, const float* gate, const float* post,
                                   const float* scale, const float* pre, const float* r1, const float* r2,
                                   const float* p, const float* q, int64_t rows, int channels, int lmax, int layout,
                                   float* grad_stream, float* grad_branch, float* grad_gate, float* grad_post,
                                   float* grad_scale, float* grad_pre, float* partial, int* status, void* stream) {
  const bool norm = q != nullptr, sums = grad_post || grad_scale || grad_pre;
  if (bad_shape(rows, channels, lmax, layout, 1.f) || (sums && !partial) ||
      (rows > 0 && ((norm && (!stream_out || !r2)) || (branch ? !r1 : !norm) || (!p && !q) ||
                    (grad_gate && (!gate || !branch)) || (grad_stream && !norm) || !status)))
    return invalid("ictc_block_backward: invalid argument%s");
  BlockArgs a{};
  a.status = status;
  a.post = post;
  a.scale = scale;
  a.partial = sums ? partial : nullptr;
  a.channels = channels;
  int blocks = 0;
  if (rows > 0) {
    a.in[kY] = branch;
    a.in[kH] = norm ? stream_out : nullptr;
    a.in[kP] = branch ? p : nullptr;
    a.in[kQ] = q;
    a.in[kGate] = branch ? gate : nullptr;
    a.in[kR1] = branch ? r1 : nullptr;
    a.in[kR2] = norm ? r2 : nullptr;
    a.out[kY] = branch ? grad_branch : nullptr;
    a.out[branch ? kP : kQ] = grad_stream;
    a.gate_out = grad_gate;
    a.pre = pre;
    a.rows = rows;
    a.norm = norm;
    if (int rc = run(kBackward, a, lmax, layout, branch != nullptr, &blocks, (cudaStream_t)stream)) return rc;
  }
  return sums ? weight_sums(a, lmax, blocks, grad_post, grad_scale, grad_pre, (cudaStream_t)stream) : ICTC_OK;
}

extern "C" int ictc_block_second(const float* stream_out, const float* branch, const float* gate, const float* post,
                                 const float* scale, const float* pre, const float* r1, const float* r2,
                                 const float* p, const float* q, const float* dot_stream, const float* dot_branch,
                                 const float* dot_gate, int64_t rows, int channels, int lmax, int layout,
                                 float* grad_stream, float* grad_branch, float* grad_gate, float* grad_post,
                                 float* grad_scale, float* grad_pre, float* grad_p, float* grad_q, float* partial,
                                 int* status, void* stream) {
  const bool norm = q != nullptr, sums = grad_post || grad_scale || grad_pre;
  if (bad_shape(rows, channels, lmax, layout, 1.f) || (sums && !partial) ||
      (rows > 0 && ((norm && (!stream_out || !r2)) || (branch ? !r1 : !norm) || (!p && !q) ||
                    ((grad_gate || dot_gate) && (!gate || !branch)) || ((grad_stream || grad_q) && !norm) || !status)))
    return invalid("ictc_block_second: invalid argument%s");
  BlockArgs a{};
  a.status = status;
  a.post = post;
  a.scale = scale;
  a.partial = sums ? partial : nullptr;
  a.channels = channels;
  int blocks = 0;
  if (rows > 0) {
    a.in[kY] = branch;
    a.in[kH] = norm ? stream_out : nullptr;
    a.in[kP] = branch ? p : nullptr;
    a.in[kQ] = q;
    a.in[kAl] = dot_stream;
    a.in[kBe] = branch ? dot_branch : nullptr;
    a.in[kGate] = branch ? gate : nullptr;
    a.in[kGateDot] = branch ? dot_gate : nullptr;
    a.in[kR1] = branch ? r1 : nullptr;
    a.in[kR2] = norm ? r2 : nullptr;
    a.out[kY] = branch ? grad_branch : nullptr;
    a.out[kH] = grad_stream;
    a.out[kQ] = grad_q;
    a.out[kAl] = branch ? grad_p : nullptr;
    a.gate_out = grad_gate;
    a.pre = pre;
    a.rows = rows;
    a.norm = norm;
    if (int rc = run(kSecond, a, lmax, layout, branch != nullptr, &blocks, (cudaStream_t)stream)) return rc;
  }
  return sums ? weight_sums(a, lmax, blocks, grad_post, grad_scale, grad_pre, (cudaStream_t)stream) : ICTC_OK;
}
