// AdamW over many tensors in one launch, with moments in 32 or in 8 bits.
//
// For a tensor whose step counter is t - 1 (g' = clip * g, all in FP32):
//   m = b1 m + (1 - b1) g'         v = b2 v + (1 - b2) g'^2
//   w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//   average = d average + (1 - d) w                                   (optional)
// clip = min(1, max_norm / (|g| + 1e-6)) comes from a first pass over the gradients
// (grad_norm_kernel) when clipping or skipping of non-finite steps is asked for.
//
// Work is cut into chunks of kChunk consecutive values of one tensor; a static device
// table gives each chunk's tensor, place and count, and the addresses of weights and
// gradients travel in the kernel's parameters (they may change from step to step).
// One block per chunk, eight values per thread.
//
// 8-bit moments: blocks of 256 values (one warp's share) have a power-of-two scale
// 2^(byte - 127), byte = exponent field of the block's largest magnitude + 1, limited to
// 1..253.  A code is the top of the FP32 pattern of |x| / scale:
//   m: sign, 4 exponent bits, 3 fraction bits    (code + 896) << 20, code 0 = zero
//   v: 5 exponent bits, 3 fraction bits          (code + 768) << 20, code 0 = zero
// so a stored m reaches down to 1.125 * 2^-15 and a stored v to 1.125 * 2^-31 of the scale
// (2^-15.5 in sqrt(v)).  Rounding is stochastic: with b2 = 0.999 a step moves v by
// 0.1%, far below half a code step (6%), and rounding to nearest would never move a
// stored value at all.  16 random bits each from Philox4x32-7 (Salmon, Moraes, Dror,
// Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011), counter (index of the four
// values, t), key = seed: the codes are a function of the inputs alone.  A positive v
// never rounds to zero (the weight's step divides by sqrt(v)).  A block whose new moments
// are not all finite is left as it was, its weights too: the codes hold no NaN.
// Every product of the moments is rounded by itself (no FMA contraction), so the codes
// do not depend on how the compiler pairs operations.
#include "ictc_cuda.h"

#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

void ictc_set_error(const char* fmt, const char* detail);

namespace ictc {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 2048;          // values per block: 8 per thread
constexpr int kQuads = 2;             // groups of 4 values per thread
constexpr int kBlockValues = 256;     // values that share a scale: 32 lanes x 8
constexpr int kNormBlocks = 1184;     // partial sums of the gradient norm at most
constexpr int kList = 240;            // tensors per launch: 16 B each, below 4 KB of parameters

static_assert(kChunk == kThreads * kQuads * 4 && kBlockValues == 32 * kQuads * 4, "a warp owns one scale block");

// Caller-owned device words, zeroed once.  The tickets count finished blocks and return
// to zero at the end of each launch.
struct Workspace {
  unsigned norm_ticket;
  unsigned step_ticket;
  float norm;   // |g| of the last step
  float clip;   // factor of the gradients
  int skip;     // 1: this step leaves everything as it was
  int pad;
  double partial[kNormBlocks];
};

struct Tensor {
  float* weight;
  const float* grad;   // null: the tensor is left out of this step
};

struct TensorList {
  Tensor t[kList];
};

struct Args {
  const int4* chunks;   // {tensor, values, first scale block, chunk of the tensor}
  int tensor0;          // the list's first tensor
  int tensors;
  int64_t chunk0;
  int64_t chunks_n;
  void* m;
  void* v;
  uint8_t* m_scale;
  uint8_t* v_scale;
  float* average;
  int64_t* steps;
  Workspace* ws;
  int use_norm;
  float b1, c1, b2, c2;      // betas and 1 - beta
  float eps, keep, avg, avg1;  // keep = 1 - lr wd
  double lr, log_b1, log_b2;
  uint32_t seed_lo, seed_hi;
};

__device__ __forceinline__ float4 load4(const float* p, int left, bool aligned) {
  if (left >= 4 && aligned) return *reinterpret_cast<const float4*>(p);
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (left > 0) r.x = p[0];
  if (left > 1) r.y = p[1];
  if (left > 2) r.z = p[2];
  if (left > 3) r.w = p[3];
  return r;
}

__device__ __forceinline__ void store4(float* p, const float (&x)[4], int left, bool aligned) {
  if (left >= 4 && aligned) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = x[i];
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Seven rounds of Philox4x32 (the fewest its authors report as passing their tests).
__device__ __forceinline__ uint4 philox7(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u;
    const uint64_t b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1, (uint32_t)a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t code, float scale) {
  const uint32_t low = SIGNED ? code & 127u : code;
  const float x = low ? __uint_as_float((low + (SIGNED ? 896u : 768u)) << 20) * scale : 0.f;
  return SIGNED && (code & 128u) ? -x : x;
}

template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float x, float inv_scale, uint32_t r16) {
  constexpr int base = SIGNED ? 896 : 768;
  constexpr float least = SIGNED ? 1.125f / 32768.f : 1.125f / 2147483648.f;
  const float a = fabsf(x) * inv_scale;
  uint32_t code;
  if (a < least) {
    code = SIGNED ? ((float)r16 < a * (65536.f / least) ? 1u : 0u) : (a > 0.f ? 1u : 0u);
  } else {
    code = ((__float_as_uint(a) + (r16 << 4)) >> 20) - base;
    code = min(code, SIGNED ? 127u : 255u);
  }
  return SIGNED && x < 0.f && code ? code | 128u : code;
}

// Exponent byte of a block from its largest magnitude's bits.
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
  const uint32_t e = (bits >> 23) + 1u;
  return e < 253u ? e : 253u;
}

// Sum over one block's threads in a fixed order, valid in thread 0.
__device__ __forceinline__ double block_sum(double x, double* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_down_sync(0xffffffffu, x, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < kThreads / 32; ++i) s += shared[i];
  return s;
}

// Squares of FP32 gradients are exact in FP64 and so is their sum to ~1e-16: the clip
// factor does not depend on the grid.  The last block of the last launch adds the
// partial sums up in order.
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ TensorList list, const Args a,
                                                             int slot0, int slots, int last_launch, float max_norm,
                                                             int clip, int skip_bad) {
  __shared__ double shared[kThreads / 32];
  __shared__ int last;
  double sum = 0.0;
  for (int64_t i = blockIdx.x; i < a.chunks_n; i += gridDim.x) {
    const int4 c = a.chunks[a.chunk0 + i];
    const float* g = list.t[c.x - a.tensor0].grad;
    if (g == nullptr) continue;
    g += (int64_t)c.w * kChunk;
    const bool al = aligned16(g);
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      const int at = (q * kThreads + threadIdx.x) * 4;
      const float4 x = load4(g + at, c.y - at, al);
      sum += (double)x.x * x.x;
      sum += (double)x.y * x.y;
      sum += (double)x.z * x.z;
      sum += (double)x.w * x.w;
    }
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) {
    a.ws->partial[slot0 + blockIdx.x] = sum;
    __threadfence();
    last = atomicAdd(&a.ws->norm_ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (last_launch) {
    sum = 0.0;
    for (int i = threadIdx.x; i < slots; i += kThreads) sum += __ldcg(&a.ws->partial[i]);
    sum = block_sum(sum, shared);
  }
  if (threadIdx.x == 0) {
    if (last_launch) {
      const float norm = (float)sqrt(sum);
      a.ws->norm = norm;
      a.ws->clip = clip ? fminf(__fmul_rn(__frcp_rn(__fadd_rn(norm, 1e-6f)), max_norm), 1.f) : 1.f;
      a.ws->skip = skip_bad && !isfinite(sum);
    }
    a.ws->norm_ticket = 0;
  }
}

template <int BITS, bool AVERAGE>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ TensorList list, const Args a) {
  __shared__ float s_size, s_rate;
  __shared__ int64_t s_t;
  __shared__ int s_last;
  const int4 c = a.chunks_n ? a.chunks[a.chunk0 + blockIdx.x] : make_int4(a.tensor0, 0, 0, 0);
  const Tensor tensor = list.t[c.x - a.tensor0];
  const bool skip = a.use_norm && a.ws->skip;
  const bool active = tensor.grad != nullptr && !skip;
  if (active) {
    if (threadIdx.x == 0) {
      const int64_t t = a.steps[c.x] + 1;
      s_t = t;
      s_size = (float)(a.lr / -expm1((double)t * a.log_b1));
      s_rate = (float)(1.0 / sqrt(-expm1((double)t * a.log_b2)));
    }
    float clip = 1.f;
    if (a.use_norm) clip = a.ws->clip;
    float* wp = tensor.weight + (int64_t)c.w * kChunk;
    const float* gp = tensor.grad + (int64_t)c.w * kChunk;
    const bool wal = aligned16(wp), gal = aligned16(gp);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int at0 = warp * kBlockValues + lane * 4;     // quads at at0 and at0 + 128
    const int64_t block = (int64_t)c.z + warp;          // scale block
    const int64_t s0 = block * kBlockValues + lane * 4; // place in the state arrays
    const bool used = warp * kBlockValues < c.y;        // this warp has values
    float w[kQuads][4], g[kQuads][4], m[kQuads][4], v[kQuads][4];
    if (used) {
      float ms = 0.f, vs = 0.f;
      if constexpr (BITS == 8) {
        ms = __uint_as_float((uint32_t)a.m_scale[block] << 23);
        vs = __uint_as_float((uint32_t)a.v_scale[block] << 23);
      }
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const int at = at0 + q * 128;
        const float4 gv = load4(gp + at, c.y - at, gal), wv = load4(wp + at, c.y - at, wal);
        g[q][0] = gv.x; g[q][1] = gv.y; g[q][2] = gv.z; g[q][3] = gv.w;
        w[q][0] = wv.x; w[q][1] = wv.y; w[q][2] = wv.z; w[q][3] = wv.w;
        if constexpr (BITS == 32) {
          const float4 mv = *reinterpret_cast<const float4*>((const float*)a.m + s0 + q * 128);
          const float4 vv = *reinterpret_cast<const float4*>((const float*)a.v + s0 + q * 128);
          m[q][0] = mv.x; m[q][1] = mv.y; m[q][2] = mv.z; m[q][3] = mv.w;
          v[q][0] = vv.x; v[q][1] = vv.y; v[q][2] = vv.z; v[q][3] = vv.w;
        } else {
          const uint32_t mc = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.m + s0 + q * 128);
          const uint32_t vc = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.v + s0 + q * 128);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            m[q][i] = decode<true>((mc >> (8 * i)) & 255u, ms);
            v[q][i] = decode<false>((vc >> (8 * i)) & 255u, vs);
          }
        }
      }
    }
    __syncthreads();
    if (used) {
      const float size = s_size, rate = s_rate;
      float mmax = 0.f, vmax = 0.f;
      bool fine = true;
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = a.use_norm ? __fmul_rn(g[q][i], clip) : g[q][i];
          m[q][i] = __fadd_rn(__fmul_rn(m[q][i], a.b1), __fmul_rn(x, a.c1));
          v[q][i] = __fadd_rn(__fmul_rn(v[q][i], a.b2), __fmul_rn(__fmul_rn(x, x), a.c2));
          if constexpr (BITS == 8) {
            fine = fine && isfinite(m[q][i]) && isfinite(v[q][i]);
            mmax = fmaxf(mmax, fabsf(m[q][i]));
            vmax = fmaxf(vmax, v[q][i]);
          }
          const float den = __fadd_rn(__fmul_rn(__fsqrt_rn(v[q][i]), rate), a.eps);
          w[q][i] = __fsub_rn(__fmul_rn(w[q][i], a.keep), __fmul_rn(size, __fdiv_rn(m[q][i], den)));
        }
      }
      bool write = true;
      if constexpr (BITS == 8) write = __all_sync(0xffffffffu, fine);
      if (write) {
        float mi = 0.f, vi = 0.f;
        if constexpr (BITS == 8) {
          const uint32_t mb = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(mmax)));
          const uint32_t vb = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(vmax)));
          mi = __uint_as_float((254u - mb) << 23);
          vi = __uint_as_float((254u - vb) << 23);
          if (lane == 0) {
            a.m_scale[block] = (uint8_t)mb;
            a.v_scale[block] = (uint8_t)vb;
          }
        }
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
          const int at = at0 + q * 128;
          store4(wp + at, w[q], c.y - at, wal);
          if constexpr (BITS == 32) {
            *reinterpret_cast<float4*>((float*)a.m + s0 + q * 128) = make_float4(m[q][0], m[q][1], m[q][2], m[q][3]);
            *reinterpret_cast<float4*>((float*)a.v + s0 + q * 128) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
          } else {
            const uint64_t quad = (uint64_t)(s0 + q * 128) >> 2;
            const uint64_t t = (uint64_t)s_t;
            const uint4 r = philox7(make_uint4((uint32_t)quad, (uint32_t)(quad >> 32), (uint32_t)t,
                                               (uint32_t)(t >> 32)), a.seed_lo, a.seed_hi);
            const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
            uint32_t mc = 0, vc = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              mc |= encode<true>(m[q][i], mi, rr[i] & 0xffffu) << (8 * i);
              vc |= encode<false>(v[q][i], vi, rr[i] >> 16) << (8 * i);
            }
            *reinterpret_cast<uint32_t*>((uint8_t*)a.m + s0 + q * 128) = mc;
            *reinterpret_cast<uint32_t*>((uint8_t*)a.v + s0 + q * 128) = vc;
          }
          if constexpr (AVERAGE) {
            float* ap = a.average + s0 + q * 128;   // padded: whole quads
            const float4 av = *reinterpret_cast<const float4*>(ap);
            float e[4] = {av.x, av.y, av.z, av.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = __fadd_rn(__fmul_rn(e[i], a.avg), __fmul_rn(w[q][i], a.avg1));
            *reinterpret_cast<float4*>(ap) = make_float4(e[0], e[1], e[2], e[3]);
          }
        }
      }
    }
  }
  // The last block to finish advances the counters: every block has read its own by then.
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(&a.ws->step_ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (s_last) {
    if (!skip)
      for (int i = threadIdx.x; i < a.tensors; i += kThreads)
        if (list.t[i].grad != nullptr) a.steps[a.tensor0 + i] += 1;
    if (threadIdx.x == 0) a.ws->step_ticket = 0;
  }
}

// Values of 8-bit moments as BF16: four significant bits times a power of two.
__global__ void __launch_bounds__(kThreads) decode_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                          const uint8_t* __restrict__ m_scale,
                                                          const uint8_t* __restrict__ v_scale,
                                                          uint32_t* __restrict__ m_out, uint32_t* __restrict__ v_out,
                                                          int64_t quads) {
  const int64_t q = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (q >= quads) return;
  const int64_t block = q / (kBlockValues / 4);
  const float ms = __uint_as_float((uint32_t)m_scale[block] << 23);
  const float vs = __uint_as_float((uint32_t)v_scale[block] << 23);
  const uint32_t mc = reinterpret_cast<const uint32_t*>(m)[q], vc = reinterpret_cast<const uint32_t*>(v)[q];
  uint32_t mo[4], vo[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mo[i] = __float_as_uint(decode<true>((mc >> (8 * i)) & 255u, ms)) >> 16;
    vo[i] = __float_as_uint(decode<false>((vc >> (8 * i)) & 255u, vs)) >> 16;
  }
  reinterpret_cast<uint2*>(m_out)[q] = make_uint2(mo[0] | mo[1] << 16, mo[2] | mo[3] << 16);
  reinterpret_cast<uint2*>(v_out)[q] = make_uint2(vo[0] | vo[1] << 16, vo[2] | vo[3] << 16);
}

int launched(const char* what) {
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    ictc_set_error(what, cudaGetErrorString(err));
    return ICTC_ERR_CUDA;
  }
  return ICTC_OK;
}

int invalid(const char* what) {
  ictc_set_error(what, "");
  return ICTC_ERR_INVALID;
}

bool bad_list(void* const* weights, const void* const* grads, int first_tensor, int tensors, const int32_t* chunks,
              const int64_t* first_chunk, const void* workspace, bool need_weights) {
  return tensors < 0 || first_tensor < 0 || !first_chunk || !workspace ||
         (tensors > 0 && (!grads || !chunks || (need_weights && !weights)));
}

}  // namespace
}  // namespace ictc

using namespace ictc;

extern "C" int ictc_adamw_chunk_values(void) { return kChunk; }

extern "C" int64_t ictc_adamw_workspace_bytes(void) { return (int64_t)sizeof(Workspace); }

extern "C" int ictc_adamw_grad_norm(const void* const* grads, int tensors, const int32_t* chunks,
                                    const int64_t* first_chunk, float max_norm, int clip, int skip_nonfinite,
                                    void* workspace, void* stream) {
  if (bad_list(nullptr, grads, 0, tensors, chunks, first_chunk, workspace, false) || (clip && !(max_norm > 0.f)))
    return invalid("ictc_adamw_grad_norm: invalid argument%s");
  const int launches = tensors ? (tensors + kList - 1) / kList : 1;
  if (launches > kNormBlocks) return invalid("ictc_adamw_grad_norm: too many tensors%s");
  Args a{};
  a.chunks = reinterpret_cast<const int4*>(chunks);
  a.ws = static_cast<Workspace*>(workspace);
  const int cap = kNormBlocks / launches;
  int slot = 0;
  for (int k = 0; k < launches; ++k) {
    TensorList list{};
    a.tensor0 = k * kList;
    a.tensors = tensors - a.tensor0 < kList ? tensors - a.tensor0 : kList;
    for (int i = 0; i < a.tensors; ++i) list.t[i].grad = static_cast<const float*>(grads[a.tensor0 + i]);
    a.chunk0 = first_chunk[a.tensor0];
    a.chunks_n = first_chunk[a.tensor0 + a.tensors] - a.chunk0;
    const int64_t want = a.chunks_n > 0 ? a.chunks_n : 1;
    const int grid = (int)(want < cap ? want : cap);
    const int last = k == launches - 1;
    grad_norm_kernel<<<grid, kThreads, 0, (cudaStream_t)stream>>>(list, a, slot, slot + grid, last, max_norm, clip,
                                                                  skip_nonfinite);
    if (int rc = launched("ictc_adamw_grad_norm: %s")) return rc;
    slot += grid;
  }
  return ICTC_OK;
}

extern "C" int ictc_adamw_step(void* const* weights, const void* const* grads, int first_tensor, int tensors,
                               const int32_t* chunks, const int64_t* first_chunk, int bits, void* m, void* v,
                               uint8_t* m_scale, uint8_t* v_scale, float* average, int64_t* steps, double lr,
                               double beta1, double beta2, double eps, double weight_decay, double average_decay,
                               uint64_t seed, int use_norm, void* workspace, void* stream) {
  if (bad_list(weights, grads, first_tensor, tensors, chunks, first_chunk, workspace, true) ||
      (bits != 8 && bits != 32) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) ||
      !((float)eps > 0.f) || (tensors > 0 && (!steps || !m || !v || (bits == 8 && (!m_scale || !v_scale)))))
    return invalid("ictc_adamw_step: invalid argument%s");
  Args a{};
  a.chunks = reinterpret_cast<const int4*>(chunks);
  a.m = m;
  a.v = v;
  a.m_scale = m_scale;
  a.v_scale = v_scale;
  a.average = average;
  a.steps = steps;
  a.ws = static_cast<Workspace*>(workspace);
  a.use_norm = use_norm;
  a.b1 = (float)beta1;
  a.c1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2;
  a.c2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.keep = (float)(1.0 - lr * weight_decay);
  a.avg = (float)average_decay;
  a.avg1 = (float)(1.0 - average_decay);
  a.lr = lr;
  a.log_b1 = log(beta1);
  a.log_b2 = log(beta2);
  a.seed_lo = (uint32_t)seed;
  a.seed_hi = (uint32_t)(seed >> 32);
  const int end = first_tensor + tensors;
  for (int t0 = first_tensor; t0 < end; t0 += kList) {
    TensorList list{};
    a.tensor0 = t0;
    a.tensors = end - t0 < kList ? end - t0 : kList;
    for (int i = 0; i < a.tensors; ++i) {
      list.t[i].weight = static_cast<float*>(weights[t0 + i]);
      list.t[i].grad = static_cast<const float*>(grads[t0 + i]);
    }
    a.chunk0 = first_chunk[t0];
    a.chunks_n = first_chunk[t0 + a.tensors] - a.chunk0;
    if (a.chunks_n > 0x7fffffff) return invalid("ictc_adamw_step: too many values in one launch%s");
    const unsigned grid = a.chunks_n ? (unsigned)a.chunks_n : 1u;   // tensors without values still count steps
    cudaStream_t s = (cudaStream_t)stream;
    if (bits == 32) {
      if (average) adamw_kernel<32, true><<<grid, kThreads, 0, s>>>(list, a);
      else adamw_kernel<32, false><<<grid, kThreads, 0, s>>>(list, a);
    } else {
      if (average) adamw_kernel<8, true><<<grid, kThreads, 0, s>>>(list, a);
      else adamw_kernel<8, false><<<grid, kThreads, 0, s>>>(list, a);
    }
    if (int rc = launched("ictc_adamw_step: %s")) return rc;
  }
  return ICTC_OK;
}

extern "C" int ictc_adamw_decode(const void* m, const void* v, const uint8_t* m_scale, const uint8_t* v_scale,
                                 int64_t values, void* m_out, void* v_out, void* stream) {
  if (values < 0 || values % kBlockValues || (values > 0 && (!m || !v || !m_scale || !v_scale || !m_out || !v_out)))
    return invalid("ictc_adamw_decode: invalid argument%s");
  if (values == 0) return ICTC_OK;
  const int64_t quads = values / 4, grid = (quads + kThreads - 1) / kThreads;
  if (grid > 0x7fffffff) return invalid("ictc_adamw_decode: too many values%s");
  decode_kernel<<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(
      (const uint8_t*)m, (const uint8_t*)v, m_scale, v_scale, (uint32_t*)m_out, (uint32_t*)v_out, quads);
  return launched("ictc_adamw_decode: %s");
}
