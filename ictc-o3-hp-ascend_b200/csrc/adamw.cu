// AdamW over many tensors in one launch, with moments in 32 or in 8 bits.
//
// For a tensor whose step counter is t - 1 (g' = clip * g, all in FP32):
//   m = b1 m + (1 - b1) g'         v = b2 v + (1 - b2) g'^2
//   w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//   average = d average + (1 - d) w                                   (optional)
// clip = min(1, max_norm / (|g| + 1e-6)) comes from a first pass over the gradients
// (grad_norm_kernel) when clipping or skipping of non-finite steps is asked for; it is NaN where |g| is.
//
// Work is cut into chunks of consecutive values of one tensor; a static device table gives
// each chunk's tensor, place and count, and the addresses of weights and gradients travel
// in the kernel's parameters (they may change from step to step).  One block per chunk,
// which it works off in turns of 1,024 values, eight per thread; how many turns a chunk
// has goes by the total (the caller's rule): one where there are few values, since
// latency counts, 8 where there are many, since a block's own costs then spread.
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
// never rounds to code zero (the weight's step divides by sqrt(v); in blocks whose scale is below 2^-119 the least
// codes' values leave FP32's range and are zero all the same: largest gradients of some 1e-17).  A block whose new moments
// are not all finite is left as it was, its weights too: the codes hold no NaN.
// Every product of the moments is rounded by itself (no FMA contraction), so the codes
// do not depend on how the compiler pairs operations.
//
// Measured on a B200 (copy rate 6,565 GB/s), 160 M values in 230 tensors: 32-bit step 674 us
// (28 B per value: 6,650 GB/s), with average 870 us (36 B: 6,620 GB/s): bound by memory.  (Above the copy's
// rate: the memory serves four reads per three writes faster than one per one; torch's addition of two arrays reaches
// 6,990 GB/s here, its copy 6,610.)  8-bit step 545 us (16 B: 4,700 GB/s), with average 701 us: neither memory (72%
// of the copy's rate) nor issue slots (63% taken, 80 instructions per value, a fifth of them Philox) are full; warps
// wait for their loads, since 20 warps per multiprocessor have no registers left to read ahead.  Gradient norm 108 us
// (4 B: 5,930 GB/s).  Decoding 148 us (6 B: 6,490 GB/s).  30,000 values in 42 tensors: 8 us (6 us with 8 bits), launch
// and latency.
#include "ictc_cuda.h"

#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

void ictc_set_error(const char* fmt, const char* detail);

namespace ictc {
namespace {

constexpr int kThreads = 128;
constexpr int kTurn = 1024;           // values that a block works on at once: 8 per thread
constexpr int kQuads = 2;             // groups of 4 values per thread
constexpr int kBlockValues = 256;     // values that share a scale: 32 lanes x 8
constexpr int kNormBlocks = 1184;     // partial sums of the gradient norm at most
constexpr int kRounds = 7;            // of Philox: the fewest its authors report as passing their tests
constexpr int kList = 240;            // tensors per launch: 16 B each, below 4 KB of parameters

static_assert(kTurn == kThreads * kQuads * 4 && kBlockValues == 32 * kQuads * 4, "a warp owns one scale block");

// A tensor's bias corrections for its next step, left behind by the last one: a block then reads
// them with its values instead of waiting for one thread's FP64 exponentials (8-bit states, 160 M
// values: 820 -> 716 us).  They hold for the step number and betas they name, else they are made again: betas by
// their FP64 logarithms, since betas near 1 that FP32 cannot tell apart may differ by a tenth of 1 - b.
struct alignas(32) Rate {
  float m;        // 1 / (1 - b1^t)
  float v;        // 1 / sqrt(1 - b2^t)
  double log_b1, log_b2;
  int64_t t;
};

__device__ __forceinline__ Rate rate_of(int64_t t, double log_b1, double log_b2) {
  return Rate{(float)(1.0 / -expm1((double)t * log_b1)), (float)(1.0 / sqrt(-expm1((double)t * log_b2))), log_b1, log_b2,
              t};
}

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
  int chunk;            // values per chunk: kTurn << shift
  int shift;
  int64_t chunk0;
  int64_t chunks_n;
  void* m;
  void* v;
  uint8_t* m_scale;
  uint8_t* v_scale;
  float* average;
  int64_t* steps;
  Rate* rates;
  Workspace* ws;
  int use_norm;
  float b1, c1, b2, c2;      // betas and 1 - beta
  float lr, eps, keep;       // keep = 1 - lr wd
  // The average as a step of `share` from one value towards the other (d and 1 - d rounded by themselves do not
  // add up to one: at d = 0.9999 an average of equal weights would drift by 1.7e-4 of them); nearer: share = -d, from
  // the new weight, so that d = 0 gives the weight itself, else share = 1 - d, from the old average.
  float share;
  int nearer;
  double log_b1, log_b2;
  uint2 keys[kRounds];       // Philox key schedule of the seed
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

// Philox4x32 with the keys of its rounds given.
__device__ __forceinline__ uint4 philox(uint4 c, const uint2 (&keys)[kRounds]) {
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u;
    const uint64_t b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ keys[r].x, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ keys[r].y,
                   (uint32_t)a);
  }
  return c;
}

// Value of the code in byte i of a word.
template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t word, int i, float scale) {
  const uint32_t top = __byte_perm(word, 0, i << 12 | 0x0444);      // the byte in bits 24..31, zeros below
  const uint32_t low = SIGNED ? top >> 4 & 0x07f00000u : top >> 4;
  uint32_t bits = low + ((SIGNED ? 896u : 768u) << 20);
  if (SIGNED) bits |= top & 0x80000000u;
  return low ? __uint_as_float(bits) * scale : 0.f;
}

// Codes of four values in a word, r16: random bits in each's lowest 16 (a's own half of the
// Philox words).  As a rule all magnitudes lie between the least code's value and the block's
// largest, and a code is the top of the pattern plus random bits below it: 896 and 768 are multiples of
// a code's range, so the low bits of the sum need no subtraction.  `rare` covers the rest: zeros and
// values below the least code, or scales at their limit.
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(const float (&x)[4], float inv_scale, const uint32_t (&r)[4], bool top) {
  constexpr float least = SIGNED ? 1.125f / 32768.f : 1.125f / 2147483648.f;
  float a[4];
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = fabsf(x[i]) * inv_scale;
    const uint32_t r16 = SIGNED ? r[i] & 0xffffu : r[i] >> 16;
    q[i] = (__float_as_uint(a[i]) + (r16 << 4)) >> 20;
  }
  const bool rare = top || fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) < least;
  if (rare) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r16 = SIGNED ? r[i] & 0xffffu : r[i] >> 16;
      if (a[i] < least) q[i] = SIGNED ? ((float)r16 < a[i] * (65536.f / least) ? 1u : 0u) : (a[i] > 0.f ? 1u : 0u);
      else q[i] = min(q[i] - (SIGNED ? 896u : 768u), SIGNED ? 127u : 255u);
    }
  }
  const uint32_t codes = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  if (!SIGNED) return codes;
  const uint32_t signs = __byte_perm(__byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x0073),
                                     __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x0073), 0x5410);
  uint32_t out = (codes & 0x7f7f7f7fu) | (signs & 0x80808080u);
  if (rare) {      // no sign without a value
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (q[i] == 0) out &= ~(0xffu << (8 * i));
  }
  return out;
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
  constexpr int kAhead = 4;      // turns whose values are in flight together
  double sum = 0.0;
  const int64_t total = a.chunks_n << a.shift;
  for (int64_t i0 = blockIdx.x; i0 < total; i0 += kAhead * (int64_t)gridDim.x) {
    float4 x[kAhead][kQuads];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * (int64_t)gridDim.x;
      const int turn = (int)(i & ((1 << a.shift) - 1)) * kTurn;
      const int4 c = i < total ? a.chunks[a.chunk0 + (i >> a.shift)] : make_int4(a.tensor0, 0, 0, 0);
      const float* g = list.t[c.x - a.tensor0].grad;
      const int count = g == nullptr ? 0 : c.y - turn;
      g += (int64_t)c.w * a.chunk + turn;
      const bool al = aligned16(g);
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const int at = (q * kThreads + threadIdx.x) * 4;
        x[k][q] = load4(g + at, count - at, al);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        sum += (double)x[k][q].x * x[k][q].x;
        sum += (double)x[k][q].y * x[k][q].y;
        sum += (double)x[k][q].z * x[k][q].z;
        sum += (double)x[k][q].w * x[k][q].w;
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
      const float share = __fmul_rn(__frcp_rn(__fadd_rn(norm, 1e-6f)), max_norm);
      a.ws->clip = clip && !(share > 1.f) ? share : 1.f;      // a NaN norm stays one, as a minimum would not
      a.ws->skip = skip_bad && !isfinite(sum);
    }
    a.ws->norm_ticket = 0;
  }
}

// What a lane reads of one turn.
template <int BITS, bool AVERAGE>
struct Turn {
  float4 w[kQuads], g[kQuads], m[BITS == 32 ? kQuads : 1], v[BITS == 32 ? kQuads : 1], e[AVERAGE ? kQuads : 1];
  uint32_t mc[BITS == 8 ? kQuads : 1], vc[BITS == 8 ? kQuads : 1];
};

// s0: place in the state arrays; left: values of the tensor from this lane's first one on.
template <int BITS, bool AVERAGE>
__device__ __forceinline__ void read(Turn<BITS, AVERAGE>& x, const Args& a, const float* w, const float* g, int64_t s0,
                                     int left, bool fast, bool wal, bool gal) {
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    if (fast) {
      x.g[q] = *reinterpret_cast<const float4*>(g + q * 128);
      x.w[q] = *reinterpret_cast<const float4*>(w + q * 128);
    } else {
      x.g[q] = load4(g + q * 128, left - q * 128, gal);
      x.w[q] = load4(w + q * 128, left - q * 128, wal);
    }
    if constexpr (BITS == 32) {
      x.m[q] = *reinterpret_cast<const float4*>((const float*)a.m + s0 + q * 128);
      x.v[q] = *reinterpret_cast<const float4*>((const float*)a.v + s0 + q * 128);
    } else {
      x.mc[q] = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.m + s0 + q * 128);
      x.vc[q] = *reinterpret_cast<const uint32_t*>((const uint8_t*)a.v + s0 + q * 128);
    }
    if constexpr (AVERAGE) x.e[q] = *reinterpret_cast<const float4*>(a.average + s0 + q * 128);   // padded
  }
}

// mb, vb: the block's scale bytes, in and out.
template <int BITS, bool AVERAGE>
__device__ __forceinline__ void update(const Turn<BITS, AVERAGE>& x, const Args& a, float* wp, int64_t s0, int left,
                                       bool fast, bool wal, float clip, float size, float rate, int64_t t,
                                       uint32_t& mb, uint32_t& vb) {
  float w[kQuads][4], m[kQuads][4], v[kQuads][4];
  uint32_t mmax = 0, vmax = 0;      // as patterns: infinities and NaN are the largest
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    const float g[4] = {x.g[q].x, x.g[q].y, x.g[q].z, x.g[q].w}, ow[4] = {x.w[q].x, x.w[q].y, x.w[q].z, x.w[q].w};
    float om[4], ov[4];
    if constexpr (BITS == 32) {
      om[0] = x.m[q].x; om[1] = x.m[q].y; om[2] = x.m[q].z; om[3] = x.m[q].w;
      ov[0] = x.v[q].x; ov[1] = x.v[q].y; ov[2] = x.v[q].z; ov[3] = x.v[q].w;
    } else {
      const float ms = __uint_as_float(mb << 23), vs = __uint_as_float(vb << 23);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        om[i] = decode<true>(x.mc[q], i, ms);
        ov[i] = decode<false>(x.vc[q], i, vs);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = __fmul_rn(g[i], clip);
      m[q][i] = __fadd_rn(__fmul_rn(om[i], a.b1), __fmul_rn(y, a.c1));
      v[q][i] = __fadd_rn(__fmul_rn(ov[i], a.b2), __fmul_rn(__fmul_rn(y, y), a.c2));
      if constexpr (BITS == 8) {
        mmax = max(mmax, __float_as_uint(fabsf(m[q][i])));
        vmax = max(vmax, __float_as_uint(v[q][i]));      // a NaN of a sum of squares is positive
        // bound by its instructions: hardware root and quotient (within 2 units in the last place)
        float root;
        asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v[q][i]));
        const float den = fmaf(root, rate, a.eps);
        w[q][i] = fmaf(ow[i], a.keep, -size * __fdividef(m[q][i], den));
      } else {
        const float den = __fadd_rn(__fmul_rn(__fsqrt_rn(v[q][i]), rate), a.eps);
        w[q][i] = __fsub_rn(__fmul_rn(ow[i], a.keep), __fmul_rn(size, __fdiv_rn(m[q][i], den)));
      }
    }
  }
  bool mtop = false, vtop = false;
  float mi = 0.f, vi = 0.f;
  if constexpr (BITS == 8) {
    mmax = __reduce_max_sync(0xffffffffu, mmax);
    vmax = __reduce_max_sync(0xffffffffu, vmax);
    if (max(mmax, vmax) >= 0x7f800000u) return;      // the codes hold no NaN: the block stays as it was
    mb = scale_byte(mmax);
    vb = scale_byte(vmax);
    mtop = mb == 253u;
    vtop = vb == 253u;
    mi = __uint_as_float((254u - mb) << 23);
    vi = __uint_as_float((254u - vb) << 23);
  }
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    if (fast) *reinterpret_cast<float4*>(wp + q * 128) = make_float4(w[q][0], w[q][1], w[q][2], w[q][3]);
    else store4(wp + q * 128, w[q], left - q * 128, wal);
    if constexpr (BITS == 32) {
      *reinterpret_cast<float4*>((float*)a.m + s0 + q * 128) = make_float4(m[q][0], m[q][1], m[q][2], m[q][3]);
      *reinterpret_cast<float4*>((float*)a.v + s0 + q * 128) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
    } else {
      const uint64_t quad = (uint64_t)(s0 + q * 128) >> 2;
      const uint4 r = philox(make_uint4((uint32_t)quad, (uint32_t)(quad >> 32), (uint32_t)t,
                                        (uint32_t)((uint64_t)t >> 32)), a.keys);
      const uint32_t rr[4] = {r.x, r.y, r.z, r.w};
      *reinterpret_cast<uint32_t*>((uint8_t*)a.m + s0 + q * 128) = encode<true>(m[q], mi, rr, mtop);
      *reinterpret_cast<uint32_t*>((uint8_t*)a.v + s0 + q * 128) = encode<false>(v[q], vi, rr, vtop);
    }
    if constexpr (AVERAGE) {
      float e[4] = {x.e[q].x, x.e[q].y, x.e[q].z, x.e[q].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = fmaf(a.share, __fsub_rn(w[q][i], e[i]), a.nearer ? w[q][i] : e[i]);
      *reinterpret_cast<float4*>(a.average + s0 + q * 128) = make_float4(e[0], e[1], e[2], e[3]);
    }
  }
}

// Blocks per multiprocessor.  32-bit states are bound by memory: the next turn's values are on their way
// while one is worked on (160 M values, 8 turns: 673 us, one turn per block 859 us).
// 8-bit ones keep most warps with five blocks and few spills (4: 585, 5: 539, 7: 613 us, one after another).
constexpr int kResident32 = 4, kResident8 = 5;
template <int BITS, bool AVERAGE>
__global__ void __launch_bounds__(kThreads, BITS == 8 ? kResident8 : kResident32)
adamw_kernel(const __grid_constant__ TensorList list, const Args a) {
  __shared__ int s_last;
  const int4 c = a.chunks_n ? a.chunks[a.chunk0 + blockIdx.x] : make_int4(a.tensor0, 0, 0, 0);
  const Tensor tensor = list.t[c.x - a.tensor0];
  const bool skip = a.use_norm && a.ws->skip;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int turns = 1 << a.shift, begin = warp * turns * kBlockValues;      // a warp's scale blocks are neighbours
  if (tensor.grad != nullptr && !skip && begin < c.y) {
    const int at = begin + lane * 4;     // quads at `at` and at + 128 of a turn
    float* w = tensor.weight + (int64_t)c.w * a.chunk + at;
    const float* g = tensor.grad + (int64_t)c.w * a.chunk + at;
    int64_t s0 = (int64_t)c.z * kBlockValues + at;     // place in the state arrays
    const bool wal = aligned16(w), gal = aligned16(g);
    const int whole = c.y / kBlockValues * kBlockValues;      // scale blocks without values to leave out
    const int mine = min(turns, (c.y - begin + kBlockValues - 1) / kBlockValues);
    int from = begin;
    Turn<BITS, AVERAGE> x;
    read(x, a, w, g, s0, c.y - at, wal && gal && from < whole, wal, gal);
    // Scale bytes are read and written once per warp, lane k that of turn k: a byte stored next to one
    // that is read soon holds that read up (four turns with a byte each: 1,421 us, together: 591 us)
    const int64_t scales = (int64_t)c.z + warp * turns + lane;
    uint32_t ms = 1, vs = 1;
    if (BITS == 8 && lane < mine) {
      ms = a.m_scale[scales];
      vs = a.v_scale[scales];
    }
    const int64_t t = a.steps[c.x] + 1;
    Rate rate = a.rates[c.x];
    const float clip = a.use_norm ? a.ws->clip : 1.f;
    if (rate.t != t || rate.log_b1 != a.log_b1 || rate.log_b2 != a.log_b2) rate = rate_of(t, a.log_b1, a.log_b2);
    const float size = a.lr * rate.m;
#pragma unroll 1
    for (int k = 0; k < mine; ++k) {
      const bool fast = wal && gal && from < whole, next = wal && gal && from + kBlockValues < whole;
      const int left = c.y - from - lane * 4;
      constexpr bool PREFETCH = BITS == 32;
      Turn<BITS, AVERAGE> y;
      if (PREFETCH && k + 1 < mine)
        read(y, a, w + kBlockValues, g + kBlockValues, s0 + kBlockValues, left - kBlockValues, next, wal, gal);
      uint32_t mb = 0, vb = 0;
      if constexpr (BITS == 8) {
        mb = __shfl_sync(0xffffffffu, ms, k);
        vb = __shfl_sync(0xffffffffu, vs, k);
      }
      update(x, a, w, s0, left, fast, wal, clip, size, rate.v, t, mb, vb);
      if (BITS == 8 && lane == k) {
        ms = mb;
        vs = vb;
      }
      w += kBlockValues;
      g += kBlockValues;
      s0 += kBlockValues;
      from += kBlockValues;
      if constexpr (PREFETCH) x = y;
      else if (k + 1 < mine) read(x, a, w, g, s0, left - kBlockValues, next, wal, gal);
    }
    if (BITS == 8 && lane < mine) {
      a.m_scale[scales] = (uint8_t)ms;
      a.v_scale[scales] = (uint8_t)vs;
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
        if (list.t[i].grad != nullptr) {
          const int64_t t = a.steps[a.tensor0 + i] + 1;
          a.steps[a.tensor0 + i] = t;
          a.rates[a.tensor0 + i] = rate_of(t + 1, a.log_b1, a.log_b2);
        }
    if (threadIdx.x == 0) a.ws->step_ticket = 0;
  }
}

// Values of 8-bit moments as BF16: four significant bits times a power of two.  16 values per thread.
__global__ void __launch_bounds__(kThreads) decode_kernel(const uint4* __restrict__ m, const uint4* __restrict__ v,
                                                          const uint8_t* __restrict__ m_scale,
                                                          const uint8_t* __restrict__ v_scale,
                                                          uint4* __restrict__ m_out, uint4* __restrict__ v_out,
                                                          int64_t groups) {
  const int64_t k = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (k >= groups) return;
  const int64_t block = k / (kBlockValues / 16);
  const uint4 mc = __ldcs(m + k), vc = __ldcs(v + k);
  const float ms = __uint_as_float((uint32_t)m_scale[block] << 23);
  const float vs = __uint_as_float((uint32_t)v_scale[block] << 23);
  const uint32_t mw[4] = {mc.x, mc.y, mc.z, mc.w}, vw[4] = {vc.x, vc.y, vc.z, vc.w};
  uint32_t mo[8], vo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int j = 2 * (i & 1);
    // the upper halves of two FP32 values side by side
    mo[i] = __byte_perm(__float_as_uint(decode<true>(mw[i / 2], j, ms)),
                        __float_as_uint(decode<true>(mw[i / 2], j + 1, ms)), 0x7632);
    vo[i] = __byte_perm(__float_as_uint(decode<false>(vw[i / 2], j, vs)),
                        __float_as_uint(decode<false>(vw[i / 2], j + 1, vs)), 0x7632);
  }
  m_out[2 * k] = make_uint4(mo[0], mo[1], mo[2], mo[3]);
  m_out[2 * k + 1] = make_uint4(mo[4], mo[5], mo[6], mo[7]);
  v_out[2 * k] = make_uint4(vo[0], vo[1], vo[2], vo[3]);
  v_out[2 * k + 1] = make_uint4(vo[4], vo[5], vo[6], vo[7]);
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
              const int64_t* first_chunk, int chunk, const void* workspace, bool need_weights) {
  return tensors < 0 || first_tensor < 0 || !first_chunk || !workspace || chunk < kTurn || chunk > 32 * kTurn || (chunk & (chunk - 1)) ||
         (tensors > 0 && (!grads || !chunks || (need_weights && !weights)));
}

}  // namespace
}  // namespace ictc

using namespace ictc;

extern "C" int ictc_adamw_turn_values(void) { return kTurn; }

extern "C" int64_t ictc_adamw_workspace_bytes(void) { return (int64_t)sizeof(Workspace); }

extern "C" int ictc_adamw_grad_norm(const void* const* grads, int tensors, const int32_t* chunks,
                                    const int64_t* first_chunk, int chunk, float max_norm, int clip, int skip_nonfinite,
                                    void* workspace, void* stream) {
  if (bad_list(nullptr, grads, 0, tensors, chunks, first_chunk, chunk, workspace, false) || (clip && !(max_norm > 0.f)))
    return invalid("ictc_adamw_grad_norm: invalid argument%s");
  const int launches = tensors ? (tensors + kList - 1) / kList : 1;
  if (launches > kNormBlocks) return invalid("ictc_adamw_grad_norm: too many tensors%s");
  Args a{};
  a.chunks = reinterpret_cast<const int4*>(chunks);
  a.chunk = chunk;
  while (kTurn << a.shift < chunk) ++a.shift;
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
    const int64_t turns = a.chunks_n << a.shift, want = turns > 0 ? turns : 1;
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
                               const int32_t* chunks, const int64_t* first_chunk, int chunk, int bits, void* m, void* v,
                               uint8_t* m_scale, uint8_t* v_scale, float* average, int64_t* steps, void* rates, double lr,
                               double beta1, double beta2, double eps, double weight_decay, double average_decay,
                               uint64_t seed, int use_norm, void* workspace, void* stream) {
  if (bad_list(weights, grads, first_tensor, tensors, chunks, first_chunk, chunk, workspace, true) ||
      (bits != 8 && bits != 32) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) ||
      !((float)eps > 0.f) || (tensors > 0 && (!steps || !rates || !m || !v || (bits == 8 && (!m_scale || !v_scale)))))
    return invalid("ictc_adamw_step: invalid argument%s");
  Args a{};
  a.chunks = reinterpret_cast<const int4*>(chunks);
  a.chunk = chunk;
  while (kTurn << a.shift < chunk) ++a.shift;
  a.m = m;
  a.v = v;
  a.m_scale = m_scale;
  a.v_scale = v_scale;
  a.average = average;
  a.steps = steps;
  a.rates = static_cast<Rate*>(rates);
  a.ws = static_cast<Workspace*>(workspace);
  a.use_norm = use_norm;
  a.b1 = (float)beta1;
  a.c1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2;
  a.c2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.keep = (float)(1.0 - lr * weight_decay);
  a.nearer = average_decay < 0.5;
  a.share = (float)(a.nearer ? -average_decay : 1.0 - average_decay);
  a.lr = (float)lr;
  a.log_b1 = log(beta1);
  a.log_b2 = log(beta2);
  for (uint32_t r = 0; r < kRounds; ++r)
    a.keys[r] = make_uint2((uint32_t)seed + r * 0x9E3779B9u, (uint32_t)(seed >> 32) + r * 0xBB67AE85u);
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
  const int64_t groups = values / 16, grid = (groups + kThreads - 1) / kThreads;
  if (grid > 0x7fffffff) return invalid("ictc_adamw_decode: too many values%s");
  decode_kernel<<<(unsigned)grid, kThreads, 0, (cudaStream_t)stream>>>(
      (const uint4*)m, (const uint4*)v, m_scale, v_scale, (uint4*)m_out, (uint4*)v_out, groups);
  return launched("ictc_adamw_decode: %s");
}
