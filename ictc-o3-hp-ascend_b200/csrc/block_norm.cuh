// Norms before and after a block, its gate and its residual scale, in one pass over the rows.
//
// A row holds degrees l = 0..L with C channels of 2l+1 components (C (L+1)^2 values; a degree
// is [C][2l+1] or [2l+1][C]).  With D = C (2l+1) and <.,.> a degree's scalar product,
//   r(x) = (<x,x> / D + eps)^(-1/2)
//   h' = h + a r(y) y,  a = post scale sigma(gate)        per (degree, channel); gate optional
//   u  = b r(h') h',    b = pre                           optional; without y: u of h itself
// First gradients for cotangents p of h' and q of u, with n = r1 y, k = r2 h', D inside <.,.>
// from here on (means):
//   T  = p + r2 (b q - k <k, b q>)                        gradient of h
//   dy = r1 (a T - n <n, a T>)
//   S  = sum_m n T                                        per channel
//   dgate = post scale sigma' S,  d(post scale) = sum_n sigma S,  db = sum_n sum_m k q
// and <n, a T> = sum_c a S / D.  Second: cotangents al, be, ga of T, dy, dgate; with
// inner = r1 (be - n <n,be>) and z = ga post scale sigma':
//   tau = al + a inner + z n                              gradient of p
//   gy  = r1^2 (3 n <n,aT> <n,be> - n <aT,be> - aT <n,be> - be <n,aT>) + r1 (z T - n <n,zT>)
//   ga' = r1 (sum_m T be - <n,be> S)                      gradient of a, per channel
//   g(post scale) = sum_n (sigma ga' + ga sigma' S),  ggate = post scale (sigma' ga' + ga sigma'' S)
//   down = r2 (tau - k <k,tau>),  gq = b down,  gb = sum_n sum_m q down
//   gh' = r2^2 (3 k <k,bq> <k,tau> - k <bq,tau> - bq <k,tau> - tau <k,bq>)
// (written with n and k, not with powers of r: r^3 leaves FP32's range for rows of 1e13).
//
// All three are bound by the rows they read and write.  A lane owns one channel with all its
// components, C lanes (one warp for several rows, or several warps for one) a row: sums over components
// and per-channel values stay in a lane, weights and their gradients' sums in its registers, and
// only the degrees' scalar products cross lanes.  A tile of rows is brought into shared memory by
// asynchronous copies, one or more tiles ahead, read once, written back in place and leaves as contiguous
// rows: a lane's channel lies 2l+1 values from its neighbour's, an odd stride, which shared
// memory serves without conflicts and device memory would not.  Low degrees take several rows
// per tile, so that a lane holds about 16 values of each tensor.  Rows wider than a
// block's lanes (HOLD false) go over their channels in turns and read shared memory again
// in every phase.  Weight gradients are summed per block and then over blocks by a second kernel, in
// a fixed order: no atomics, the same bits every time.
//
// Measured on a B200 (copy rate 6,565 GB/s; bytes: every row array once), with gate:
//   262,144 rows of C64/lmax 2: forward 436 us (6,010 GB/s), backward with weights 647 us (6,220),
//   second 1,250 us (5,320);  8,192 rows of C128/lmax 3: 51 us (5,620), 80 us (5,420), 175 us (4,120);
//   50,000 rows of C132/lmax 1: 91 us (5,210), 162 us (4,570), 392 us (3,100);
//   100,000 rows of C128/lmax 0: 63 us (4,040), 101 us (4,050), 218 us (3,050);
//   without bulk copies (addresses off by one value): C64/lmax 2 642 us, 1,013 us, 2,098 us; C128/lmax 3
//   80 us, 134 us, 292 us; C132/lmax 1 156 us, 248 us, 556 us; 32,768 rows of C50/lmax 2 93 us (2,740), 151 us, 286 us;
//   wide rows (HOLD false: more than 512 channels, 384 or 256 in some derivatives): 20,000 rows of C512/lmax 1 173 us
//   (4,260), 257 us (4,460), 1,283 us (1,470); 4,000 rows of C450/lmax 3 106 us (4,640), 314 us (2,390), 516 us (2,400);
//   20,000 rows of C1028/lmax 0 597 us (690), 779 us (840), 1,119 us (960).
// The forward and the first gradients are near the memory's rate at lmax 2 and 3.  The second derivatives at lmax 3 stage 53 KB per
// row of C128, so two rows are worked on and two are under way per multiprocessor: eight warps, bound by the
// latency of their instructions (issue slots 37% taken; with no row written and half of the inputs 600 of 646 us
// at 32,768 rows).  Two sets of warps per row, one for degree 3 and one for the rest, gave 615 us there but lost at
// C64 and were dropped.  At lmax 0 a row is short and the fixed work per tile (sums, barriers, copies) shows.
#pragma once

#include "ictc_common.cuh"
#include "ictc_cuda.h"
#include "tc_sm100.cuh"

#include <atomic>
#include <cstdio>

void ictc_set_error(const char* fmt, const char* detail);

namespace ictc {
namespace block_norm {

constexpr int kMaxL = 3;
constexpr int kMaxDevices = 64;
constexpr int kSharedLimit = 227 * 1024;

enum Mode : int { kForward = 0, kBackward = 1, kSecond = 2 };

// Of 227 KB; the forward does better with some left as L1 (32,768 rows of C128/lmax 3: 196 us with 220 KB).
__host__ __device__ constexpr int shared_budget(int mode) { return (mode == kForward ? 200 : 220) * 1024; }

// Staged tensors: 0..5 rows, then per-channel and per-degree ones.
//   forward  y h . . . .      backward  y h' p q . .      second  y h' p q al be
// (without a branch, the norm alone: . h, . h' . q, . h' . q al .)
enum Slot : int { kY, kH, kP, kQ, kAl, kBe, kGate, kGateDot, kR1, kR2, kSlots };

// Rows that a lane works on at once, and warps per block, by mode and lmax.  Low degrees have few
// values per row: several rows share a tile's barriers, sums and copies.  More rows per lane mean
// more registers and so fewer warps; measured on 50,000 to 100,000 rows, both sides of each choice:
//   forward  lmax 0, C128: 8 rows 74 us, 4 rows 96;  lmax 1, C132: 4 rows 98, 2 rows 127;
//            lmax 2, 262,144 rows of C64: 2 rows 454 (20 warps), 1 row 437 (24 warps);  lmax 3, 32,768
//            rows of C128: 20 warps 196, 16 warps 190
//   backward lmax 0, C128: 8 rows 104, 4 rows 141;  lmax 1, C132: 4 rows 223 (16 warps), 2 rows 162 (20 warps);
//            lmax 2, C64: 2 rows 217, 1 row 178;  lmax 3, 8,192 rows of C128: 16 warps 90, 12 warps 84
//   second   lmax 0, C128: 4 rows 218 (16 warps) or 263 (12), 2 rows 347;  lmax 1, C50: 2 rows 142, 1 row 171;
//            lmax 2, C64: 2 rows 404, 1 row 331
__host__ __device__ constexpr int rows_per_lane(int mode, int L, bool hold) {
  constexpr int rows[3][kMaxL + 1] = {{8, 4, 1, 1}, {8, 2, 1, 1}, {4, 2, 1, 1}};
  return hold ? rows[mode][L] : 1;
}
__host__ __device__ constexpr int max_warps(int mode, int L) {
  constexpr int warps[3][kMaxL + 1] = {{24, 24, 24, 16}, {16, 20, 20, 12}, {16, 12, 12, 8}};
  return warps[mode][L];
}
// Warps of one row at most; wider rows take turns (HOLD false), and the widest ones leave room
// for the scratch of twelve.
__host__ __device__ constexpr int max_row_warps(int mode, int L) {
  const int most = mode == kSecond ? 12 : 16;
  return max_warps(mode, L) < most ? max_warps(mode, L) : most;
}
constexpr int kScratch = 16;                          // sums of one warp
constexpr int kBarrierFloats = 8;                     // room of four mbarriers
constexpr uint64_t kWaitNs = 2000000000ull;           // BlockArgs::wait_ns, unless a test shortens it; limit of draining

struct BlockArgs {
  const float* in[kSlots];  // null: zeros, or not there
  float* out[6];            // where rows go afterwards, or null
  int at[kSlots];           // floats from the start of a stage, -1: no place
  unsigned wide;            // bit s: tensor s is copied 16 bytes at a time
  float* gate_out;          // dgate / its adjoint, or null
  const float* post;        // [L+1, C] or null (1)
  const float* scale;
  const float* pre;
  int* status;              // 1 (3) after a copy did not land in time (nor while draining)
  uint64_t wait_ns;         // a copy that takes longer is given up; 0: every copy is, unseen
  float* r1_out;            // [N, 4], or null (forward)
  float* r2_out;
  float* partial;           // [blocks][2][(L+1) C] weight-gradient sums, or null
  int64_t rows;
  int channels;
  int lanes;                // lanes per row
  int warps;                // warps per group
  int per;                  // rows of a tile
  int stages;
  int stage_floats;
  int group_floats;
  int row_bytes;            // staged bytes of one row
  int norm;                 // u (or its cotangent) takes part
  float eps;
  float inv[kMaxL + 1];     // 1 / D of every degree
};

struct Shape {
  int hold, bulk, lanes, warps, per, stages, groups;
};

__device__ __forceinline__ void copy_async16(float* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_async4(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait(int pending) {
  if (pending >= 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// One warp (holding 32 / lanes rows at a time) or several warps of one row.
struct Group {
  int id;        // in the block
  int thread;    // in the group
  int threads;
  int lanes;
  float* scratch;   // two buffers, used in turn: one barrier per sum
  int turn;

  __device__ __forceinline__ void sync() const {
    if (threads == 32) __syncwarp();
    else tc::named_barrier(id + 1, threads);
  }
  __device__ __forceinline__ bool sync_all(bool x) const {
    return threads == 32 ? __all_sync(0xffffffffu, x) : tc::named_barrier_all(id + 1, threads, x);
  }
  // Sums of N values over a row's lanes, in a fixed order, in every lane.  Over whole warps
  // each exchange halves the values that a lane carries on (N - 1 + 5 - log2 N exchanges
  // instead of 5 N); the sums then go round through shared memory, as they must between warps.
  template <int N>
  __device__ __forceinline__ void sum(float (&x)[N]) {
    static_assert(N <= kScratch, "scratch");
    if (lanes < 32) {
      for (int o = lanes >> 1; o; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
      }
      return;
    }
    constexpr int P = N > 8 ? 16 : N > 4 ? 8 : N > 2 ? 4 : N;
    float v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = i < N ? x[i] : 0.f;
    const int lane = thread & 31;
    int index = 0;
#pragma unroll
    for (int step = 0; step < 5; ++step) {
      const int o = 16 >> step, half = P >> (step + 1);
      if (half > 0) {
        const bool upper = lane & o;
        index += upper ? half : 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float keep = upper ? v[i + half] : v[i], give = upper ? v[i] : v[i + half];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      }
    }
    const int warps = threads >> 5;
    float* s = scratch + turn * warps * kScratch;
    turn ^= 1;
    if ((lane & (32 / P - 1)) == 0) s[(thread >> 5) * kScratch + index] = v[0];
    sync();
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    for (int w = 0; w < warps; ++w) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 t = *reinterpret_cast<const float4*>(s + w * kScratch + i);
        x[i] += t.x;
        if (i + 1 < N) x[i + 1] += t.y;
        if (i + 2 < N) x[i + 2] += t.z;
        if (i + 3 < N) x[i + 3] += t.w;
      }
    }
  }
};

// 1 / (1 + exp(-g)) from the hardware's 2^x and quotient, with the rounding of g log2(e) put
// back (2^x alone is off by |g| half steps).
__device__ __forceinline__ float sigmoid(float g) {
  constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.9259629911266175e-8f;
  const float t = -g * kLog2e;
  const float rest = (fmaf(-g, kLog2e, -t) - g * kLog2eRest) * 0.6931471805599453f;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  if (fabsf(t) < 126.f) e = fmaf(e, rest, e);     // beyond, 0 and infinity stay what they are
  return __fdividef(1.f, 1.f + e);
}

// Values of one channel in R rows.
template <int R, int L>
struct Vals {
  float v[R][(L + 1) * (L + 1)];
};

template <int L, int LAYOUT, int R>
__device__ __forceinline__ void load(Vals<R, L>& x, const float* rows, int step, int C, int c) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int l = 0; l <= L; ++l)
#pragma unroll
      for (int m = 0; m < 2 * l + 1; ++m)
        x.v[r][l * l + m] = rows[r * step + C * l * l + (LAYOUT == kMulIr ? c * (2 * l + 1) + m : m * C + c)];
}
template <int L, int LAYOUT, int R>
__device__ __forceinline__ void store(const Vals<R, L>& x, float* rows, int step, int C, int c) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int l = 0; l <= L; ++l)
#pragma unroll
      for (int m = 0; m < 2 * l + 1; ++m)
        rows[r * step + C * l * l + (LAYOUT == kMulIr ? c * (2 * l + 1) + m : m * C + c)] = x.v[r][l * l + m];
}
template <int R, int L>
__device__ __forceinline__ void zero(Vals<R, L>& x) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int e = 0; e < (L + 1) * (L + 1); ++e) x.v[r][e] = 0.f;
}

// Channel weights of a lane: w = post scale, b = pre.
template <int N>
struct Weights {
  float w[N], b[N];
  __device__ __forceinline__ void load(const BlockArgs& a, int c) {
#pragma unroll
    for (int l = 0; l < N; ++l) {
      const int at = l * a.channels + c;
      w[l] = (a.post ? __ldg(a.post + at) : 1.f) * (a.scale ? __ldg(a.scale + at) : 1.f);
      b[l] = a.pre ? __ldg(a.pre + at) : 1.f;
    }
  }
};

#define ICTC_ROWS(r, R) _Pragma("unroll") for (int r = 0; r < R; ++r)
#define ICTC_DEGREES(l, N) _Pragma("unroll") for (int l = 0; l < N; ++l)
#define ICTC_PARTS(e, l) _Pragma("unroll") for (int e = l * l; e < (l + 1) * (l + 1); ++e)

__device__ __forceinline__ void bulk_store(float* dst, const float* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(tc::smem_u32(src)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All bulk stores of this thread have read shared memory.
__device__ __forceinline__ void bulk_read_wait() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// HOLD: a lane has one channel and keeps its values between phases.  BULK: every tensor of a tile is
// 16-byte aligned and a multiple of 16 bytes and moves by one bulk copy each way, issued by the group's
// first thread; otherwise all threads copy, 16 or 4 bytes at a time.
template <int L, int LAYOUT, int MODE, bool BRANCH, bool HOLD, bool BULK>
__global__ void __launch_bounds__(32 * max_warps(MODE, L)) block_kernel(const __grid_constant__ BlockArgs a) {
  extern __shared__ __align__(16) float shared[];
  constexpr int N = L + 1, R = rows_per_lane(MODE, L, HOLD);
  using V = Vals<R, L>;
  const int C = a.channels, W = C * N * N, width = N * C;
  Group g;
  g.threads = 32 * a.warps;
  g.id = threadIdx.x / g.threads;
  g.thread = threadIdx.x % g.threads;
  g.lanes = a.lanes;
  g.turn = 0;
  const int groups = blockDim.x / g.threads;
  float* ring = shared + g.id * a.group_floats;
  g.scratch = ring + a.stages * a.stage_floats;
  uint64_t* full = reinterpret_cast<uint64_t*>(g.scratch + 2 * a.warps * kScratch);      // one per stage
  float* acc = g.scratch + 2 * a.warps * kScratch + kBarrierFloats;      // weight-gradient sums (HOLD false)
  const int sub = g.thread / a.lanes;                   // this lane's rows are sub + r * (rows / R) of the tile
  const int c0 = g.thread - sub * a.lanes;
  const int apart = a.per / R;
  const int64_t tiles = (a.rows + a.per - 1) / a.per;
  const int64_t first = (int64_t)blockIdx.x * groups + g.id, stride = (int64_t)gridDim.x * groups;
  if (!HOLD && a.partial)
    for (int i = g.thread; i < 2 * width; i += g.threads) acc[i] = 0.f;

  int issued = 0;      // tiles asked for by bulk copies (the group's first thread)
  // The tile t goes into `stage`; with bulk copies this is the first thread's business alone.
  auto fetch = [&](int64_t t, int stage) {
    if constexpr (BULK) {
      if (g.thread == 0 && t < tiles) {
        const int64_t row0 = t * a.per;
        const uint32_t rows = (uint32_t)(a.rows - row0 < a.per ? a.rows - row0 : a.per);
        float* base = ring + stage * a.stage_floats;
        tc::mbar_arrive_expect(full + stage, rows * a.row_bytes);
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
          if (a.in[s] == nullptr) continue;
          const int wd = s < kGate ? W : s < kR1 ? width : 4;
          tc::bulk_load(base + a.at[s], a.in[s] + row0 * wd, rows * wd * 4, full + stage);
        }
        ++issued;
      }
      return;
    }
    if (t < tiles) {
      const int64_t row0 = t * a.per;
      const int rows = (int)(a.rows - row0 < a.per ? a.rows - row0 : a.per);
      float* base = ring + stage * a.stage_floats;
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        if (a.in[s] == nullptr || a.at[s] < 0) continue;
        const int wd = s < kGate ? W : s < kR1 ? width : 4;
        float* dst = base + a.at[s];
        const float* src = a.in[s] + row0 * wd;
        const int count = rows * wd;
        int i = 0;
        if (a.wide >> s & 1u) {
#pragma unroll 4
          for (int j = 4 * g.thread; j + 3 < count; j += 4 * g.threads) copy_async16(dst + j, src + j);
          i = count & ~3;
        }
        for (i += g.thread; i < count; i += g.threads) copy_async4(dst + i, src + i);
      }
    }
    copies_commit();
  };
  // f(c) for the lane's channels: one, or (HOLD false) several in turn.
  auto each = [&](auto&& f) {
    if constexpr (HOLD) {
      if (c0 < C) f(c0);
    } else {
      for (int c = c0; c < C; c += a.lanes) f(c);
    }
  };

  Weights<N> own;
  float sum_w[N], sum_b[N];
  ICTC_DEGREES(l, N) sum_w[l] = sum_b[l] = own.w[l] = own.b[l] = 0.f;
  if (HOLD && c0 < C) own.load(a, c0);

  if constexpr (BULK) {
    if (g.thread == 0)
      for (int s = 0; s < a.stages; ++s) tc::mbar_init(full + s, 1);
    g.sync();
  }
  for (int s = 0; s + 1 < a.stages; ++s) fetch(first + s * stride, s);
  int stage = 0, waited = 0;
  uint32_t parity = 0;
  int64_t t = first;
  for (; t < tiles; t += stride) {
    if constexpr (BULK) {
      const bool landed =
          g.sync_all(g.thread != 0 || (a.wait_ns != 0 && tc::mbar_wait(full + stage, parity, a.wait_ns)));
      if (!landed) break;
      ++waited;
    } else if (a.stages == 1) {
      g.sync();
      fetch(t, 0);
      copies_wait(0);
      g.sync();
    } else {
      copies_wait(a.stages - 2);
      g.sync();       // the tile is there, and everyone has left the stage that is filled next
      fetch(t + (a.stages - 1) * stride, stage == 0 ? a.stages - 1 : stage - 1);
    }
    // The stage that the last tile left is filled once its rows have been read out.
    auto refill = [&]() {
      if constexpr (BULK) {
        if (g.thread == 0) {
          bulk_read_wait();
          fetch(t + (a.stages - 1) * stride, stage == 0 ? a.stages - 1 : stage - 1);
        }
      }
    };
    float* tile = ring + stage * a.stage_floats;
    const int64_t row0 = t * a.per;
    const int rows = (int)(a.rows - row0 < a.per ? a.rows - row0 : a.per);
    bool real[R];
    ICTC_ROWS(r, R) real[r] = sub + r * apart < rows;
    const int step = apart * W;
    auto at = [&](int s) { return tile + a.at[s] + sub * W; };
    auto get = [&](V& x, int s, int c) { load<L, LAYOUT, R>(x, at(s), step, C, c); };
    auto put = [&](const V& x, int s, int c) { store<L, LAYOUT, R>(x, at(s), step, C, c); };
    auto rate = [&](float sum, int l) { return rsqrtf(fmaf(sum, a.inv[l], a.eps)); };
    // a value per row, degree and channel (the widest rows leave no room for these)
    auto channel = [&](int s, int r, int l, int c) {
      return HOLD ? tile[a.at[s] + (sub + r * apart) * width + l * C + c] : __ldg(a.in[s] + row0 * width + l * C + c);
    };
    // a row's rates, four floats
    auto keep = [&](float* to, int r, const float* x) {
      *reinterpret_cast<float4*>(to + (row0 + sub + r * apart) * 4) =
          make_float4(x[0], N > 1 ? x[1 % N] : 0.f, N > 2 ? x[2 % N] : 0.f, N > 3 ? x[3 % N] : 0.f);
    };
    // sigma(gate) of a channel, per row and degree
    auto sigma = [&](float (&s)[R][N], int c) {
      ICTC_ROWS(r, R) ICTC_DEGREES(l, N)
        s[r][l] = a.in[kGate] ? sigmoid(channel(kGate, r, l, c)) : 1.f;
    };
    auto weights = [&](int c) {
      if constexpr (!HOLD) own.load(a, c);
    };
    // HOLD false: a phase starts by reading again what an earlier one read or wrote
    auto again = [&](V& x, int s, int c) {
      if constexpr (!HOLD) get(x, s, c);
    };

    if constexpr (MODE == kForward) {
      V y, h;
      float r1[R][N], s[R * N];
      if constexpr (BRANCH) {
        ICTC_ROWS(r, R) ICTC_DEGREES(l, N) s[r * N + l] = 0.f;
        each([&](int c) {
          get(y, kY, c);
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N) ICTC_PARTS(e, l) s[r * N + l] = fmaf(y.v[r][e], y.v[r][e], s[r * N + l]);
        });
        refill();
        g.sum(s);
        ICTC_ROWS(r, R) ICTC_DEGREES(l, N) r1[r][l] = rate(s[r * N + l], l);
        if (a.r1_out && c0 == 0) ICTC_ROWS(r, R) if (real[r]) keep(a.r1_out, r, r1[r]);
      } else {
        refill();
      }
      ICTC_ROWS(r, R) ICTC_DEGREES(l, N) s[r * N + l] = 0.f;
      each([&](int c) {
        get(h, kH, c);
        if constexpr (BRANCH) {
          again(y, kY, c);
          weights(c);
          float sg[R][N];
          sigma(sg, c);
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
            const float f = own.w[l] * sg[r][l] * r1[r][l];
            ICTC_PARTS(e, l) h.v[r][e] = fmaf(f, y.v[r][e], h.v[r][e]);
          }
          put(h, kH, c);
        }
        ICTC_ROWS(r, R) ICTC_DEGREES(l, N) ICTC_PARTS(e, l) s[r * N + l] = fmaf(h.v[r][e], h.v[r][e], s[r * N + l]);
      });
      if (a.norm) {
        g.sum(s);
        ICTC_ROWS(r, R) ICTC_DEGREES(l, N) s[r * N + l] = rate(s[r * N + l], l);
        if (a.r2_out && c0 == 0) ICTC_ROWS(r, R) if (real[r]) keep(a.r2_out, r, s + r * N);
        each([&](int c) {
          again(h, kH, c);
          weights(c);
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
            const float f = own.b[l] * s[r * N + l];
            ICTC_PARTS(e, l) h.v[r][e] *= f;
          }
          put(h, kY, c);
        });
      }
    } else {
      V h, q, T, y;
      float r1[R][N], r2[R][N], kq[R * N];
      ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
        const int from = (sub + r * apart) * 4 + l;
        r1[r][l] = BRANCH ? tile[a.at[kR1] + from] : 0.f;
        r2[r][l] = a.norm ? tile[a.at[kR2] + from] : 0.f;
        kq[r * N + l] = 0.f;
      }
      if (a.norm) {
        each([&](int c) {
          get(h, kH, c);
          get(q, kQ, c);
          weights(c);
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
            float s = 0.f;
            ICTC_PARTS(e, l) s = fmaf(r2[r][l] * h.v[r][e], q.v[r][e], s);
            kq[r * N + l] = fmaf(own.b[l], s, kq[r * N + l]);
            if (MODE == kBackward && real[r]) {
              if constexpr (HOLD) sum_b[l] += s;
              else if (a.partial) acc[width + l * C + c] += s;
            }
          }
        });
        refill();
        g.sum(kq);
        ICTC_ROWS(r, R) ICTC_DEGREES(l, N) kq[r * N + l] *= a.inv[l];      // <k, b q>
      }
      if (!a.norm) refill();
      // T = p + r2 (b q - k <k, b q>)
      auto total = [&](int c) {
        if constexpr (BRANCH) {
          if (a.in[kP]) get(T, kP, c);
          else zero(T);
        } else {
          zero(T);
        }
        weights(c);
        if (a.norm) {
          again(h, kH, c);
          again(q, kQ, c);
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
            const float f = r2[r][l] * kq[r * N + l];
            ICTC_PARTS(e, l) T.v[r][e] = fmaf(r2[r][l], own.b[l] * q.v[r][e] - f * h.v[r][e], T.v[r][e]);
          }
        }
      };
      if constexpr (MODE == kBackward) {
        float nT[R * N];
        float sg[R][N];
        ICTC_ROWS(r, R) ICTC_DEGREES(l, N) nT[r * N + l] = 0.f;
        each([&](int c) {
          total(c);
          if (a.out[BRANCH ? kP : kQ] || !HOLD) put(T, BRANCH ? kP : kQ, c);
          if constexpr (BRANCH) {
            get(y, kY, c);
            sigma(sg, c);
            ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
              float S = 0.f;
              ICTC_PARTS(e, l) S = fmaf(r1[r][l] * y.v[r][e], T.v[r][e], S);
              nT[r * N + l] = fmaf(own.w[l] * sg[r][l], S, nT[r * N + l]);
              if (real[r]) {
                if (a.gate_out)
                  a.gate_out[(row0 + sub + r * apart) * width + l * C + c] =
                      own.w[l] * sg[r][l] * (1.f - sg[r][l]) * S;
                if constexpr (HOLD) sum_w[l] = fmaf(sg[r][l], S, sum_w[l]);
                else if (a.partial) acc[l * C + c] += sg[r][l] * S;
              }
            }
          }
        });
        if constexpr (BRANCH) {
          if (a.out[kY]) {
            g.sum(nT);
            each([&](int c) {
              if constexpr (!HOLD) {
                get(T, kP, c);
                get(y, kY, c);
                weights(c);
                sigma(sg, c);
              }
              ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
                const float f = r1[r][l] * nT[r * N + l] * a.inv[l], aw = own.w[l] * sg[r][l];
                ICTC_PARTS(e, l) y.v[r][e] = r1[r][l] * (aw * T.v[r][e] - f * y.v[r][e]);
              }
              put(y, kY, c);
            });
          }
        }
      } else {
        V be, tau;
        float sg[R][N], dt[R][N], k[4 * R * N];      // <n,aT>, <n,be>, <aT,be>, <n,zT>
        auto dots = [&](int c) {
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N)
            dt[r][l] = a.in[kGateDot] ? channel(kGateDot, r, l, c) : 0.f;
        };
        if constexpr (BRANCH) {
#pragma unroll
          for (int i = 0; i < 4 * R * N; ++i) k[i] = 0.f;
          each([&](int c) {
            total(c);
            if constexpr (!HOLD) put(T, kP, c);
            get(y, kY, c);
            if (a.in[kBe]) get(be, kBe, c);
            else zero(be);
            sigma(sg, c);
            dots(c);
            ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
              float S = 0.f, nb = 0.f, tb = 0.f;
              ICTC_PARTS(e, l) {
                const float n = r1[r][l] * y.v[r][e];
                S = fmaf(n, T.v[r][e], S);
                nb = fmaf(n, be.v[r][e], nb);
                tb = fmaf(T.v[r][e], be.v[r][e], tb);
              }
              float* kk = k + 4 * (r * N + l);
              const float aw = own.w[l] * sg[r][l];
              kk[0] = fmaf(aw, S, kk[0]);
              kk[1] += nb;
              kk[2] = fmaf(aw, tb, kk[2]);
              kk[3] = fmaf(dt[r][l] * aw * (1.f - sg[r][l]), S, kk[3]);
            }
          });
          g.sum(k);
          ICTC_ROWS(r, R) ICTC_DEGREES(l, N)
#pragma unroll
            for (int i = 0; i < 4; ++i) k[4 * (r * N + l) + i] *= a.inv[l];
        }
        float kt[2 * R * N];                         // <k,tau>, <bq,tau>
#pragma unroll
        for (int i = 0; i < 2 * R * N; ++i) kt[i] = 0.f;
        each([&](int c) {
          if (a.in[kAl]) get(tau, kAl, c);
          else zero(tau);
          weights(c);
          if constexpr (BRANCH) {
            if constexpr (!HOLD) {
              get(T, kP, c);
              get(y, kY, c);
              if (a.in[kBe]) get(be, kBe, c);
              else zero(be);
              sigma(sg, c);
              dots(c);
            }
            ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
              const float* kk = k + 4 * (r * N + l);
              const float r0 = r1[r][l], nT = kk[0], nb = kk[1], Tb = kk[2], nz = kk[3];
              const float slope = sg[r][l] * (1.f - sg[r][l]), aw = own.w[l] * sg[r][l];
              const float z = dt[r][l] * own.w[l] * slope;
              // gy = cn n + ct T + cb be
              const float cn = r0 * (r0 * (3.f * nT * nb - Tb) - nz), ct = r0 * (z - r0 * nb * aw), cb = -r0 * r0 * nT;
              float S = 0.f, tb = 0.f;
              ICTC_PARTS(e, l) {
                const float n = r0 * y.v[r][e], tv = T.v[r][e], bv = be.v[r][e];
                S = fmaf(n, tv, S);
                tb = fmaf(tv, bv, tb);
                tau.v[r][e] += aw * r0 * (bv - nb * n) + z * n;
                y.v[r][e] = cn * n + ct * tv + cb * bv;
              }
              const float ga = r0 * (tb - nb * S);
              if (real[r]) {
                if (a.gate_out)
                  a.gate_out[(row0 + sub + r * apart) * width + l * C + c] =
                      own.w[l] * slope * (ga + dt[r][l] * (1.f - 2.f * sg[r][l]) * S);
                const float gw = sg[r][l] * ga + dt[r][l] * slope * S;
                if constexpr (HOLD) sum_w[l] += gw;
                else if (a.partial) acc[l * C + c] += gw;
              }
            }
            if (a.out[kY]) put(y, kY, c);
          }
          if (BRANCH || !HOLD) put(tau, kAl, c);
          if (a.norm) {
            again(h, kH, c);
            again(q, kQ, c);
            ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
              float* kk = kt + 2 * (r * N + l);
              float qt = 0.f;
              ICTC_PARTS(e, l) {
                kk[0] = fmaf(r2[r][l] * h.v[r][e], tau.v[r][e], kk[0]);
                qt = fmaf(q.v[r][e], tau.v[r][e], qt);
              }
              kk[1] = fmaf(own.b[l], qt, kk[1]);
            }
          }
        });
        if (a.norm) {
          g.sum(kt);
          each([&](int c) {
            if constexpr (!HOLD) {
              get(tau, kAl, c);
              get(h, kH, c);
              get(q, kQ, c);
              weights(c);
            }
            ICTC_ROWS(r, R) ICTC_DEGREES(l, N) {
              const float inv = a.inv[l], r0 = r2[r][l], b = own.b[l];
              const float kt0 = kt[2 * (r * N + l)] * inv, qt = kt[2 * (r * N + l) + 1] * inv, kq0 = kq[r * N + l];
              const float ck = r0 * r0 * (3.f * kq0 * kt0 - qt);
              float gb = 0.f;
              ICTC_PARTS(e, l) {
                const float kv = r0 * h.v[r][e], qv = q.v[r][e], tv = tau.v[r][e];
                const float down = r0 * (tv - kt0 * kv);
                gb = fmaf(qv, down, gb);
                q.v[r][e] = b * down;
                h.v[r][e] = ck * kv - r0 * r0 * (kt0 * b * qv + kq0 * tv);
              }
              if (real[r]) {
                if constexpr (HOLD) sum_b[l] += gb;
                else if (a.partial) acc[width + l * C + c] += gb;
              }
            }
            put(h, kH, c);
            put(q, kQ, c);
          });
        }
      }
    }
    // The rows leave (forward: u from y's place).
    if constexpr (BULK) {
      tc::fence_async_smem();
      g.sync();
      if (g.thread == 0) {
#pragma unroll
        for (int s = 0; s < 6; ++s)
          if (a.out[s]) bulk_store(a.out[s] + row0 * W, tile + a.at[s], rows * W * 4);
        bulk_commit();
      }
      if (stage + 1 == a.stages) parity ^= 1;
    } else {
      g.sync();
#pragma unroll
      for (int s = 0; s < 6; ++s) {
        if (a.out[s] == nullptr) continue;
        float* dst = a.out[s] + row0 * W;
        const float* src = tile + a.at[s];
        const int count = rows * W;
        int i = 0;
        if (a.wide >> (16 + s) & 1u) {
          for (int j = 4 * g.thread; j + 3 < count; j += 4 * g.threads)
            *reinterpret_cast<float4*>(dst + j) = *reinterpret_cast<const float4*>(src + j);
          i = count & ~3;
        }
        for (i += g.thread; i < count; i += g.threads) dst[i] = src[i];
      }
    }
    stage = stage + 1 == a.stages ? 0 : stage + 1;
  }
  if constexpr (BULK) {
    // A copy did not land in time: report it, let those in flight end, and leave NaN in all rows that are
    // left and in the weights' gradients (unwritten memory could pass for a result).
    if (t < tiles) {
      if (g.thread == 0) {
        bool drained = true;
        for (int j = waited; j < issued; ++j)
          drained = tc::mbar_wait(full + j % a.stages, (j / a.stages) & 1, kWaitNs) && drained;
        atomicMax(a.status, drained ? 1 : 3);
      }
      const float nan = __int_as_float(0x7fffffff);
#pragma unroll 1
      for (; t < tiles; t += stride) {
        const int64_t row0 = t * a.per;
        const int rows = (int)(a.rows - row0 < a.per ? a.rows - row0 : a.per);
        // (the loop's form moves the registers of the code before it: rolled, the norm alone takes 53 us instead of 49
        // for 50,000 rows of C132/lmax 1; unrolled, the forward with a branch 93 us instead of 91)
#pragma unroll (BRANCH ? 1 : 9)
        for (int s = 0; s < 9; ++s) {
          float* to = s < 6 ? a.out[s] : s == 6 ? a.gate_out : s == 7 ? a.r1_out : a.r2_out;
          const int wd = s < 6 ? W : s == 6 ? width : 4;
          if (to == nullptr) continue;
#pragma unroll 1
          for (int i = g.thread; i < rows * wd; i += g.threads) to[row0 * wd + i] = nan;
        }
      }
      if constexpr (MODE != kForward) {
        ICTC_DEGREES(l, N) sum_w[l] = sum_b[l] = nan;
      }
    }
    if (g.thread == 0) bulk_read_wait();      // shared memory outlives the stores that read it
  }
  if (a.partial == nullptr) return;
  // Sums of the block's groups (and of a warp's rows side by side), in order.
  __syncthreads();
  const int beside = 32 * a.warps / a.lanes;      // rows side by side in a group
  if constexpr (HOLD) {
    float* mine = shared + (int64_t)(g.id * beside + sub) * 2 * width;
    if (c0 < C) ICTC_DEGREES(l, N) {
      mine[l * C + c0] = sum_w[l];
      mine[width + l * C + c0] = sum_b[l];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < 2 * width; i += blockDim.x) {
    float s = 0.f;
    if constexpr (HOLD) {
      for (int k = 0; k < groups * beside; ++k) s += shared[(int64_t)k * 2 * width + i];
    } else {
      for (int k = 0; k < groups; ++k)
        s += shared[k * a.group_floats + a.stages * a.stage_floats + 2 * a.warps * kScratch + kBarrierFloats + i];
    }
    a.partial[(int64_t)blockIdx.x * 2 * width + i] = s;
  }
}

template <int L, int LAYOUT, int MODE, bool BRANCH, bool HOLD, bool BULK>
cudaError_t launch_one(const BlockArgs& a, const Shape& s, int grid, int shared_bytes, cudaStream_t stream) {
  auto kernel = block_kernel<L, LAYOUT, MODE, BRANCH, HOLD, BULK>;
  static std::atomic<bool> ready[kMaxDevices];   // shared-memory limit raised on this device
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device >= kMaxDevices || !ready[device].load(std::memory_order_relaxed)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedLimit);
    if (err != cudaSuccess) return err;
    if (device < kMaxDevices) ready[device].store(true, std::memory_order_relaxed);
  }
  kernel<<<grid, s.groups * s.warps * 32, shared_bytes, stream>>>(a);
  return cudaGetLastError();
}

template <int L, int LAYOUT, int MODE, bool BRANCH>
cudaError_t launch_copies(const BlockArgs& a, const Shape& s, int grid, int bytes, cudaStream_t stream) {
  if (!s.hold) return launch_one<L, LAYOUT, MODE, BRANCH, false, false>(a, s, grid, bytes, stream);
  return s.bulk ? launch_one<L, LAYOUT, MODE, BRANCH, true, true>(a, s, grid, bytes, stream)
                : launch_one<L, LAYOUT, MODE, BRANCH, true, false>(a, s, grid, bytes, stream);
}
template <int L, int MODE, bool BRANCH>
cudaError_t launch_layout(const BlockArgs& a, const Shape& s, int grid, int bytes, int layout, cudaStream_t stream) {
  return layout == kMulIr ? launch_copies<L, kMulIr, MODE, BRANCH>(a, s, grid, bytes, stream)
                          : launch_copies<L, kIrMul, MODE, BRANCH>(a, s, grid, bytes, stream);
}
template <int MODE, bool BRANCH>
cudaError_t launch_degree(const BlockArgs& a, const Shape& s, int grid, int bytes, int lmax, int layout,
                          cudaStream_t stream) {
  switch (lmax) {
    case 0: return launch_layout<0, MODE, BRANCH>(a, s, grid, bytes, layout, stream);
    case 1: return launch_layout<1, MODE, BRANCH>(a, s, grid, bytes, layout, stream);
    case 2: return launch_layout<2, MODE, BRANCH>(a, s, grid, bytes, layout, stream);
    default: return launch_layout<3, MODE, BRANCH>(a, s, grid, bytes, layout, stream);
  }
}
template <int MODE>
cudaError_t launch_mode(const BlockArgs& a, const Shape& s, int grid, int bytes, int lmax, int layout, bool branch,
                        cudaStream_t stream) {
  return branch ? launch_degree<MODE, true>(a, s, grid, bytes, lmax, layout, stream)
                : launch_degree<MODE, false>(a, s, grid, bytes, lmax, layout, stream);
}

// One per mode, each in a file of its own (they compile side by side).
cudaError_t launch_forward(const BlockArgs&, const Shape&, int, int, int, int, bool, cudaStream_t);
cudaError_t launch_backward(const BlockArgs&, const Shape&, int, int, int, int, bool, cudaStream_t);
cudaError_t launch_second(const BlockArgs&, const Shape&, int, int, int, int, bool, cudaStream_t);

}  // namespace block_norm
}  // namespace ictc
