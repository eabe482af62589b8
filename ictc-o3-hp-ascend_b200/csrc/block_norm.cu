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
// All three are bound by the rows they read and write.  A group of lanes owns one row, a lane
// whole channels (four neighbours where C allows), so that sums over components and per-channel
// values stay in a lane and only the degrees' scalar products cross lanes.  Rows are brought into shared
// memory by asynchronous copies one tile ahead, worked on in place and written back as
// contiguous rows: a lane's channels lie 2l+1 values apart, an odd stride, which shared memory
// serves without conflicts and device memory would not.  Weight gradients are summed per
// group in shared memory, per block, and over blocks by a second kernel, in a fixed order.
#include "ictc_common.cuh"
#include "ictc_cuda.h"

#include <atomic>
#include <cstdio>

void ictc_set_error(const char* fmt, const char* detail);

namespace ictc {
namespace {

constexpr int kMaxL = 3;
constexpr int kMaxGroupWarps = 8;
// Warps per block: the second derivatives keep up to 170 values per lane.
__host__ __device__ constexpr int max_warps(int mode) { return mode == 2 ? 8 : 16; }
constexpr int kMaxDevices = 64;
constexpr int kSharedLimit = 227 * 1024;
constexpr int kSharedBudget = 200 * 1024; // of 227 KB: the rest serves gates and weights as L1

enum Mode : int { kForward = 0, kBackward = 1, kSecond = 2 };

__host__ __device__ constexpr int slots_of(int mode, bool branch) {
  return mode == kForward ? (branch ? 2 : 1) : mode == kBackward ? (branch ? 4 : 2) : (branch ? 6 : 3);
}

struct BlockArgs {
  const float* in[6];       // rows staged in shared memory, by slot (null: zeros)
  float* out[6];            // where a slot goes afterwards (null: nowhere)
  const float* gate;        // [N, (L+1) C] or null
  const float* gate_dot;    // cotangent of dgate, or null
  float* gate_out;          // dgate / its adjoint, or null
  const float* post;        // [L+1, C] or null (1)
  const float* scale;       // [L+1, C] or null (1)
  const float* pre;         // [L+1, C] or null (1)
  float* r1;                // [N, L+1], written by the forward, read by the others
  float* r2;
  float* partial;           // [blocks][2][(L+1) C] weight-gradient sums, or null
  int64_t rows;
  int channels;
  int lanes;                // lanes per row
  int warps;                // warps per group
  int stages;
  int wide;                 // rows move 16 bytes at a time
  int vec_gate;             // gate arrays and weights may be read 16 bytes at a time
  int norm;                 // u (or its cotangent) takes part
  float eps;
};

// Slots: forward y, h; backward y, h', p, q; second y, h', p, q, al, be.  Without a branch
// (norm alone): h;  h', q;  h', q, al.
template <int V> struct Reg { float v[V]; };

template <int V>
__device__ __forceinline__ Reg<V> lds(const float* p) {
  Reg<V> r;
  if constexpr (V == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    r.v[0] = t.x; r.v[1] = t.y; r.v[2] = t.z; r.v[3] = t.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <int V>
__device__ __forceinline__ void sts(float* p, const Reg<V>& r) {
  if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
  else *p = r.v[0];
}
template <int V>
__device__ __forceinline__ Reg<V> ldg(const float* p, bool vec) {
  Reg<V> r;
  if constexpr (V == 4) {
    if (vec) {
      const float4 t = __ldg(reinterpret_cast<const float4*>(p));
      r.v[0] = t.x; r.v[1] = t.y; r.v[2] = t.z; r.v[3] = t.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r.v[i] = __ldg(p + i);
    }
  } else {
    r.v[0] = __ldg(p);
  }
  return r;
}
template <int V>
__device__ __forceinline__ void stg(float* p, const Reg<V>& r, bool vec) {
  if constexpr (V == 4) {
    if (vec) {
      *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] = r.v[i];
}

__device__ __forceinline__ void copy_async16(float* dst, const float* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_async4(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait(int ahead) {
  if (ahead >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (ahead == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (ahead == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A group: one warp (holding 32 / lanes rows) or several warps of one row.
struct Group {
  int id;        // in the block
  int thread;    // in the group
  int threads;
  int lanes;     // per row
  float* scratch;

  __device__ __forceinline__ void sync() const {
    if (threads == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(threads) : "memory");
  }
  // Sums of N values over a row's lanes, in a fixed order, in every lane.
  template <int N>
  __device__ __forceinline__ void sum(float (&x)[N]) const {
    const int top = threads == 32 ? lanes : 32;
    for (int o = top >> 1; o; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
    }
    if (threads > 32) {
      if ((thread & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[(thread >> 5) * 16 + i] = x[i];
      }
      sync();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float s = 0.f;
        for (int w = 0; w < threads >> 5; ++w) s += scratch[w * 16 + i];
        x[i] = s;
      }
      sync();
    }
  }
};

// V channels of degree l in registers: x[m].v[i] (channel c + i).  In the [C][2l+1] layout the
// V (2l+1) values are contiguous and move as 2l+1 vectors.
template <int l, int LAYOUT, int V>
__device__ __forceinline__ void load_degree(Reg<V> (&x)[2 * l + 1], const float* row, int C, int c) {
  constexpr int M = 2 * l + 1;
  const float* p = row + C * l * l + (LAYOUT == kMulIr ? c * M : c);
  if constexpr (LAYOUT == kMulIr) {
    float flat[V * M];
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const Reg<V> t = lds<V>(p + j * V);
#pragma unroll
      for (int i = 0; i < V; ++i) flat[j * V + i] = t.v[i];
    }
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < V; ++i) x[m].v[i] = flat[i * M + m];
  } else {
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] = lds<V>(p + m * C);
  }
}
template <int l, int LAYOUT, int V>
__device__ __forceinline__ void store_degree(const Reg<V> (&x)[2 * l + 1], float* row, int C, int c) {
  constexpr int M = 2 * l + 1;
  float* p = row + C * l * l + (LAYOUT == kMulIr ? c * M : c);
  if constexpr (LAYOUT == kMulIr) {
    float flat[V * M];
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < V; ++i) flat[i * M + m] = x[m].v[i];
#pragma unroll
    for (int j = 0; j < M; ++j) {
      Reg<V> t;
#pragma unroll
      for (int i = 0; i < V; ++i) t.v[i] = flat[j * V + i];
      sts<V>(p + j * V, t);
    }
  } else {
#pragma unroll
    for (int m = 0; m < M; ++m) sts<V>(p + m * C, x[m]);
  }
}

// post scale of V channels.
template <int V>
__device__ __forceinline__ Reg<V> weight_of(const BlockArgs& a, int at) {
  Reg<V> w;
#pragma unroll
  for (int i = 0; i < V; ++i) w.v[i] = 1.f;
  if (a.post) w = ldg<V>(a.post + at, a.vec_gate);
  if (a.scale) {
    const Reg<V> s = ldg<V>(a.scale + at, a.vec_gate);
#pragma unroll
    for (int i = 0; i < V; ++i) w.v[i] *= s.v[i];
  }
  return w;
}
template <int V>
__device__ __forceinline__ Reg<V> pre_of(const BlockArgs& a, int at) {
  if (a.pre) return ldg<V>(a.pre + at, a.vec_gate);
  Reg<V> w;
#pragma unroll
  for (int i = 0; i < V; ++i) w.v[i] = 1.f;
  return w;
}
template <int V>
__device__ __forceinline__ Reg<V> sigma_of(const BlockArgs& a, int64_t row, int width, int at) {
  Reg<V> s;
#pragma unroll
  for (int i = 0; i < V; ++i) s.v[i] = 1.f;
  if (a.gate) {
    const Reg<V> g = ldg<V>(a.gate + row * width + at, a.vec_gate);
#pragma unroll
    for (int i = 0; i < V; ++i) s.v[i] = 1.f / (1.f + expf(-g.v[i]));
  }
  return s;
}

template <int L, int LAYOUT, int V, int MODE, bool BRANCH>
__device__ __forceinline__ void work_row(const BlockArgs& a, const Group& g, float* tile, int64_t slot, int64_t row,
                                         bool real, int u0, float* acc_w, float* acc_b) {
  constexpr int N = L + 1;
  const int C = a.channels, units = C / V, width = N * C;
  float* y = tile;                                        // slot 0
  float* h = BRANCH ? tile + slot : tile;                 // slot 1, or 0 without a branch
  if constexpr (MODE == kForward) {
    float r1[N], s[N];
    if constexpr (BRANCH) {
#pragma unroll
      for (int l = 0; l < N; ++l) s[l] = 0.f;
      for (int u = u0; u < units; u += g.lanes)
        static_for<N>([&](auto lc) {
          constexpr int l = decltype(lc)::value;
          Reg<V> x[2 * l + 1];
          load_degree<l, LAYOUT, V>(x, y, C, u * V);
#pragma unroll
          for (int m = 0; m < 2 * l + 1; ++m)
#pragma unroll
            for (int i = 0; i < V; ++i) s[l] = fmaf(x[m].v[i], x[m].v[i], s[l]);
        });
      g.sum(s);
#pragma unroll
      for (int l = 0; l < N; ++l) r1[l] = 1.f / sqrtf(s[l] / (float)(C * (2 * l + 1)) + a.eps);
    }
#pragma unroll
    for (int l = 0; l < N; ++l) s[l] = 0.f;
    for (int u = u0; u < units; u += g.lanes)
      static_for<N>([&](auto lc) {
        constexpr int l = decltype(lc)::value;
        Reg<V> xh[2 * l + 1];
        load_degree<l, LAYOUT, V>(xh, h, C, u * V);
        if constexpr (BRANCH) {
          Reg<V> xy[2 * l + 1];
          load_degree<l, LAYOUT, V>(xy, y, C, u * V);
          Reg<V> w = weight_of<V>(a, l * C + u * V);
          const Reg<V> sg = sigma_of<V>(a, row, width, l * C + u * V);
#pragma unroll
          for (int i = 0; i < V; ++i) w.v[i] *= sg.v[i] * r1[l];
#pragma unroll
          for (int m = 0; m < 2 * l + 1; ++m)
#pragma unroll
            for (int i = 0; i < V; ++i) xh[m].v[i] = fmaf(w.v[i], xy[m].v[i], xh[m].v[i]);
          store_degree<l, LAYOUT, V>(xh, h, C, u * V);
        }
#pragma unroll
        for (int m = 0; m < 2 * l + 1; ++m)
#pragma unroll
          for (int i = 0; i < V; ++i) s[l] = fmaf(xh[m].v[i], xh[m].v[i], s[l]);
      });
    if (a.norm) {
      g.sum(s);
      float r2[N];
#pragma unroll
      for (int l = 0; l < N; ++l) r2[l] = 1.f / sqrtf(s[l] / (float)(C * (2 * l + 1)) + a.eps);
      for (int u = u0; u < units; u += g.lanes)
        static_for<N>([&](auto lc) {
          constexpr int l = decltype(lc)::value;
          Reg<V> x[2 * l + 1];
          load_degree<l, LAYOUT, V>(x, h, C, u * V);
          const Reg<V> b = pre_of<V>(a, l * C + u * V);
#pragma unroll
          for (int m = 0; m < 2 * l + 1; ++m)
#pragma unroll
            for (int i = 0; i < V; ++i) x[m].v[i] *= b.v[i] * r2[l];
          store_degree<l, LAYOUT, V>(x, y, C, u * V);      // over y (over h without a branch)
        });
      if (a.r2 && real && u0 == 0)
#pragma unroll
        for (int l = 0; l < N; ++l) a.r2[row * N + l] = r2[l];
    }
    if (BRANCH && a.r1 && real && u0 == 0)
#pragma unroll
      for (int l = 0; l < N; ++l) a.r1[row * N + l] = r1[l];
  } else {
    float* p = tile + 2 * slot;                            // only with a branch
    float* q = BRANCH ? tile + 3 * slot : tile + slot;
    float r1[N], r2[N], k2[N];
#pragma unroll
    for (int l = 0; l < N; ++l) {
      r1[l] = BRANCH && real ? a.r1[row * N + l] : 0.f;
      r2[l] = a.norm && real ? a.r2[row * N + l] : 0.f;
      k2[l] = 0.f;
    }
    if (a.norm) {
      for (int u = u0; u < units; u += g.lanes)
        static_for<N>([&](auto lc) {
          constexpr int l = decltype(lc)::value;
          Reg<V> xh[2 * l + 1], xq[2 * l + 1];
          load_degree<l, LAYOUT, V>(xh, h, C, u * V);
          load_degree<l, LAYOUT, V>(xq, q, C, u * V);
          const Reg<V> b = pre_of<V>(a, l * C + u * V);
          Reg<V> hq;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            hq.v[i] = 0.f;
#pragma unroll
            for (int m = 0; m < 2 * l + 1; ++m) hq.v[i] = fmaf(xh[m].v[i], xq[m].v[i], hq.v[i]);
            k2[l] = fmaf(b.v[i], hq.v[i], k2[l]);
          }
          if (MODE == kBackward && acc_b) {
            float* at = acc_b + l * C + u * V;
            Reg<V> t = lds<V>(at);
#pragma unroll
            for (int i = 0; i < V; ++i) t.v[i] = fmaf(r2[l], hq.v[i], t.v[i]);
            sts<V>(at, t);
          }
        });
      g.sum(k2);
#pragma unroll
      for (int l = 0; l < N; ++l) k2[l] *= r2[l] / (float)(C * (2 * l + 1));      // <k, b q>
    }
    if constexpr (MODE == kBackward) {
      float k1[N];
#pragma unroll
      for (int l = 0; l < N; ++l) k1[l] = 0.f;
      for (int u = u0; u < units; u += g.lanes)
        static_for<N>([&](auto lc) {
          constexpr int l = decltype(lc)::value;
          constexpr int M = 2 * l + 1;
          const int at = l * C + u * V;
          Reg<V> T[M];
          if constexpr (BRANCH) load_degree<l, LAYOUT, V>(T, p, C, u * V);
          if (a.norm) {
            Reg<V> xh[M], xq[M];
            load_degree<l, LAYOUT, V>(xh, h, C, u * V);
            load_degree<l, LAYOUT, V>(xq, q, C, u * V);
            const Reg<V> b = pre_of<V>(a, at);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int i = 0; i < V; ++i) {
                const float t = r2[l] * (b.v[i] * xq[m].v[i] - r2[l] * xh[m].v[i] * k2[l]);
                T[m].v[i] = BRANCH ? T[m].v[i] + t : t;
              }
            store_degree<l, LAYOUT, V>(T, BRANCH ? p : q, C, u * V);
          }
          if constexpr (BRANCH) {
            Reg<V> xy[M];
            load_degree<l, LAYOUT, V>(xy, y, C, u * V);
            const Reg<V> w = weight_of<V>(a, at), sg = sigma_of<V>(a, row, width, at);
            Reg<V> S, dg;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              S.v[i] = 0.f;
#pragma unroll
              for (int m = 0; m < M; ++m) S.v[i] = fmaf(xy[m].v[i], T[m].v[i], S.v[i]);
              S.v[i] *= r1[l];
              k1[l] = fmaf(w.v[i] * sg.v[i], S.v[i], k1[l]);
              dg.v[i] = w.v[i] * sg.v[i] * (1.f - sg.v[i]) * S.v[i];
            }
            if (a.gate_out && real) stg<V>(a.gate_out + row * width + at, dg, a.vec_gate);
            if (acc_w) {
              Reg<V> t = lds<V>(acc_w + at);
#pragma unroll
              for (int i = 0; i < V; ++i) t.v[i] = fmaf(sg.v[i], S.v[i], t.v[i]);
              sts<V>(acc_w + at, t);
            }
          }
        });
      if constexpr (BRANCH) {
        if (a.out[0]) {
          g.sum(k1);
          for (int u = u0; u < units; u += g.lanes)
            static_for<N>([&](auto lc) {
              constexpr int l = decltype(lc)::value;
              constexpr int M = 2 * l + 1;
              const int at = l * C + u * V;
              const float f = k1[l] / (float)(C * M);
              Reg<V> T[M], xy[M];
              load_degree<l, LAYOUT, V>(T, p, C, u * V);
              load_degree<l, LAYOUT, V>(xy, y, C, u * V);
              Reg<V> w = weight_of<V>(a, at);
              const Reg<V> sg = sigma_of<V>(a, row, width, at);
#pragma unroll
              for (int i = 0; i < V; ++i) w.v[i] *= sg.v[i];
#pragma unroll
              for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < V; ++i)
                  xy[m].v[i] = r1[l] * (w.v[i] * T[m].v[i] - r1[l] * xy[m].v[i] * f);
              store_degree<l, LAYOUT, V>(xy, y, C, u * V);
            });
        }
      }
    } else {
      float* al = BRANCH ? tile + 4 * slot : tile + 2 * slot;
      float* be = tile + 5 * slot;
      float k[4 * N];      // <n,aT>, <n,be>, <aT,be>, <n,zT>
      if constexpr (BRANCH) {
#pragma unroll
        for (int l = 0; l < 4 * N; ++l) k[l] = 0.f;
        for (int u = u0; u < units; u += g.lanes)
          static_for<N>([&](auto lc) {
            constexpr int l = decltype(lc)::value;
            constexpr int M = 2 * l + 1;
            const int at = l * C + u * V;
            Reg<V> T[M];
            load_degree<l, LAYOUT, V>(T, p, C, u * V);
            if (a.norm) {
              Reg<V> xh[M], xq[M];
              load_degree<l, LAYOUT, V>(xh, h, C, u * V);
              load_degree<l, LAYOUT, V>(xq, q, C, u * V);
              const Reg<V> b = pre_of<V>(a, at);
#pragma unroll
              for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < V; ++i)
                  T[m].v[i] += r2[l] * (b.v[i] * xq[m].v[i] - r2[l] * xh[m].v[i] * k2[l]);
              store_degree<l, LAYOUT, V>(T, p, C, u * V);
            }
            Reg<V> xy[M], xb[M];
            load_degree<l, LAYOUT, V>(xy, y, C, u * V);
            load_degree<l, LAYOUT, V>(xb, be, C, u * V);
            const Reg<V> w = weight_of<V>(a, at), sg = sigma_of<V>(a, row, width, at);
            Reg<V> dt;
#pragma unroll
            for (int i = 0; i < V; ++i) dt.v[i] = 0.f;
            if (a.gate_dot && real) dt = ldg<V>(a.gate_dot + row * width + at, a.vec_gate);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float S = 0.f, yb = 0.f, tb = 0.f;
#pragma unroll
              for (int m = 0; m < M; ++m) {
                const float n = r1[l] * xy[m].v[i];
                S = fmaf(n, T[m].v[i], S);
                yb = fmaf(n, xb[m].v[i], yb);
                tb = fmaf(T[m].v[i], xb[m].v[i], tb);
              }
              const float aw = w.v[i] * sg.v[i];
              k[4 * l] = fmaf(aw, S, k[4 * l]);
              k[4 * l + 1] += yb;
              k[4 * l + 2] = fmaf(aw, tb, k[4 * l + 2]);
              k[4 * l + 3] = fmaf(dt.v[i] * w.v[i] * sg.v[i] * (1.f - sg.v[i]), S, k[4 * l + 3]);
            }
          });
        g.sum(k);
#pragma unroll
        for (int l = 0; l < 4 * N; ++l) k[l] /= (float)(C * (2 * (l / 4) + 1));
      }
      float kt[2 * N];
#pragma unroll
      for (int l = 0; l < 2 * N; ++l) kt[l] = 0.f;
      for (int u = u0; u < units; u += g.lanes)
        static_for<N>([&](auto lc) {
          constexpr int l = decltype(lc)::value;
          constexpr int M = 2 * l + 1;
          const int at = l * C + u * V;
          Reg<V> tau[M];
          load_degree<l, LAYOUT, V>(tau, al, C, u * V);
          if constexpr (BRANCH) {
            Reg<V> T[M], xy[M], xb[M];
            load_degree<l, LAYOUT, V>(T, p, C, u * V);
            load_degree<l, LAYOUT, V>(xy, y, C, u * V);
            load_degree<l, LAYOUT, V>(xb, be, C, u * V);
            const Reg<V> w = weight_of<V>(a, at), sg = sigma_of<V>(a, row, width, at);
            Reg<V> dt, gg, gw;
#pragma unroll
            for (int i = 0; i < V; ++i) dt.v[i] = 0.f;
            if (a.gate_dot && real) dt = ldg<V>(a.gate_dot + row * width + at, a.vec_gate);
            const float r = r1[l], nT = k[4 * l], nb = k[4 * l + 1], Tb = k[4 * l + 2], nz = k[4 * l + 3];
            // gy = cn n + ct T + cb be
            const float cn = r * (r * (3.f * nT * nb - Tb) - nz), cb = -r * r * nT;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float slope = sg.v[i] * (1.f - sg.v[i]);
              const float aw = w.v[i] * sg.v[i], z = dt.v[i] * w.v[i] * slope;
              const float ct = r * (z - r * nb * aw);
              float S = 0.f, tb = 0.f;
#pragma unroll
              for (int m = 0; m < M; ++m) {
                const float nv = r * xy[m].v[i], tv = T[m].v[i], bv = xb[m].v[i];
                S = fmaf(nv, tv, S);
                tb = fmaf(tv, bv, tb);
                tau[m].v[i] += aw * r * (bv - nb * nv) + z * nv;
                xy[m].v[i] = cn * nv + ct * tv + cb * bv;
              }
              const float ga = r * (tb - nb * S);
              gw.v[i] = sg.v[i] * ga + dt.v[i] * slope * S;
              gg.v[i] = w.v[i] * slope * (ga + dt.v[i] * (1.f - 2.f * sg.v[i]) * S);
            }
            store_degree<l, LAYOUT, V>(xy, y, C, u * V);
            store_degree<l, LAYOUT, V>(tau, al, C, u * V);
            if (a.gate_out && real) stg<V>(a.gate_out + row * width + at, gg, a.vec_gate);
            if (acc_w) {
              Reg<V> t = lds<V>(acc_w + at);
#pragma unroll
              for (int i = 0; i < V; ++i) t.v[i] += gw.v[i];
              sts<V>(acc_w + at, t);
            }
          }
          if (a.norm) {
            Reg<V> xh[M], xq[M];
            load_degree<l, LAYOUT, V>(xh, h, C, u * V);
            load_degree<l, LAYOUT, V>(xq, q, C, u * V);
            const Reg<V> b = pre_of<V>(a, at);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float qt = 0.f;
#pragma unroll
              for (int m = 0; m < M; ++m) {
                kt[2 * l] = fmaf(r2[l] * xh[m].v[i], tau[m].v[i], kt[2 * l]);
                qt = fmaf(xq[m].v[i], tau[m].v[i], qt);
              }
              kt[2 * l + 1] = fmaf(b.v[i], qt, kt[2 * l + 1]);
            }
          }
        });
      if (a.norm) {
        g.sum(kt);
        for (int u = u0; u < units; u += g.lanes)
          static_for<N>([&](auto lc) {
            constexpr int l = decltype(lc)::value;
            constexpr int M = 2 * l + 1;
            const int at = l * C + u * V;
            const float inv = 1.f / (float)(C * M);
            const float r = r2[l], kt0 = kt[2 * l] * inv, qt = kt[2 * l + 1] * inv, kq = k2[l];
            const float ck = r * r * (3.f * kq * kt0 - qt);
            Reg<V> tau[M], xh[M], xq[M];
            load_degree<l, LAYOUT, V>(tau, al, C, u * V);
            load_degree<l, LAYOUT, V>(xh, h, C, u * V);
            load_degree<l, LAYOUT, V>(xq, q, C, u * V);
            const Reg<V> b = pre_of<V>(a, at);
            Reg<V> gb;
#pragma unroll
            for (int i = 0; i < V; ++i) {
              gb.v[i] = 0.f;
#pragma unroll
              for (int m = 0; m < M; ++m) {
                const float kv = r * xh[m].v[i], qv = xq[m].v[i], tv = tau[m].v[i];
                const float down = r * (tv - kt0 * kv);
                gb.v[i] = fmaf(qv, down, gb.v[i]);
                xq[m].v[i] = b.v[i] * down;
                xh[m].v[i] = ck * kv - r * r * (kt0 * b.v[i] * qv + kq * tv);
              }
            }
            store_degree<l, LAYOUT, V>(xh, h, C, u * V);
            store_degree<l, LAYOUT, V>(xq, q, C, u * V);
            if (acc_b) {
              Reg<V> t = lds<V>(acc_b + at);
#pragma unroll
              for (int i = 0; i < V; ++i) t.v[i] += gb.v[i];
              sts<V>(acc_b + at, t);
            }
          });
      }
    }
  }
}

template <int L, int LAYOUT, int V, int MODE, bool BRANCH>
__global__ void __launch_bounds__(32 * max_warps(MODE)) block_kernel(const __grid_constant__ BlockArgs a) {
  extern __shared__ __align__(16) float shared[];
  constexpr int N = L + 1, SLOTS = slots_of(MODE, BRANCH);
  const int C = a.channels, W = C * N * N;
  Group g;
  g.threads = 32 * a.warps;
  g.id = threadIdx.x / g.threads;
  g.thread = threadIdx.x % g.threads;
  g.lanes = a.lanes;
  const int groups = blockDim.x / g.threads;
  const int per = a.warps == 1 ? 32 / a.lanes : 1;             // rows of a tile
  const int slot = (per * W + 3) & ~3;                         // floats of one staged tensor
  const int sums = a.partial ? 2 * N * C : 0;                  // floats of one row's weight sums
  const int sums4 = (per * sums + 3) & ~3;
  float* ring = shared + (int64_t)g.id * (a.stages * SLOTS * slot + sums4 + 16 * kMaxGroupWarps);
  float* acc = ring + a.stages * SLOTS * slot;
  g.scratch = acc + sums4;
  const int mine = g.thread / a.lanes;                         // this lane's row in the tile (0 for several warps)
  const int u0 = g.thread % a.lanes;
  for (int i = g.thread; i < per * sums; i += g.threads) acc[i] = 0.f;
  const int64_t tiles = (a.rows + per - 1) / per;
  const int64_t first = (int64_t)blockIdx.x * groups + g.id, stride = (int64_t)gridDim.x * groups;

  auto fetch = [&](int64_t t, int stage) {
    if (t < tiles) {
      const int64_t row0 = t * per;
      const int count = (int)(a.rows - row0 < per ? a.rows - row0 : per) * W;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        float* dst = ring + (stage * SLOTS + s) * slot;
        const float* src = a.in[s];
        if (src == nullptr) {
          for (int i = g.thread; i < per * W; i += g.threads) dst[i] = 0.f;
          continue;
        }
        src += row0 * W;
        if (a.wide) {
          for (int i = 4 * g.thread; i < count; i += 4 * g.threads) copy_async16(dst + i, src + i);
        } else {
          for (int i = g.thread; i < count; i += g.threads) copy_async4(dst + i, src + i);
        }
        for (int i = count + g.thread; i < per * W; i += g.threads) dst[i] = 0.f;   // rows past the end
      }
    }
    copies_commit();
  };

  for (int s = 0; s + 1 < a.stages; ++s) fetch(first + s * stride, s);
  int stage = 0;
  for (int64_t t = first; t < tiles; t += stride) {
    const int ahead = stage + a.stages - 1;
    fetch(t + (a.stages - 1) * stride, ahead >= a.stages ? ahead - a.stages : ahead);
    copies_wait(a.stages - 1);
    g.sync();
    float* tile = ring + stage * SLOTS * slot;
    const int64_t row0 = t * per, row = row0 + mine;
    const bool real = row < a.rows;
    work_row<L, LAYOUT, V, MODE, BRANCH>(a, g, tile + mine * W, slot, real ? row : a.rows - 1, real, u0,
                                         sums ? acc + mine * sums : nullptr,
                                         sums ? acc + mine * sums + N * C : nullptr);
    g.sync();
    const int count = (int)(a.rows - row0 < per ? a.rows - row0 : per) * W;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      float* dst = a.out[s];
      if (dst == nullptr) continue;
      dst += row0 * W;
      const float* src = tile + s * slot;
      if (a.wide) {
        for (int i = 4 * g.thread; i < count; i += 4 * g.threads)
          *reinterpret_cast<float4*>(dst + i) = *reinterpret_cast<const float4*>(src + i);
      } else {
        for (int i = g.thread; i < count; i += g.threads) dst[i] = src[i];
      }
    }
    g.sync();
    stage = stage + 1 == a.stages ? 0 : stage + 1;
  }
  if (!sums) return;
  __syncthreads();
  // Sum over the block's groups and their rows, in order.
  const int64_t group_floats = a.stages * SLOTS * slot + sums4 + 16 * kMaxGroupWarps;
  for (int i = threadIdx.x; i < sums; i += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < groups; ++k) {
      const float* from = shared + k * group_floats + a.stages * SLOTS * slot + i;
      for (int r = 0; r < per; ++r) s += from[r * sums];
    }
    a.partial[(int64_t)blockIdx.x * sums + i] = s;
  }
}

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

struct Shape {
  int lanes, warps, stages, groups, shared_bytes;
};

// Lanes per row, warps per group, copy stages and groups per block that fit shared memory.
bool shape_of(int C, int L, int mode, bool branch, bool sums, int64_t rows, int sms, Shape* s) {
  const int slots = slots_of(mode, branch), warps = max_warps(mode), N = L + 1, V = C % 4 == 0 ? 4 : 1, units = C / V;
  const int64_t W = (int64_t)C * N * N;
  if (W > (1 << 20)) return false;
  s->warps = 1;
  s->lanes = 1;
  if (units <= 32) {
    while (s->lanes < units) s->lanes *= 2;
  } else {
    while (s->warps < kMaxGroupWarps && s->warps * 32 < units) s->warps *= 2;
    s->lanes = 32 * s->warps;
  }
  const int per = s->warps == 1 ? 32 / s->lanes : 1;
  const int64_t slot = (per * W + 3) & ~3ll;
  const int64_t sum4 = sums ? (per * 2 * N * C + 3) & ~3ll : 0;
  const int64_t fixed = sum4 + 16 * kMaxGroupWarps;
  const int most = warps / s->warps;
  const int64_t tiles = (rows + per - 1) / per, wanted = (tiles + sms - 1) / sms;
  for (s->stages = 4; s->stages >= 1; --s->stages) {
    const int64_t bytes = 4 * (s->stages * slots * slot + fixed);
    int64_t groups = kSharedBudget / bytes;
    if (groups < 1 && s->stages == 1 && bytes <= kSharedLimit) groups = 1;   // the widest rows
    if (groups > most) groups = most;
    if (groups > wanted) groups = wanted;
    if (groups < 1) {
      if (s->stages > 1) continue;
      return false;
    }
    // fewer stages where they make room for groups (two at least while two fit)
    if (s->stages > 2 && groups < most && groups < wanted) continue;
    s->groups = (int)groups;
    s->shared_bytes = (int)(groups * bytes);
    return true;
  }
  return false;
}

template <int L, int LAYOUT, int V, int MODE, bool BRANCH>
cudaError_t launch_one(const BlockArgs& a, const Shape& s, int grid, cudaStream_t stream) {
  auto kernel = block_kernel<L, LAYOUT, V, MODE, BRANCH>;
  static std::atomic<bool> ready[kMaxDevices];   // shared-memory limit raised on this device
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  if (device >= kMaxDevices || !ready[device].load(std::memory_order_relaxed)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedLimit);
    if (err != cudaSuccess) return err;
    if (device < kMaxDevices) ready[device].store(true, std::memory_order_relaxed);
  }
  kernel<<<grid, s.groups * s.warps * 32, s.shared_bytes, stream>>>(a);
  return cudaGetLastError();
}

template <int L, int LAYOUT, int V, int MODE>
cudaError_t launch_branch(const BlockArgs& a, const Shape& s, int grid, bool branch, cudaStream_t stream) {
  return branch ? launch_one<L, LAYOUT, V, MODE, true>(a, s, grid, stream)
                : launch_one<L, LAYOUT, V, MODE, false>(a, s, grid, stream);
}
template <int L, int MODE>
cudaError_t launch_layout(const BlockArgs& a, const Shape& s, int grid, int layout, bool branch, cudaStream_t stream) {
  const bool four = a.channels % 4 == 0;
  if (layout == kMulIr)
    return four ? launch_branch<L, kMulIr, 4, MODE>(a, s, grid, branch, stream)
                : launch_branch<L, kMulIr, 1, MODE>(a, s, grid, branch, stream);
  return four ? launch_branch<L, kIrMul, 4, MODE>(a, s, grid, branch, stream)
              : launch_branch<L, kIrMul, 1, MODE>(a, s, grid, branch, stream);
}
template <int MODE>
cudaError_t launch_degree(const BlockArgs& a, const Shape& s, int grid, int lmax, int layout, bool branch,
                          cudaStream_t stream) {
  switch (lmax) {
    case 0: return launch_layout<0, MODE>(a, s, grid, layout, branch, stream);
    case 1: return launch_layout<1, MODE>(a, s, grid, layout, branch, stream);
    case 2: return launch_layout<2, MODE>(a, s, grid, layout, branch, stream);
    default: return launch_layout<3, MODE>(a, s, grid, layout, branch, stream);
  }
}

int invalid(const char* what) {
  ictc_set_error(what, "");
  return ICTC_ERR_INVALID;
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int sm_count() {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return sms > 0 ? sms : 1;
}

// Runs one mode over all rows; `sums` >= 0: weight-gradient sums wanted (blocks written to *blocks).
int run(int mode, BlockArgs& a, int lmax, int layout, bool branch, bool sums, int* blocks, cudaStream_t stream) {
  const int slots = slots_of(mode, branch), C = a.channels;
  const int sms = sm_count();
  Shape s{};
  if (!shape_of(C, lmax, mode, branch, sums, a.rows, sms, &s)) {
    ictc_set_error("ictc_block: rows of this width do not fit shared memory%s", "");
    return ICTC_ERR_UNSUPPORTED;
  }
  const int64_t W = (int64_t)C * (lmax + 1) * (lmax + 1);
  bool wide = W % 4 == 0;
  for (int i = 0; i < slots; ++i) wide = wide && aligned(a.in[i]) && aligned(a.out[i]);
  a.wide = wide;
  a.vec_gate = aligned(a.gate) && aligned(a.gate_dot) && aligned(a.gate_out) && aligned(a.post) && aligned(a.scale) &&
               aligned(a.pre);
  a.lanes = s.lanes;
  a.warps = s.warps;
  a.stages = s.stages;
  const int per = s.warps == 1 ? 32 / s.lanes : 1;
  const int64_t tiles = (a.rows + per - 1) / per, want = (tiles + s.groups - 1) / s.groups;
  const int grid = (int)(want < sms ? want : sms);
  if (blocks) *blocks = grid;
  cudaError_t err = mode == kForward    ? launch_degree<kForward>(a, s, grid, lmax, layout, branch, stream)
                    : mode == kBackward ? launch_degree<kBackward>(a, s, grid, lmax, layout, branch, stream)
                                        : launch_degree<kSecond>(a, s, grid, lmax, layout, branch, stream);
  if (err != cudaSuccess) {
    ictc_set_error("ictc_block: %s", cudaGetErrorString(err));
    return ICTC_ERR_CUDA;
  }
  return ICTC_OK;
}

int weight_sums(const BlockArgs& a, int lmax, int blocks, float* grad_post, float* grad_scale, float* grad_pre,
                cudaStream_t stream) {
  const int columns = (lmax + 1) * a.channels;
  weight_sum_kernel<<<(columns + 7) / 8, 256, 0, stream>>>(a.partial, blocks, columns, a.post, a.scale, grad_post,
                                                           grad_scale, grad_pre);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    ictc_set_error("ictc_block: %s", cudaGetErrorString(err));
    return ICTC_ERR_CUDA;
  }
  return ICTC_OK;
}

bool bad_shape(int64_t rows, int channels, int lmax, int layout, float eps) {
  return rows < 0 || channels < 1 || lmax < 0 || lmax > kMaxL || (layout != kIrMul && layout != kMulIr) ||
         !(eps > 0.f);
}

}  // namespace
}  // namespace ictc

using namespace ictc;

extern "C" int64_t ictc_block_partial_floats(int channels, int lmax) {
  if (channels < 1 || lmax < 0 || lmax > kMaxL) return -1;
  return (int64_t)sm_count() * 2 * (lmax + 1) * channels;
}

extern "C" int ictc_block_supported(int channels, int lmax) {
  Shape s{};
  return channels >= 1 && lmax >= 0 && lmax <= kMaxL && shape_of(channels, lmax, kSecond, true, true, 1, 1, &s);
}

extern "C" int ictc_block_forward(const float* stream_in, const float* branch, const float* gate, const float* post,
                                  const float* scale, const float* pre, int norm, int64_t rows, int channels,
                                  int lmax, int layout, float eps, float* stream_out, float* normed, float* r1,
                                  float* r2, void* stream) {
  if (bad_shape(rows, channels, lmax, layout, eps) ||
      (rows > 0 && (!stream_in || (branch ? !stream_out : !norm) || (norm && !normed))))
    return invalid("ictc_block_forward: invalid argument%s");
  if (rows == 0) return ICTC_OK;
  BlockArgs a{};
  if (branch) {
    a.in[0] = branch;
    a.in[1] = stream_in;
    a.out[0] = norm ? normed : nullptr;
    a.out[1] = stream_out;
  } else {
    a.in[0] = stream_in;
    a.out[0] = normed;
  }
  a.gate = gate;
  a.post = post;
  a.scale = scale;
  a.pre = pre;
  a.r1 = r1;
  a.r2 = r2;
  a.rows = rows;
  a.channels = channels;
  a.norm = norm;
  a.eps = eps;
  return run(kForward, a, lmax, layout, branch != nullptr, false, nullptr, (cudaStream_t)stream);
}

extern "C" int ictc_block_backward(const float* stream_out, const float* branch, const float* gate, const float* post,
                                   const float* scale, const float* pre, const float* r1, const float* r2,
                                   const float* p, const float* q, int64_t rows, int channels, int lmax, int layout,
                                   float* grad_stream, float* grad_branch, float* grad_gate, float* grad_post,
                                   float* grad_scale, float* grad_pre, float* partial, void* stream) {
  const bool norm = q != nullptr, sums = grad_post || grad_scale || grad_pre;
  if (bad_shape(rows, channels, lmax, layout, 1.f) || (sums && !partial) ||
      (rows > 0 && ((norm && (!stream_out || !r2)) || (branch ? !r1 : !norm) || (!p && !q) ||
                    (grad_gate && (!gate || !branch)) || (grad_stream && !norm))))
    return invalid("ictc_block_backward: invalid argument%s");
  BlockArgs a{};
  a.post = post;
  a.scale = scale;
  a.partial = sums ? partial : nullptr;
  a.channels = channels;
  int blocks = 0;
  if (rows > 0) {
    if (branch) {
      a.in[0] = branch;
      a.in[1] = norm ? stream_out : nullptr;
      a.in[2] = p;
      a.in[3] = q;
      a.out[0] = grad_branch;
      a.out[2] = grad_stream;
    } else {
      a.in[0] = stream_out;
      a.in[1] = q;
      a.out[1] = grad_stream;
    }
    a.gate = gate;
    a.gate_out = grad_gate;
    a.pre = pre;
    a.r1 = const_cast<float*>(r1);
    a.r2 = const_cast<float*>(r2);
    a.rows = rows;
    a.norm = norm;
    if (int rc = run(kBackward, a, lmax, layout, branch != nullptr, sums, &blocks, (cudaStream_t)stream)) return rc;
  }
  return sums ? weight_sums(a, lmax, blocks, grad_post, grad_scale, grad_pre, (cudaStream_t)stream) : ICTC_OK;
}

extern "C" int ictc_block_second(const float* stream_out, const float* branch, const float* gate, const float* post,
                                 const float* scale, const float* pre, const float* r1, const float* r2,
                                 const float* p, const float* q, const float* dot_stream, const float* dot_branch,
                                 const float* dot_gate, int64_t rows, int channels, int lmax, int layout,
                                 float* grad_stream, float* grad_branch, float* grad_gate, float* grad_post,
                                 float* grad_scale, float* grad_pre, float* grad_p, float* grad_q, float* partial,
                                 void* stream) {
  const bool norm = q != nullptr, sums = grad_post || grad_scale || grad_pre;
  if (bad_shape(rows, channels, lmax, layout, 1.f) || (sums && !partial) ||
      (rows > 0 && ((norm && (!stream_out || !r2)) || (branch ? !r1 : !norm) || (!p && !q) ||
                    ((grad_gate || dot_gate) && (!gate || !branch)) || ((grad_stream || grad_q) && !norm))))
    return invalid("ictc_block_second: invalid argument%s");
  BlockArgs a{};
  a.post = post;
  a.scale = scale;
  a.partial = sums ? partial : nullptr;
  a.channels = channels;
  int blocks = 0;
  if (rows > 0) {
    if (branch) {
      a.in[0] = branch;
      a.in[1] = norm ? stream_out : nullptr;
      a.in[2] = p;
      a.in[3] = q;
      a.in[4] = dot_stream;
      a.in[5] = dot_branch;
      a.out[0] = grad_branch;
      a.out[1] = grad_stream;
      a.out[3] = grad_q;
      a.out[4] = grad_p;
    } else {
      a.in[0] = stream_out;
      a.in[1] = q;
      a.in[2] = dot_stream;
      a.out[0] = grad_stream;
      a.out[1] = grad_q;
    }
    a.gate = gate;
    a.gate_dot = dot_gate;
    a.gate_out = grad_gate;
    a.pre = pre;
    a.r1 = const_cast<float*>(r1);
    a.r2 = const_cast<float*>(r2);
    a.rows = rows;
    a.norm = norm;
    if (int rc = run(kSecond, a, lmax, layout, branch != nullptr, sums, &blocks, (cudaStream_t)stream)) return rc;
  }
  return sums ? weight_sums(a, lmax, blocks, grad_post, grad_scale, grad_pre, (cudaStream_t)stream) : ICTC_OK;
}
