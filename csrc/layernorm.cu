// Layer norm over the last dimension, forward and backward.
//
//   forward    mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps),  xhat = (x - mu) r,  y = xhat w + b
//   backward   g = dy w,  dx = r (g - mean(g) - xhat mean(g xhat)),  dw = sum_rows dy xhat,  db = sum_rows dy
//
// Both are bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx.  A row is read once and stays in
// registers, so the variance is the centred one at no extra traffic (the difference of two large sums would lose it where |mu| is large).
// A group of threads holds a row, E elements per thread: a warp where the row fits one, whole warps that meet at a barrier of their own otherwise.
// In the backward a thread keeps its columns over all rows of its group, so the weight sums stay in registers; groups of a CTA are added in shared
// memory, CTAs by a second kernel in a fixed order (no atomics: the sums have the same bits in every run).  The next row is on its way while the current
// one is reduced.  All sums are fp32.
// Replayed on a B200: 16384 x 1024 bf16 forward 14.4 us (4.7 TB/s, 71 % of the copy bandwidth), backward with its sums 22.5 us (4.5 TB/s); 4096 x 2304 fp32 15.0 and
// 22.9 us; 5001 x 2305 fp32, where rows are not on 16 bytes and elements come one by one, 18.9 and 29 us.  fp16 takes the times of bf16; 8192 x 1024 fp32 to bf16 12.0 and 17.7.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "f32x2.cuh"
#include "packs.cuh"
#include "host.h"
#include "launch.cuh"
#include "training.h"

namespace q38 {

enum ParamType : int { PARAM_F32 = 0, PARAM_BF16 = 1, PARAM_F16 = 2 };       // type of a weight's gradient

struct LnArgs {
  const void *x, *dy;
  const float *w, *b;
  void* out;                       // y or dx
  float *mean, *rstd, *partial;    // [rows], [rows], [CTAs][2][dim]
  long long rows, ldx, lddy;
  int dim, groups;                 // groups of threads per CTA
  float eps;
};

// VEC parameters at `at`, or `none` where the layer has none
template <int VEC>
__device__ __forceinline__ void ln_param(const float* p, int at, float (&out)[VEC], float none) {
  if (p != nullptr) {
    float part[VEC < 4 ? VEC : 4];
#pragma unroll
    for (int q = 0; q < VEC; q += 4) {                           // 16 bytes at a time
      unpack(load_pack<float, VEC < 4 ? VEC : 4>(p + at + q), part);
#pragma unroll
      for (int i = 0; i < (VEC < 4 ? VEC : 4); ++i) out[q + i] = part[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = none;
  }
}

// Pairs of neighbouring elements, for instructions that work on two at once
template <typename T, int VEC> __device__ __forceinline__ void pairs_of(const Pack<T, VEC>& p, uint64_t (&v)[VEC / 2]) {
  float f[VEC];
  unpack(p, f);
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) v[i] = pair2(f[2 * i], f[2 * i + 1]);
}
template <int VEC> __device__ __forceinline__ void param_pairs(const float* p, int at, uint64_t (&v)[VEC / 2], float none) {
  float f[VEC];
  ln_param<VEC>(p, at, f, none);
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) v[i] = pair2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ uint64_t twice(float a) { return pair2(a, a); }
__device__ __forceinline__ float both(uint64_t a) { const float2 f = unpair(a); return f.x + f.y; }

// Sums of N values over a group of G threads.  `scratch` belongs to the group (two halves of 32 per value, used in turn, so that one barrier per sum is enough:
// a thread writes a half again only after a barrier that all reach after they have read it).
template <bool WARP, int N>
__device__ __forceinline__ void ln_group_sum(float (&v)[N], float* scratch, int& turn, int G, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  if constexpr (!WARP) {
    const int t = threadIdx.x - group * G, warps = G >> 5;
    float* s = scratch + turn * 32 * N;
    turn ^= 1;
    if ((t & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * 32 + (t >> 5)] = v[i];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(G) : "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (t & 31) < warps ? s[i * 32 + (t & 31)] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
  }
}

// A thread's part of the weight and the bias: read once for all its rows where registers allow.  Read for every row they cost more of L1 than the row itself:
// four bytes an element against two, in accesses whose lanes are 32 bytes apart (16384 x 1024 bf16: backward 30 -> 21 us).
template <int VEC, int N, bool KEPT> struct LnParams {
  using Unit = std::conditional_t<(VEC > 1), uint64_t, float>;
  static constexpr int PER = VEC > 1 ? VEC / 2 : 1;
  Unit v[KEPT ? N : 1][PER];
  const float* p;
  float none;
  __device__ __forceinline__ void read(int at, Unit (&out)[PER]) const {
    if constexpr (VEC > 1) param_pairs<VEC>(p, at, out, none); else ln_param<1>(p, at, out, none);
  }
  // zeros behind a row's end
  __device__ __forceinline__ LnParams(const float* p_, float none_, int first, int dim) : p(p_), none(none_) {
    if constexpr (KEPT) {
#pragma unroll
      for (int c = 0; c < N; ++c) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[c][i] = 0;
        if (first + c * 32 * VEC < dim) read(first + c * 32 * VEC, v[c]);
      }
    }
  }
  // chunk c of the thread, at element `at` of the row (inside it, unless kept)
  __device__ __forceinline__ void get(int c, int at, Unit (&out)[PER]) const {
    if constexpr (KEPT) {
#pragma unroll
      for (int i = 0; i < PER; ++i) out[i] = v[c][i];
    } else read(at, out);
  }
};

template <typename InT, typename OutT, int VEC, int E, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024, !WARP ? 1 : E == 8 ? 4 : E == 16 ? 3 : 2) layer_norm_fwd_kernel(LnArgs p) {
  grid_wait();
  __shared__ float scratch[WARP ? 1 : 8][64];
  constexpr int N = E / VEC;
  constexpr bool KEPT = WARP || E == 8;                          // otherwise 1024 threads leave no registers for it
  constexpr bool AHEAD = E <= 16 || (VEC > 1 && sizeof(InT) == 2);
  const int G = WARP ? 32 : blockDim.x / p.groups, group = threadIdx.x / G, t = threadIdx.x - group * G;
  const int first = (t >> 5) * 32 * E + (t & 31) * VEC;          // a warp's columns lie side by side, a thread's at fixed distances: accesses need no arithmetic
  const float inv = 1.f / p.dim;
  const long long stride = (long long)gridDim.x * p.groups;
  const LnParams<VEC, N, KEPT> weight(p.w, 1.f, first, p.dim), bias(p.b, 0.f, first, p.dim);
  Pack<InT, VEC> v[N] = {}, next[AHEAD ? N : 1] = {};            // rows as they came: half the registers for 16-bit types
  auto fetch = [&](long long at_row, auto& to) {
    if (at_row >= p.rows) return;
    const InT* x = reinterpret_cast<const InT*>(p.x) + at_row * p.ldx;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int at = first + c * 32 * VEC;
      if (at < p.dim) to[c] = load_pack<InT, VEC>(x + at);
    }
  };
  int turn = 0;
  long long row = (long long)blockIdx.x * p.groups + group;
  if constexpr (AHEAD) fetch(row, next);
#pragma unroll 1
  for (; row < p.rows; row += stride) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int c = 0; c < N; ++c) v[c] = next[c];
      fetch(row + stride, next);
    } else fetch(row, v);
    float one[1], mu, ss = 0.f;
    if constexpr (VEC > 1) {
      uint64_t acc = 0;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        uint64_t f[VEC / 2];
        pairs_of(v[c], f);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) acc = add2(acc, f[i]);
      }
      mu = both(acc);
    } else {
      mu = 0.f;
#pragma unroll
      for (int c = 0; c < E; ++c) { float f[1]; unpack(v[c], f); mu += f[0]; }
    }
    one[0] = mu;
    ln_group_sum<WARP>(one, scratch[WARP ? 0 : group], turn, G, group);
    mu = one[0] * inv;
#pragma unroll
    for (int c = 0; c < N; ++c) forget(v[c]);
    if constexpr (VEC > 1) {
      const uint64_t minus = twice(-mu);
#pragma unroll
      for (int c = 0; c < N; ++c) {
        uint64_t f[VEC / 2], acc = 0;
        pairs_of(v[c], f);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) { const uint64_t d = add2(f[i], minus); acc = fma2(d, d, acc); }
        ss += first + c * 32 * VEC < p.dim ? both(acc) : 0.f;
      }
    } else {
#pragma unroll
      for (int c = 0; c < E; ++c) { float f[1]; unpack(v[c], f); const float d = first + c * 32 < p.dim ? f[0] - mu : 0.f; ss += d * d; }
    }
    one[0] = ss;
    ln_group_sum<WARP>(one, scratch[WARP ? 0 : group], turn, G, group);
    const float r = rsqrtf(one[0] * inv + p.eps);
    if (t == 0 && p.mean != nullptr) { p.mean[row] = mu; p.rstd[row] = r; }
#pragma unroll
    for (int c = 0; c < N; ++c) forget(v[c]);
    OutT* y = reinterpret_cast<OutT*>(p.out) + row * p.dim;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int at = first + c * 32 * VEC;
      if (at < p.dim) {
        float o[VEC];
        if constexpr (VEC > 1) {
          uint64_t f[VEC / 2], w[VEC / 2], b[VEC / 2];
          pairs_of(v[c], f);
          weight.get(c, at, w);
          bias.get(c, at, b);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float2 y2 = unpair(fma2(mul2(add2(f[i], twice(-mu)), twice(r)), w[i], b[i]));
            o[2 * i] = y2.x; o[2 * i + 1] = y2.y;
          }
        } else {
          float w[1], b[1];
          unpack(v[c], o);
          weight.get(c, at, w);
          bias.get(c, at, b);
          o[0] = (o[0] - mu) * r * w[0] + b[0];
        }
        store_pack<OutT, VEC>(y + at, pack<OutT, VEC>(o));
      }
    }
  }
}

// ACC: where the weight sums of a thread's columns live (registers, or shared memory for rows so long that registers would spill; each cell has one owner).
template <typename InT, typename OutT, int VEC, int E, bool WARP, bool ACC_SMEM>
__global__ void __launch_bounds__(ACC_SMEM ? 1024 : E == 32 ? 256 : E == 8 ? (VEC == 8 ? 384 : 640) : 512, E == 8 && VEC == 8 ? 2 : 1) layer_norm_bwd_kernel(LnArgs p) {
  grid_wait();
  extern __shared__ float sums[];                                // [groups][2][dim]
  __shared__ float scratch[WARP ? 1 : 16][128];
  constexpr int N = E / VEC;
  const int G = WARP ? 32 : blockDim.x / p.groups, group = threadIdx.x / G, t = threadIdx.x - group * G;
  const int first = (t >> 5) * 32 * E + (t & 31) * VEC;          // a warp's columns lie side by side, a thread's at fixed distances: accesses need no arithmetic
  const bool wanted = p.partial != nullptr;
  constexpr bool KEPT = !ACC_SMEM && (E != 16 || (VEC > 1 && sizeof(InT) == 2));
  const LnParams<VEC, N, KEPT> weight(p.w, 1.f, first, p.dim);
  const float inv = 1.f / p.dim;
  using Acc = std::conditional_t<(VEC > 1), uint64_t, float>;    // pairs of columns, or single ones
  constexpr int ACCS = ACC_SMEM ? 1 : VEC > 1 ? E / 2 : E;
  Acc aw[ACCS], ab[ACCS];
  if constexpr (ACC_SMEM) {
    for (int i = threadIdx.x; i < 2 * p.dim; i += blockDim.x) sums[i] = 0.f;
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < ACCS; ++i) aw[i] = ab[i] = 0;
  }
  const long long stride = (long long)gridDim.x * p.groups;
  long long row = (long long)blockIdx.x * p.groups + group;
  constexpr bool AHEAD = !ACC_SMEM;                              // with 1024 threads there are no registers for a row ahead
  Pack<InT, VEC> x[N], nx[N] = {};                               // zeros behind a row's end: no gradient there, so no share in any sum
  Pack<OutT, VEC> d[N], nd[N] = {};
  float mu = 0.f, r = 0.f, nmu = 0.f, nr = 0.f;
  auto fetch = [&](long long at_row) {
    if (at_row >= p.rows) return;
    const InT* px = reinterpret_cast<const InT*>(p.x) + at_row * p.ldx;
    const OutT* pd = reinterpret_cast<const OutT*>(p.dy) + at_row * p.lddy;
    nmu = p.mean[at_row]; nr = p.rstd[at_row];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int at = first + c * 32 * VEC;
      if (at < p.dim) {
        nx[c] = load_pack<InT, VEC>(px + at);
        nd[c] = load_pack<OutT, VEC>(pd + at);
      }
    }
  };
  if (AHEAD) fetch(row);
  int turn = 0;
#pragma unroll 1
  for (; row < p.rows; row += stride) {
    if (!AHEAD) fetch(row);
#pragma unroll
    for (int c = 0; c < N; ++c) { x[c] = nx[c]; d[c] = nd[c]; }
    mu = nmu; r = nr;
    if (AHEAD) fetch(row + stride);
    float s1 = 0.f, s2 = 0.f;
    if constexpr (VEC > 1 && !ACC_SMEM) {
      uint64_t t1 = 0, t2 = 0;
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const int at = first + c * 32 * VEC;
        uint64_t xv[VEC / 2], dv[VEC / 2], w[VEC / 2] = {};
        pairs_of(x[c], xv);
        pairs_of(d[c], dv);
        if (KEPT || at < p.dim) weight.get(c, at, w);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const uint64_t hat = mul2(add2(xv[i], twice(-mu)), twice(r)), g = mul2(dv[i], w[i]);
          aw[c * VEC / 2 + i] = fma2(dv[i], hat, aw[c * VEC / 2 + i]);
          ab[c * VEC / 2 + i] = add2(dv[i], ab[c * VEC / 2 + i]);
          t1 = add2(t1, g);
          t2 = fma2(g, hat, t2);
        }
      }
      s1 = both(t1); s2 = both(t2);
    } else {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const int at = first + c * 32 * VEC;
        if (at < p.dim) {
          float xv[VEC], dv[VEC], w[VEC];
          unpack(x[c], xv);
          unpack(d[c], dv);
          if constexpr (VEC == 1) weight.get(c, at, w); else ln_param<VEC>(p.w, at, w, 1.f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float hat = (xv[i] - mu) * r, g = dv[i] * w[i];
            if constexpr (ACC_SMEM) { sums[at + i] += dv[i] * hat; sums[p.dim + at + i] += dv[i]; }
            else { aw[c] += dv[i] * hat; ab[c] += dv[i]; }
            s1 += g; s2 += g * hat;
          }
        }
      }
    }
    float s[2] = {s1, s2};
    ln_group_sum<WARP>(s, scratch[WARP ? 0 : group], turn, G, group);
#pragma unroll
    for (int c = 0; c < N; ++c) { forget(x[c]); forget(d[c]); }
    if (p.out != nullptr) {
      const float k0 = s[0] * inv * r, k1 = s[1] * inv * r;        // dx = r g - k0 - xhat k1 (r r could overflow where eps is zero)
      InT* dx = reinterpret_cast<InT*>(p.out) + row * p.dim;
#pragma unroll
      for (int c = 0; c < N; ++c) {                              // from the packed row again: the values themselves would take twice its registers
        const int at = first + c * 32 * VEC;
        if (at < p.dim) {
          float o[VEC];
          if constexpr (VEC > 1) {
            uint64_t xv[VEC / 2], dv[VEC / 2], w[VEC / 2];
            pairs_of(x[c], xv);
            pairs_of(d[c], dv);
            weight.get(c, at, w);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
              const uint64_t hat = mul2(add2(xv[i], twice(-mu)), twice(r));
              const float2 f = unpair(fma2(dv[i], mul2(w[i], twice(r)), fma2(hat, twice(-k1), twice(-k0))));
              o[2 * i] = f.x; o[2 * i + 1] = f.y;
            }
          } else {
            float dv[1], w[1];
            unpack(x[c], o);
            unpack(d[c], dv);
            weight.get(c, at, w);
            o[0] = dv[0] * (w[0] * r) - ((o[0] - mu) * r * k1 + k0);
          }
          store_pack<InT, VEC>(dx + at, pack<InT, VEC>(o));
        }
      }
    }
  }
  if (!wanted) return;
  float* mine = p.partial + (long long)blockIdx.x * 2 * p.dim;
  if constexpr (!ACC_SMEM) {
    // every group leaves its sums side by side, then each column is added over the groups in order
    float* to = p.groups == 1 ? mine : sums + (long long)group * 2 * p.dim;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int at = first + c * 32 * VEC;
      if (at < p.dim) {
        if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            *reinterpret_cast<float2*>(to + at + 2 * i) = unpair(aw[c * VEC / 2 + i]);
            *reinterpret_cast<float2*>(to + p.dim + at + 2 * i) = unpair(ab[c * VEC / 2 + i]);
          }
        } else { to[at] = aw[c]; to[p.dim + at] = ab[c]; }
      }
    }
    if (p.groups == 1) return;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.dim; i += blockDim.x) {
    float s = sums[i];
    if constexpr (!ACC_SMEM)
      for (int k = 1; k < p.groups; ++k) s += sums[(long long)k * 2 * p.dim + i];
    mine[i] = s;
  }
}

// Rows of any length, a CTA each, read again for every sum (the row comes from L2).  The weight sums are kept in the CTA's part of `partial`.  Bound by those reads, an
// element per access: 1000 x 20000 bf16 forward 86 us, with backward 246 (floors 12 and 31).
template <typename InT, typename OutT>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(LnArgs p, bool backward) {
  grid_wait();
  __shared__ float scratch[32];
  float* mine = p.partial == nullptr ? nullptr : p.partial + (long long)blockIdx.x * 2 * p.dim;
  if (mine != nullptr)
    for (int i = threadIdx.x; i < 2 * p.dim; i += blockDim.x) mine[i] = 0.f;      // a cell is touched by one thread only
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const InT* x = reinterpret_cast<const InT*>(p.x) + row * p.ldx;
    float w[1], b[1];
    if (!backward) {
      float sum = 0.f, ss = 0.f;
      for (int i = threadIdx.x; i < p.dim; i += blockDim.x) sum += to_float(x[i]);
      const float mu = block_sum(sum, scratch) / p.dim;
      for (int i = threadIdx.x; i < p.dim; i += blockDim.x) { const float d = to_float(x[i]) - mu; ss += d * d; }
      const float r = rsqrtf(block_sum(ss, scratch) / p.dim + p.eps);
      if (threadIdx.x == 0 && p.mean != nullptr) { p.mean[row] = mu; p.rstd[row] = r; }
      OutT* y = reinterpret_cast<OutT*>(p.out) + row * p.dim;
      for (int i = threadIdx.x; i < p.dim; i += blockDim.x) {
        ln_param<1>(p.w, i, w, 1.f);
        ln_param<1>(p.b, i, b, 0.f);
        y[i] = from_float<OutT>((to_float(x[i]) - mu) * r * w[0] + b[0]);
      }
    } else {
      const OutT* dy = reinterpret_cast<const OutT*>(p.dy) + row * p.lddy;
      const float mu = p.mean[row], r = p.rstd[row];
      float s1 = 0.f, s2 = 0.f;
      for (int i = threadIdx.x; i < p.dim; i += blockDim.x) {
        ln_param<1>(p.w, i, w, 1.f);
        const float d = to_float(dy[i]), hat = (to_float(x[i]) - mu) * r;
        s1 += d * w[0]; s2 += d * w[0] * hat;
        if (mine != nullptr) { mine[i] += d * hat; mine[p.dim + i] += d; }
      }
      const float m1 = block_sum(s1, scratch) / p.dim, m2 = block_sum(s2, scratch) / p.dim;
      if (p.out == nullptr) continue;
      InT* dx = reinterpret_cast<InT*>(p.out) + row * p.dim;
      for (int i = threadIdx.x; i < p.dim; i += blockDim.x) {
        ln_param<1>(p.w, i, w, 1.f);
        dx[i] = from_float<InT>(r * (to_float(dy[i]) * w[0] - m1 - (to_float(x[i]) - mu) * r * m2));
      }
    }
  }
}

// dw and db from the CTAs' parts: 32 columns per CTA, 32 threads per column in strides of 32 parts (four reads in flight), then in order.
__global__ void __launch_bounds__(1024) layer_norm_sums_kernel(const float* __restrict__ partial, int parts, int dim, void* dw, int wt, void* db, int bt) {
  grid_wait();
  __shared__ float acc[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x, which = blockIdx.y;
  void* to = which ? db : dw;
  if (to == nullptr) return;
  float s = 0.f;
  if (col < dim) {
    const float* in = partial + (long long)which * dim + col;
    const long long step = 2ll * dim;
    for (int q = threadIdx.y; q < parts; q += 128) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = q + 32 * e < parts ? in[(q + 32 * e) * step] : 0.f;
      s += (v[0] + v[1]) + (v[2] + v[3]);
    }
  }
  acc[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = warp_sum(acc[threadIdx.x][threadIdx.y]);                   // a warp per column from here
  const int mine = blockIdx.x * 32 + threadIdx.y, type = which ? bt : wt;
  if (threadIdx.x != 0 || mine >= dim) return;
  if (type == PARAM_F32) reinterpret_cast<float*>(to)[mine] = s;
  else if (type == PARAM_BF16) reinterpret_cast<__nv_bfloat16*>(to)[mine] = __float2bfloat16_rn(s);
  else reinterpret_cast<__half*>(to)[mine] = __float2half_rn(s);
}

namespace {

int param_type(const OptTensor& t) {
  return !t.has_value() || t->scalar_type() == at::kFloat ? PARAM_F32 : t->scalar_type() == at::kBFloat16 ? PARAM_BF16 : PARAM_F16;
}
// Parameters as the kernels take them: fp32 (a vector in another type is converted, which costs a small launch and no branch in the kernels)
at::Tensor param(const OptTensor& t) {
  return !t.has_value() ? at::Tensor() : t->scalar_type() == at::kFloat && t->is_contiguous() ? *t : t->to(at::kFloat).contiguous();
}
const float* param_ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int LN_LONGEST = 16384;          // longest row that a CTA of 1024 threads holds in registers

// Threads per row: elements come in vectors, a thread holds E of them
int group_of(int dim, int E) { return (dim + 32 * E - 1) / (32 * E) * 32; }

// Calls f(InT, OutT) for the supported pairs of input and output type.
template <typename F>
void by_type(at::ScalarType in, at::ScalarType out, F&& f) {
  if (in == at::kFloat && out == at::kFloat) f(float{}, float{});
  else if (in == at::kFloat && out == at::kBFloat16) f(float{}, __nv_bfloat16{});
  else if (in == at::kBFloat16 && out == at::kBFloat16) f(__nv_bfloat16{}, __nv_bfloat16{});
  else if (in == at::kHalf && out == at::kHalf) f(__half{}, __half{});
  else TORCH_CHECK_VALUE(false, "layer_norm: output type ", out, " for an input of type ", in, " is not supported");
}

template <typename InT, typename OutT, int VEC>
void launch_fwd(LnArgs& p, cudaStream_t stream) {
  // A warp per row up to 512 elements, 1024 packed ones: no barrier.  Eight rows per CTA.  (8192 x 1024 fp32 by warps 20.0 us, by groups of 128 threads 17.)
  auto warp_rows = [&](auto kernel, int resident) {
    p.groups = 8;
    launch(kernel, (unsigned)std::min<long long>((p.rows + 7) / 8, resident * kNumSMs), 256, 0, stream, p);
  };
  if (p.dim <= 256) warp_rows(layer_norm_fwd_kernel<InT, OutT, VEC, 8, true>, 4);
  else if (p.dim <= 512) warp_rows(layer_norm_fwd_kernel<InT, OutT, VEC, 16, true>, 3);
  else if (VEC == 8 && p.dim <= 1024) warp_rows(layer_norm_fwd_kernel<InT, OutT, VEC, VEC == 8 ? 32 : 16, true>, 2);
  else {
    const bool wide = p.dim > 8192;
    const int G = group_of(p.dim, wide ? 16 : 8);
    p.groups = std::max(1, std::min(8, 256 / G));
    const unsigned grid = (unsigned)std::min<long long>((p.rows + p.groups - 1) / p.groups, std::max(1, 1024 / (G * p.groups)) * kNumSMs);
    if (wide) launch(layer_norm_fwd_kernel<InT, OutT, VEC, 16, false>, grid, G * p.groups, 0, stream, p);
    else launch(layer_norm_fwd_kernel<InT, OutT, VEC, 8, false>, grid, G * p.groups, 0, stream, p);
  }
}

struct BwdShape { int G, groups, ctas; };
// Elements per thread: eight, or more.  The sums over a group cost some sixty instructions per thread and row, so packed rows, which have the registers, take sixteen or thirty-two.
bool eight_each(int dim, bool packed16) { return dim <= 256 || (!packed16 && dim > 512 && dim <= 4096); }

// Threads per row, rows per CTA and CTAs.  Eight 16-bit elements per thread take 80 registers (768 threads per SM), eight others up to 96 (640), sixteen up to 128 (512), thirty-two 234 (256);
// what counts is the bytes on their way, 32 to 64 KB per SM in each case.  As many CTAs as are resident at once.
BwdShape bwd_shape(long long rows, int dim, bool packed16) {
  if (dim > LN_LONGEST) return {1024, 1, (int)std::min<long long>(rows, kNumSMs)};
  BwdShape s;
  const bool eight = eight_each(dim, packed16);
  const bool warp32 = packed16 && dim > 512 && dim <= 1024;      // thirty-two per thread: a warp holds the row, no barrier
  const int threads = warp32 ? 256 : eight ? (packed16 ? 384 : 320) : 512, resident = warp32 ? 256 : eight ? (packed16 ? 768 : 640) : 512;
  s.G = dim <= 512 || warp32 ? 32 : group_of(dim, eight ? 8 : 16);
  s.groups = std::max(1, threads / s.G);
  s.ctas = (int)std::min<long long>((rows + s.groups - 1) / s.groups, std::max(1, resident / (s.G * s.groups)) * kNumSMs);
  return s;
}

template <typename InT, typename OutT, int VEC>
void launch_bwd(LnArgs& p, const BwdShape& s, cudaStream_t stream) {
  p.groups = s.groups;
  // Several groups: 64 KB at most.  One group with its sums in shared memory: both sums of the longest row.
  constexpr int most = 2 * LN_LONGEST * 4;
  static_assert(most <= 192 * 1024, "shared memory of a CTA, beside the scratch");
  const size_t smem = s.groups > 1 || p.dim > 8192 ? size_t(s.groups) * 2 * p.dim * 4 : 0;
  TORCH_CHECK(smem <= most, "layer_norm: shared memory of the backward");
  auto go = [&](auto kernel) {
    if (smem > 40 * 1024) allow_shared_memory((const void*)kernel, most);
    launch(kernel, (unsigned)s.ctas, s.G * s.groups, smem, stream, p);
  };
  if (p.dim <= 256) go(layer_norm_bwd_kernel<InT, OutT, VEC, 8, true, false>);
  else if (p.dim <= 512) go(layer_norm_bwd_kernel<InT, OutT, VEC, 16, true, false>);
  else if (VEC == 8 && p.dim <= 1024) go(layer_norm_bwd_kernel<InT, OutT, VEC, VEC == 8 ? 32 : 8, true, false>);
  else if (VEC != 8 && p.dim <= 4096) go(layer_norm_bwd_kernel<InT, OutT, VEC, VEC == 8 ? 16 : 8, false, false>);
  else if (p.dim <= 8192) go(layer_norm_bwd_kernel<InT, OutT, VEC, 16, false, false>);
  else go(layer_norm_bwd_kernel<InT, OutT, VEC, 16, false, true>);
}

void check_params(const at::Tensor& x, const OptTensor& w, const OptTensor& b) {
  for (const auto* t : {&w, &b})
    if (t->has_value())
      TORCH_CHECK_VALUE((*t)->device() == x.device() && (*t)->dim() == 1 && (*t)->size(0) == x.size(-1) &&
                        ((*t)->scalar_type() == at::kFloat || (*t)->scalar_type() == at::kBFloat16 || (*t)->scalar_type() == at::kHalf),
                        "layer_norm: weight and bias are fp32, bf16 or fp16 vectors of the last dimension's length on the input's device");
}

// A tensor as rows with contiguous columns and one distance between them; copied where it has not that already.
struct Rows {
  at::Tensor held;
  long long rows, ld;
  explicit Rows(const at::Tensor& t) : held(t), rows(1), ld(t.size(-1)) {
    const auto sizes = t.sizes(), strides = t.strides();
    const int64_t last = t.dim() - 1;
    bool ok = strides[last] == 1 || sizes[last] == 1, set = false;
    long long next = 0;
    for (int64_t i = last - 1; i >= 0; --i) {
      rows *= sizes[i];
      if (sizes[i] == 1) continue;
      if (!set) { ld = strides[i]; set = true; }
      else if (strides[i] != next) ok = false;
      next = strides[i] * sizes[i];
    }
    if (!ok && rows) { held = t.contiguous(); ld = t.size(-1); }
  }
};

}  // namespace

std::pair<at::Tensor, at::Tensor> layer_norm_fwd(const at::Tensor& x, const OptTensor& w, const OptTensor& b, double eps, at::ScalarType out_type, bool save) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() > 0 && x.size(-1) > 0 && x.size(-1) <= INT_MAX / 2, "layer_norm: a CUDA input with a last dimension that is not empty is required");
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must not be negative");
  check_params(x, w, b);
  const c10::cuda::CUDAGuard guard(x.device());
  const Rows in(x);
  LnArgs p{};
  p.rows = in.rows; p.dim = (int)x.size(-1); p.ldx = in.ld; p.eps = (float)eps;
  auto y = new_tensor(x.sizes(), out_type, x.device());
  const at::Tensor wf = param(w), bf = param(b);
  p.x = in.held.data_ptr(); p.out = y.data_ptr(); p.w = param_ptr(wf); p.b = param_ptr(bf);
  at::Tensor stats;
  if (save) {
    stats = new_tensor({2, p.rows}, at::kFloat, x.device());
    p.mean = stats.data_ptr<float>(); p.rstd = p.mean + p.rows;
  }
  by_type(x.scalar_type(), out_type, [&](auto in_zero, auto out_zero) {
    using InT = decltype(in_zero);
    using OutT = decltype(out_zero);
    constexpr int VEC = 16 / sizeof(InT);
    if (p.rows == 0) return;
    TORCH_CHECK_VALUE(p.rows < (1ll << 31), "layer_norm: at most 2^31 - 1 rows");
    auto stream = at::cuda::getCurrentCUDAStream();
    const bool vec = p.dim % VEC == 0 && p.ldx % VEC == 0 && on16(p.x) && on16(p.out) && on16(p.w) && on16(p.b);
    if (p.dim > LN_LONGEST) launch(layer_norm_long_kernel<InT, OutT>, (unsigned)std::min<long long>(p.rows, 2 * kNumSMs), 1024, 0, stream, p, false);
    else if (vec) launch_fwd<InT, OutT, VEC>(p, stream);
    else launch_fwd<InT, OutT, 1>(p, stream);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launch();
  });
  return {y, stats};
}

std::array<at::Tensor, 3> layer_norm_bwd(const at::Tensor& dy_, const at::Tensor& x_, const OptTensor& w, const OptTensor& b, const at::Tensor& stats, bool want_dx, bool want_dw, bool want_db) {
  TORCH_CHECK(x_.is_cuda() && dy_.device() == x_.device() && dy_.sizes() == x_.sizes(), "layer_norm: a gradient of the result's shape and device required");
  check_params(x_, w, b);
  const c10::cuda::CUDAGuard guard(x_.device());
  const Rows x(x_), dy(dy_);
  const auto device = x_.device();
  LnArgs p{};
  p.rows = x.rows; p.dim = (int)x_.size(-1); p.ldx = x.ld; p.lddy = dy.ld;
  at::Tensor dx, dw, db;
  if (want_dx) dx = new_tensor(x_.sizes(), x_.scalar_type(), device);
  if (want_dw) dw = new_tensor({p.dim}, w->scalar_type(), device);
  if (want_db) db = new_tensor({p.dim}, b->scalar_type(), device);
  if (p.rows == 0) {
    if (want_dw) dw.zero_();
    if (want_db) db.zero_();
    return {dx, dw, db};
  }
  TORCH_CHECK(stats.numel() == 2 * p.rows, "layer_norm: statistics of every row required");
  const int per16 = 16 / (int)x_.element_size();
  const at::Tensor wf = param(w);
  p.x = x.held.data_ptr(); p.dy = dy.held.data_ptr(); p.w = param_ptr(wf);
  p.out = want_dx ? dx.data_ptr() : nullptr;
  p.mean = stats.data_ptr<float>(); p.rstd = p.mean + p.rows;
  const bool vec = p.dim % per16 == 0 && p.ldx % per16 == 0 && p.lddy % per16 == 0 && on16(p.x) && on16(p.dy) && on16(p.out) && on16(p.w);
  const BwdShape s = bwd_shape(p.rows, p.dim, vec && per16 == 8);
  at::Tensor partial;
  if (want_dw || want_db) {
    partial = new_tensor({s.ctas, 2, p.dim}, at::kFloat, device);
    p.partial = partial.data_ptr<float>();
  }
  auto stream = at::cuda::getCurrentCUDAStream();
  by_type(x_.scalar_type(), dy_.scalar_type(), [&](auto in_zero, auto out_zero) {
    using InT = decltype(in_zero);
    using OutT = decltype(out_zero);
    constexpr int VEC = 16 / sizeof(InT);
    if (p.dim > LN_LONGEST) launch(layer_norm_long_kernel<InT, OutT>, (unsigned)s.ctas, 1024, 0, stream, p, true);
    else if (vec) launch_bwd<InT, OutT, VEC>(p, s, stream);
    else launch_bwd<InT, OutT, 1>(p, s, stream);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launch();
  });
  if (partial.defined()) {
    launch(layer_norm_sums_kernel, dim3((p.dim + 31) / 32, 2), dim3(32, 32), 0, stream, (const float*)p.partial, s.ctas, p.dim, want_dw ? dw.data_ptr() : nullptr,
           param_type(w), want_db ? db.data_ptr() : nullptr, param_type(b));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launch();
  }
  return {dx, dw, db};
}

}  // namespace q38
