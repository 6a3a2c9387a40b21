// Global 2-norm of many tensors and their scaling by min(1, max_norm / (norm + 1e-6)).
//
// Two launches for up to 512 tensors of any sizes: the tensors' addresses travel as kernel parameters (no table to copy to the device, so a captured
// graph replays without host memory), and each CTA walks pieces of equal size of the whole list.
//   norm    each CTA leaves its sum of squares in 64 bits, in a fixed order: squares of fp32 values are formed there too, so they neither overflow nor vanish; those of
//           16-bit values, exact in fp32, are added by fours in fp32 first (clip_four)
//   scale   each CTA adds up all sums in one order (a few KB from L2, instead of a third launch), takes the factor and scales its pieces
// Bound by memory: one read for the norm, one read and one write for the scaling.  The scaling walks backwards, since what the norm read last is still in L2.
// Where the factor is 1 and a tensor is its own result, there is nothing to write.
// Replayed on a B200: 2e8 bf16 gradients norm 74 us (5.4 TB/s), scaling into other buffers 126 (6.3 TB/s); 1e8 fp32 61 (6.5 TB/s) and 138 (5.8 TB/s).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "packs.cuh"
#include "host.h"
#include "launch.cuh"
#include "training.h"

namespace q38 {

enum ClipType : int { CLIP_F32 = 0, CLIP_BF16 = 1, CLIP_F16 = 2 };

struct ClipEntry {
  const void* in;
  void* out;
  long long n;
  int first;                       // first piece of this tensor among the launch's
  int type;                        // ClipType; + 4: not on 16 bytes
};
template <int CAP> struct ClipList {
  ClipEntry e[CAP];
  int count, pieces, piece;        // tensors, pieces, elements per piece (a multiple of 8)
};

constexpr int CLIP_THREADS = 512;

// The build flushes denormal fp32 values; a factor of one is to leave every value as it is, and small squares are to count
__device__ __forceinline__ float clip_times(float a, float b) { float r; asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ double clip_wide(float a) { double r; asm("cvt.f64.f32 %0, %1;" : "=d"(r) : "f"(a)); return r; }

template <int CAP>
__device__ __forceinline__ int clip_find(const ClipList<CAP>& l, int piece) {
  int lo = 0, hi = l.count - 1;    // the last tensor whose first piece is not behind `piece`
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.e[mid].first <= piece) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Squares of four 16-bit values one by one in 64 bits
template <typename T>
__device__ __noinline__ double clip_apart(uint32_t w0, uint32_t w1) {
  Pack<T, 4> p;
  p.w[0] = w0; p.w[1] = w1;
  float f[4];
  unpack(p, f);
  double s = 0.0;
#pragma unroll 1
  for (int e = 0; e < 4; ++e) { const double d = clip_wide(e == 0 ? f[0] : e == 1 ? f[1] : e == 2 ? f[2] : f[3]); s += d * d; }
  return s;
}

// Four 16-bit values: their squares are exact in fp32, and the sum of four has two roundings on a way, so one conversion to 64 bits does for four
// (conversions run at an eighth of the fp32 rate).  bf16 has fp32's range: a sum that is near its ends, zeros aside, is taken apart.
template <typename T>
__device__ __forceinline__ double clip_four(uint32_t w0, uint32_t w1) {
  Pack<T, 4> p;
  p.w[0] = w0; p.w[1] = w1;
  float f[4];
  unpack(p, f);
  const float s = fmaf(f[0], f[0], f[1] * f[1]) + fmaf(f[2], f[2], f[3] * f[3]);
  if (s < 1e-28f || s > 1e38f) return ((w0 | w1) & 0x7fff7fffu) == 0u ? 0.0 : clip_apart<T>(w0, w1);
  return (double)s;
}

template <typename T, int VEC>
__device__ __forceinline__ void clip_squares(const T* in, int n, double (&acc)[2]) {
  constexpr int BATCH = 4;
  const int packs = n / VEC;
#pragma unroll 1
  for (int base = threadIdx.x; base < packs; base += CLIP_THREADS * BATCH) {
    Pack<T, VEC> v[BATCH] = {};                                  // zeros behind the end
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      if (base + j * CLIP_THREADS < packs) v[j] = load_pack<T, VEC>(in + (base + j * CLIP_THREADS) * VEC);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if constexpr (VEC == 8) {
        acc[0] += clip_four<T>(v[j].w[0], v[j].w[1]);
        acc[1] += clip_four<T>(v[j].w[2], v[j].w[3]);
      } else {
        float f[VEC];
        unpack(v[j], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const double d = clip_wide(f[e]); acc[(VEC == 1 ? j : e) & 1] += d * d; }
      }
    }
  }
#pragma unroll 1
  for (int i = packs * VEC + threadIdx.x; i < n; i += CLIP_THREADS) { const double d = clip_wide(to_float(in[i])); acc[0] += d * d; }
}

template <typename T, int VEC>
__device__ __forceinline__ void clip_scale(const T* in, T* out, int n, float factor) {
  constexpr int BATCH = 4;
  const int packs = n / VEC;
#pragma unroll 1
  for (int base = threadIdx.x; base < packs; base += CLIP_THREADS * BATCH) {
    Pack<T, VEC> v[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      if (base + j * CLIP_THREADS < packs) v[j] = load_pack<T, VEC>(in + (base + j * CLIP_THREADS) * VEC);
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      if (base + j * CLIP_THREADS < packs) {
        float f[VEC];
        unpack(v[j], f);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = clip_times(f[e], factor);
        store_pack<T, VEC>(out + (base + j * CLIP_THREADS) * VEC, pack<T, VEC>(f));
      }
  }
#pragma unroll 1
  for (int i = packs * VEC + threadIdx.x; i < n; i += CLIP_THREADS) out[i] = from_float<T>(clip_times(to_float(in[i]), factor));
}

// Calls f(typed pointer, elements per 16 bytes) of a tensor
#define Q38_CLIP_BY_TYPE(TYPE, CALL)                                                    \
  switch (TYPE) {                                                                       \
    case CLIP_F32: { using T = float; constexpr int VEC = 4; CALL; break; }             \
    case CLIP_BF16: { using T = __nv_bfloat16; constexpr int VEC = 8; CALL; break; }    \
    case CLIP_F16: { using T = __half; constexpr int VEC = 8; CALL; break; }            \
    case CLIP_F32 + 4: { using T = float; constexpr int VEC = 1; CALL; break; }         \
    case CLIP_BF16 + 4: { using T = __nv_bfloat16; constexpr int VEC = 1; CALL; break; }\
    default: { using T = __half; constexpr int VEC = 1; CALL; break; }                  \
  }

template <int CAP>
__global__ void __launch_bounds__(CLIP_THREADS, 2) clip_norm_kernel(const __grid_constant__ ClipList<CAP> l, double* __restrict__ partial) {
  grid_wait();
  __shared__ double sums[CLIP_THREADS / 32];
  double acc[2] = {0.0, 0.0};
  for (int c = blockIdx.x; c < l.pieces; c += gridDim.x) {
    const ClipEntry& t = l.e[clip_find(l, c)];
    const long long at = (long long)(c - t.first) * l.piece;
    const int n = (int)min((long long)l.piece, t.n - at);
    Q38_CLIP_BY_TYPE(t.type, (clip_squares<T, VEC>(reinterpret_cast<const T*>(t.in) + at, n, acc)))
  }
  double s = acc[0] + acc[1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < CLIP_THREADS / 32; ++w) s += sums[w];
    partial[blockIdx.x] = s;
  }
}

// The norm from all launches' sums, the same in every CTA: thread t adds sums t, t + 512, ..., then a tree.
__device__ __forceinline__ double clip_total(const double* partial, int parts, double* sums) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += CLIP_THREADS) s += partial[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_THREADS / 32; ++w) s += sums[w];
  return sqrt(s);
}

template <int CAP>
__global__ void __launch_bounds__(CLIP_THREADS, 2) clip_scale_kernel(const __grid_constant__ ClipList<CAP> l, const double* __restrict__ partial, int parts, float max_norm, float* norm) {
  grid_wait();
  __shared__ double sums[CLIP_THREADS / 32];
  const float total = (float)clip_total(partial, parts, sums);
  if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const float ratio = __fdiv_rn(max_norm, total + 1e-6f);
  const float factor = ratio > 1.f ? 1.f : ratio;                // a norm that is no number makes every result none
  for (int c = l.pieces - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const ClipEntry& t = l.e[clip_find(l, c)];
    if (factor == 1.f && t.in == t.out) continue;
    const long long at = (long long)(c - t.first) * l.piece;
    const int n = (int)min((long long)l.piece, t.n - at);
    Q38_CLIP_BY_TYPE(t.type, (clip_scale<T, VEC>(reinterpret_cast<const T*>(t.in) + at, reinterpret_cast<T*>(t.out) + at, n, factor)))
  }
}

__global__ void __launch_bounds__(CLIP_THREADS) clip_total_kernel(const double* __restrict__ partial, int parts, float* norm) {
  grid_wait();
  __shared__ double sums[CLIP_THREADS / 32];
  const float total = (float)clip_total(partial, parts, sums);
  if (threadIdx.x == 0) *norm = total;
}

namespace {

using at::Tensor;

// Pieces of the whole list: enough for every SM where there is little, 16384 elements (a few loads per thread in flight) where there is much
int piece_size(long long elements) {
  int piece = 16384;
  while (piece > 2048 && elements / piece < 4 * kNumSMs) piece /= 2;
  return piece;
}

template <int CAP>
std::vector<ClipList<CAP>> lists_of(at::TensorList grads, at::TensorList outs, int piece) {
  std::vector<ClipList<CAP>> lists;
  for (size_t i = 0; i < grads.size(); ++i) {
    const long long n = grads[i].numel();
    if (!n) continue;
    const long long pieces = (n + piece - 1) / piece;
    if (lists.empty() || lists.back().count == CAP || lists.back().pieces + pieces > (1ll << 30)) { lists.emplace_back(); lists.back().count = lists.back().pieces = 0; lists.back().piece = piece; }
    TORCH_CHECK_VALUE(pieces < (1ll << 30), "clip_grad_norm: tensor too large");
    ClipList<CAP>& l = lists.back();
    ClipEntry& e = l.e[l.count++];
    e.in = grads[i].data_ptr(); e.out = outs.empty() ? const_cast<void*>(e.in) : outs[i].data_ptr(); e.n = n; e.first = l.pieces;
    e.type = grads[i].scalar_type() == at::kFloat ? CLIP_F32 : grads[i].scalar_type() == at::kBFloat16 ? CLIP_BF16 : CLIP_F16;
    if ((reinterpret_cast<uintptr_t>(e.in) | reinterpret_cast<uintptr_t>(e.out)) & 15) e.type += 4;
    l.pieces += (int)pieces;
  }
  return lists;
}

template <int CAP>
void run(at::TensorList grads, at::TensorList outs, int piece, double max_norm, bool scale, const Tensor& norm, cudaStream_t stream) {
  const auto lists = lists_of<CAP>(grads, outs, piece);
  int parts = 0;
  std::vector<int> grid;
  for (const auto& l : lists) { grid.push_back(std::min(l.pieces, 2 * kNumSMs)); parts += grid.back(); }
  const Tensor partial = new_tensor({std::max(parts, 1)}, at::kDouble, norm.device());
  double* sums = partial.data_ptr<double>();
  for (size_t i = 0, at = 0; i < lists.size(); at += grid[i++]) {
    launch(clip_norm_kernel<CAP>, grid[i], CLIP_THREADS, 0, stream, lists[i], sums + at);
    count_launch();
  }
  if (scale && !lists.empty()) {
    for (size_t i = 0; i < lists.size(); ++i) {
      launch(clip_scale_kernel<CAP>, grid[i], CLIP_THREADS, 0, stream, lists[i], (const double*)sums, parts, (float)max_norm, i == 0 ? norm.data_ptr<float>() : nullptr);
      count_launch();
    }
  } else {
    launch(clip_total_kernel, 1, CLIP_THREADS, 0, stream, (const double*)sums, parts, norm.data_ptr<float>());
    count_launch();
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

struct Range { uintptr_t begin, end; size_t owner; };

}  // namespace

// The norm of all tensors together.  With `scale` the scaled tensors go to `outs`, or in place where there are none.
Tensor clip_grad_norm(at::TensorList grads, at::TensorList outs, double max_norm, bool scale) {
  TORCH_CHECK_VALUE(!grads.empty(), "clip_grad_norm: at least one gradient required");
  TORCH_CHECK_VALUE(max_norm > 0, "clip_grad_norm: max_norm must be positive");
  TORCH_CHECK_VALUE(outs.empty() || outs.size() == grads.size(), "clip_grad_norm: as many results as gradients required");
  const auto device = grads[0].device();
  TORCH_CHECK_VALUE(device.is_cuda(), "clip_grad_norm: CUDA tensors required");
  long long elements = 0;
  std::vector<Range> written, read;
  written.reserve(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& g = grads[i];
    const auto type = g.scalar_type();
    TORCH_CHECK_VALUE(g.device() == device, "clip_grad_norm: gradients on one device required");
    TORCH_CHECK_VALUE(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, "clip_grad_norm: fp32, bf16 or fp16 gradients required");
    TORCH_CHECK_VALUE(g.is_non_overlapping_and_dense(), "clip_grad_norm: gradients without gaps or overlaps in memory required");
    if (!outs.empty()) {
      const Tensor& o = outs[i];
      TORCH_CHECK_VALUE(o.device() == device && o.scalar_type() == type && o.sizes() == g.sizes() && (o.strides() == g.strides() || (o.is_contiguous() && g.is_contiguous())),
                  "clip_grad_norm: a result has its gradient's device, type, shape and layout");
    }
    if (!g.numel()) continue;
    elements += g.numel();
    if (scale) {
      const Tensor& o = outs.empty() ? g : outs[i];
      const auto at = reinterpret_cast<uintptr_t>(o.data_ptr());
      written.push_back({at, at + o.nbytes(), i});
      if (!outs.empty() && o.data_ptr() != g.data_ptr()) read.push_back({reinterpret_cast<uintptr_t>(g.data_ptr()), reinterpret_cast<uintptr_t>(g.data_ptr()) + g.nbytes(), i});
    }
  }
  // What is written twice, or written while another tensor's values are still to be read, has no defined result
  const auto by_begin = [](const Range& a, const Range& b) { return a.begin < b.begin; };
  if (!std::is_sorted(written.begin(), written.end(), by_begin)) std::sort(written.begin(), written.end(), by_begin);
  for (size_t i = 1; i < written.size(); ++i) TORCH_CHECK_VALUE(written[i].begin >= written[i - 1].end, "clip_grad_norm: a tensor, or a part of one, is listed twice");
  for (const Range& r : read) {
    auto it = std::lower_bound(written.begin(), written.end(), r, [](const Range& a, const Range& b) { return a.end <= b.begin; });
    TORCH_CHECK_VALUE(it == written.end() || it->begin >= r.end, "clip_grad_norm: a result overlaps a gradient that is not its own");
  }
  const c10::cuda::CUDAGuard guard(device);
  auto norm = new_tensor({}, at::kFloat, device);
  auto stream = at::cuda::getCurrentCUDAStream();
  const int piece = piece_size(elements);
  if (grads.size() <= 64) run<64>(grads, outs, piece, max_norm, scale, norm, stream);
  else run<512>(grads, outs, piece, max_norm, scale, norm, stream);
  if (scale)
    for (const Tensor& o : outs.empty() ? grads : outs)
      if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();        // autograd notices that a saved tensor was changed
  return norm;
}

}  // namespace q38
