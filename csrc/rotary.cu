// Rotary positions of queries and keys in one launch.
//
//   pair i of a head at position t:  a' = m (a cos(t f_i) - b sin(t f_i)),  b' = m (b cos(t f_i) + a sin(t f_i))
//
// where the pair is (x[i], x[i + r/2]) or, interleaved, (x[2i], x[2i + 1]); elements from r on pass through.  The gradient is the same with
// the opposite angle.  Frequencies f come from the caller in 64 bits (however they were scaled) and angles are reduced to turns in 64 bits: at
// position 10^6 an angle in 32 bits is off by 0.03.
//
// Bound by memory: every element is read and written once.  A CTA takes a few tokens, makes their cosines and sines once for all heads (shared memory), and
// walks the tokens' heads in pieces of 16 bytes: a piece of each half, two neighbouring pieces of an interleaved head, or two that pass through.
// Tensors are addressed by their strides, so packed projections and head-major tensors are read in place.
// Replayed on a B200: 65537 tokens of 10 heads of 128, all rotated, 61 us (5.5 TB/s, 84 % of the copy bandwidth); 16384 tokens of 24 heads of 64, a quarter rotated, out of
// a packed projection 20.7 us (4.9 TB/s).  fp32: 105 us (98 %) and 35.3 (87 %).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "packs.cuh"
#include "host.h"
#include "launch.cuh"
#include "training.h"

namespace q38 {

// Quotients by a number that is fixed for the launch: two multiplications, exact for any 32-bit dividend
struct Divisor {
  uint64_t inverse;                // floor(2^64 / d) + 1, or 0 for d = 1
  uint32_t d;
};
__device__ __forceinline__ int quotient(int n, const Divisor& by) {
  const uint64_t low = (uint64_t)(uint32_t)n * (uint32_t)by.inverse, high = (uint64_t)(uint32_t)n * (uint32_t)(by.inverse >> 32) + (low >> 32);
  return by.d == 1 ? n : (int)(high >> 32);
}

struct RotarySide {                // queries or keys: strides of batch, token and head
  const void* in;
  void* out;
  long long in_b, in_s, in_h, out_b, out_s, out_h;
};
struct RotaryArgs {
  RotarySide q, k;
  const double* freq;              // [r / 2]
  const void* pos;                 // [batch or 1, tokens], 32 or 64 bits
  long long pos_b, pos_s, tokens;  // tokens = batch * seq
  Divisor units, heads, half;      // units per head; heads of both sides; pairs per head
  int seq, q_heads, dim, per_cta, pos64;
  float magnitude, sign;
};

constexpr int ROT_THREADS = 256, ROT_BATCH = 2, ROT_TOKENS = 64;

// VEC == 1: a unit is one pair, or one element that passes through.  VEC > 1: two packs: one of each half, two neighbours of an interleaved head, or two
// (the last unit perhaps one) that pass through.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(ROT_THREADS, 5) rotary_kernel(const __grid_constant__ RotaryArgs p) {
  grid_wait();
  // cos, sin [per_cta][VEC][half / VEC]: the units of neighbouring lanes side by side (in order of pairs, a read would meet sixteen times in a bank)
  extern __shared__ float2 turns[];
  __shared__ long long base_of[ROT_TOKENS][4];           // where a token's queries and keys begin, in and out
  const long long first = (long long)blockIdx.x * p.per_cta;
  const int count = (int)min((long long)p.per_cta, p.tokens - first), half = p.half.d;
  if (threadIdx.x < count) {
    const long long token = first + threadIdx.x, b = token / p.seq, s = token - b * p.seq;
    base_of[threadIdx.x][0] = b * p.q.in_b + s * p.q.in_s;
    base_of[threadIdx.x][1] = b * p.q.out_b + s * p.q.out_s;
    base_of[threadIdx.x][2] = b * p.k.in_b + s * p.k.in_s;
    base_of[threadIdx.x][3] = b * p.k.out_b + s * p.k.out_s;
  }
  for (int i = threadIdx.x; i < count * half; i += ROT_THREADS) {
    const int local = quotient(i, p.half), f = i - local * half;
    const long long token = first + local, b = p.pos_b ? token / p.seq : 0, at = p.pos_b ? b * p.pos_b + (token - b * p.seq) * p.pos_s : token % p.seq * p.pos_s;
    const double t = p.pos64 ? (double)reinterpret_cast<const long long*>(p.pos)[at] : (double)reinterpret_cast<const int*>(p.pos)[at];
    const double turn = t * (p.freq[f] * 0.15915494309189533576888);            // 1 / (2 pi)
    float sn, cs;
    sincospif(2.f * (float)(turn - rint(turn)), &sn, &cs);
    turns[local * half + f % VEC * (half / VEC) + f / VEC] = make_float2(cs * p.magnitude, sn * p.magnitude * p.sign);
  }
  __syncthreads();

  const int rot_units = VEC == 1 ? half : half / VEC, units = p.units.d, heads = p.heads.d;
  const int total = count * heads * units;
  for (int base = threadIdx.x; base < total; base += ROT_THREADS * ROT_BATCH) {
    Pack<T, VEC> v[ROT_BATCH][2];
    T* dst[ROT_BATCH];
    int second[ROT_BATCH], angle[ROT_BATCH];             // distance of the second pack (0: there is none); first angle, or -1 where elements pass through
#pragma unroll
    for (int j = 0; j < ROT_BATCH; ++j) {
      const int i = base + j * ROT_THREADS;
      dst[j] = nullptr;
      if (i < total) {
        const int row = quotient(i, p.units), unit = i - row * units, local = quotient(row, p.heads), head = row - local * heads;
        int at;
        if (unit < rot_units) {
          at = INTERLEAVED ? 2 * VEC * unit : VEC * unit;
          second[j] = INTERLEAVED ? VEC : half;
          angle[j] = local * half + unit;
        } else {
          const int rest = unit - rot_units;
          at = 2 * half + (VEC == 1 ? rest : 2 * VEC * rest);
          second[j] = VEC > 1 && at + VEC < p.dim ? VEC : 0;
          angle[j] = -1;
        }
        const bool key = head >= p.q_heads;
        const RotarySide& side = key ? p.k : p.q;
        const int h = key ? head - p.q_heads : head;
        const T* src = reinterpret_cast<const T*>(side.in) + base_of[local][key ? 2 : 0] + h * side.in_h + at;
        dst[j] = reinterpret_cast<T*>(side.out) + base_of[local][key ? 3 : 1] + h * side.out_h + at;
        v[j][0] = load_pack<T, VEC>(src);
        if (second[j]) v[j][1] = load_pack<T, VEC>(src + second[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < ROT_BATCH; ++j) {
      if (dst[j] != nullptr) {
        if (angle[j] >= 0) {
          float f[2][VEC];
          unpack(v[j][0], f[0]);
          unpack(v[j][1], f[1]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float2 cs = turns[angle[j] + e * (half / VEC)];
            float& lo = INTERLEAVED && VEC > 1 ? f[2 * e / VEC][2 * e % VEC] : f[0][e];
            float& hi = INTERLEAVED && VEC > 1 ? f[(2 * e + 1) / VEC][(2 * e + 1) % VEC] : f[1][e];
            const float a = lo, b = hi;
            lo = a * cs.x - b * cs.y;
            hi = b * cs.x + a * cs.y;
          }
          v[j][0] = pack<T, VEC>(f[0]);
          v[j][1] = pack<T, VEC>(f[1]);
        }
        store_pack<T, VEC>(dst[j], v[j][0]);
        if (second[j]) store_pack<T, VEC>(dst[j] + second[j], v[j][1]);
      }
    }
  }
}

namespace {

using at::Tensor;

// A tensor of t's shape with its order of dimensions in memory
Tensor like(const Tensor& t) {
  const bool in_order = t.stride(0) >= t.stride(1) && t.stride(1) >= t.stride(2) && t.stride(2) >= t.stride(3);
  return in_order ? new_tensor(t.sizes(), t.scalar_type(), t.device()) : at::empty_like(t);
}
Tensor with_columns(const Tensor& t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); }

RotarySide side_of(const Tensor& in, const Tensor& out) {
  return {in.data_ptr(), out.data_ptr(), in.stride(0), in.stride(1), in.stride(2), out.stride(0), out.stride(1), out.stride(2)};
}
// The largest power of two up to 8 that divides a tensor's address (in elements) and strides
int packs_fit(const Tensor& t) {
  const uintptr_t size = t.element_size();
  uintptr_t bits = reinterpret_cast<uintptr_t>(t.data_ptr()) / size | (uintptr_t)t.stride(0) | (uintptr_t)t.stride(1) | (uintptr_t)t.stride(2) | 8;
  return (int)(bits & (~bits + 1));
}

Divisor divisor(int d) { return {d > 1 ? ~0ull / d + 1 : 0, (uint32_t)d}; }

template <typename T, int VEC>
void launch_rotary(RotaryArgs& p, bool interleaved, cudaStream_t stream) {
  const int half = (int)p.half.d, rest = p.dim - 2 * half;
  p.units = divisor(VEC > 1 ? half / VEC + (rest / VEC + 1) / 2 : half + rest);
  // Tokens per CTA: eight units per thread, fewer where that leaves an SM without work; their angles fit 32 KB
  const long long per_token = (long long)p.heads.d * p.units.d;
  long long n = std::min<long long>(ROT_TOKENS, std::max<long long>(1, 8 * ROT_THREADS / per_token));
  n = std::min(n, std::max<long long>(1, p.tokens / (2 * kNumSMs)));
  // whole rounds of the five blocks that an SM holds (16384 tokens of 24 heads of 64: 781 blocks, six per cent of them in a second round, 21.9 us; 713 blocks 20.7)
  const long long slots = 5 * kNumSMs, rounds = std::max<long long>(1, (p.tokens + n * slots / 2) / (n * slots));
  if (p.tokens > n * slots / 2) n = std::min<long long>(ROT_TOKENS, (p.tokens + rounds * slots - 1) / (rounds * slots));
  if (half) n = std::max<long long>(1, std::min<long long>(n, 4096 / half));
  p.per_cta = (int)n;
  const long long grid = (p.tokens + n - 1) / n;
  TORCH_CHECK_VALUE(grid < (1ll << 31) && per_token * n < (1ll << 30), "rotary: tensor too large");
  const size_t smem = size_t(p.per_cta) * half * sizeof(float2);
  auto go = [&](auto kernel) {
    launch(kernel, (unsigned)grid, ROT_THREADS, smem, stream, p);
  };
  if (interleaved) go(rotary_kernel<T, VEC, true>); else go(rotary_kernel<T, VEC, false>);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
}

// Elements per access: as many as 16 bytes hold, or the largest half of that which divides the rotated half, the head and all distances and addresses
// (2 x 4096 x 40 heads of 80, 20 rotated: 97 us by single elements, 36 by pairs).
template <typename T>
void by_width(RotaryArgs& p, int fit, bool interleaved, cudaStream_t stream) {
  const int half = (int)p.half.d;
  auto ok = [&](int vec) { return fit % vec == 0 && p.dim % vec == 0 && half % vec == 0; };
  if (sizeof(T) == 2 && ok(8)) launch_rotary<T, 16 / sizeof(T)>(p, interleaved, stream);
  else if (ok(4)) launch_rotary<T, 4>(p, interleaved, stream);
  else if (ok(2)) launch_rotary<T, 2>(p, interleaved, stream);
  else launch_rotary<T, 1>(p, interleaved, stream);
}

}  // namespace

// q, k [batch, seq, heads, dim] of any strides -> tensors of their layout (either may be absent).  `sign` -1: the gradient.
std::pair<Tensor, Tensor> rotary_apply(const Tensor& q_in, const Tensor& k_in, const Tensor& pos, const Tensor& freq, double magnitude, bool interleaved, double sign) {
  const Tensor& any = q_in.defined() ? q_in : k_in;
  const c10::cuda::CUDAGuard guard(any.device());
  Tensor q, k, qo, ko;
  if (q_in.defined()) { q = with_columns(q_in); qo = like(q); }
  if (k_in.defined()) { k = with_columns(k_in); ko = like(k); }
  RotaryArgs p{};
  int fit = 8;
  if (q.defined()) { p.q = side_of(q, qo); fit = std::min({fit, packs_fit(q), packs_fit(qo)}); }
  if (k.defined()) { p.k = side_of(k, ko); fit = std::min({fit, packs_fit(k), packs_fit(ko)}); }
  p.q_heads = q.defined() ? (int)q.size(2) : 0;
  p.heads = divisor(p.q_heads + (k.defined() ? (int)k.size(2) : 0));
  p.seq = (int)any.size(1); p.tokens = any.size(0) * any.size(1); p.dim = (int)any.size(3); p.half = divisor((int)freq.size(0));
  p.freq = freq.data_ptr<double>(); p.pos = pos.data_ptr(); p.pos64 = pos.scalar_type() == at::kLong;
  p.pos_b = pos.dim() == 2 && pos.size(0) > 1 ? pos.stride(0) : 0; p.pos_s = pos.stride(-1);
  p.magnitude = (float)magnitude; p.sign = (float)sign;
  if (p.tokens > 0 && p.heads.d > 0 && p.dim > 0) {
    auto stream = at::cuda::getCurrentCUDAStream();
    if (any.scalar_type() == at::kBFloat16) by_width<__nv_bfloat16>(p, fit, interleaved, stream);
    else if (any.scalar_type() == at::kHalf) by_width<__half>(p, fit, interleaved, stream);
    else by_width<float>(p, fit, interleaved, stream);
  }
  return {qo, ko};
}

void rotary_check(const Tensor& q, const OptTensor& k, const Tensor& pos, const Tensor& freq) {
  TORCH_CHECK_VALUE(q.is_cuda() && q.dim() == 4 && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat),
              "rotary: bf16, fp16 or fp32 CUDA tensors [batch, seq, heads, dim] required");
  TORCH_CHECK_VALUE(!k.has_value() || (k->device() == q.device() && k->scalar_type() == q.scalar_type() && k->dim() == 4 && k->size(0) == q.size(0) && k->size(1) == q.size(1) && k->size(3) == q.size(3)),
              "rotary: keys have the type, device, batch, length and head size of the queries");
  TORCH_CHECK_VALUE(pos.device() == q.device() && (pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt) &&
              ((pos.dim() == 1 && pos.size(0) == q.size(1)) || (pos.dim() == 2 && pos.size(1) == q.size(1) && (pos.size(0) == q.size(0) || pos.size(0) == 1))),
              "rotary: whole positions [seq], [1, seq] or [batch, seq] on the queries' device required");
  TORCH_CHECK_VALUE(freq.device() == q.device() && freq.scalar_type() == at::kDouble && freq.dim() == 1 && 2 * freq.size(0) <= q.size(3),
              "rotary: 64-bit frequencies on the queries' device, at most half a head of them, required");
  TORCH_CHECK_VALUE(q.size(1) < (1ll << 31) && q.size(3) <= 8192, "rotary: sequence or head too long");
}

}  // namespace q38
