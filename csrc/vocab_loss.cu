// Softmax cross entropy over a large vocabulary in pieces of the vocabulary, without keeping the logits.
//
//   z = h W^T,  lse_t = ln sum_v e^z_tv,  loss_t = lse_t - z_t,target;   dz = s_t (e^(z - lse) - onehot),  dh = dz W,  dW = dz^T h
//
// Forward: the product's tiles are reduced where they arise.  Each 128 x bn accumulator is read from tensor memory once, and leaves per row and half tile the
// pair (k, s) with sum = s 2^k and the target's logit; a small kernel joins the pairs.  Nothing of size rows x vocabulary is written.
// Backward: for one piece of the vocabulary after the other the same tiles are formed again, turned into dz (bf16, a workspace of one piece) and
// multiplied by W and h on the framework's GEMM.  The logits stay fp32 in tensor memory: storing them in bf16 (half a step of 2^-9 of a logit of ten) would put an
// error of 2 % into a probability.  dz is rounded to bf16 because the tensor cores take it so; its target entry is -1 + p, whose rounding is small.
//
// The kernel follows csrc/gemm_persistent.cu: one CTA per SM, warp 0 loads by TMA, one lane of warp 1 issues the MMAs into one of two accumulators, and eight
// warps (two warpgroups on alternate 32-column chunks) read the other.  Tiles are walked with the rows fastest, in groups of rows whose hidden states
// stay in L2: all SMs work on the same few columns of W, which so comes from memory once per group.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "f32x2.cuh"
#include "ptx.cuh"
#include "host.h"
#include "launch.cuh"

namespace q38 {

constexpr int V_BM = 128, V_BK = 64, V_MAX_STAGES = 8, V_THREADS = 320, V_ACC_COLS = 256;
constexpr float V_LOG2E = 1.44269504088896340736f;
constexpr long long V_IGNORE = -100;

struct VocabArgs {
  int rows, cols, K, bn;                       // cols: of this piece
  int tiles_m, tiles_n, group_m, total_kb, items, stages, first_col, vocab;
  const long long* target;
  float2* partial;                             // [2 tiles_n][rows]: (k, s) of a half tile
  float* target_logit;                         // [rows]
  const float *lse2, *upstream, *count;        // backward: log2 of the row's sum; gradient of each row (or of all); divisor (or null)
  int upstream_step;
  int* err;
};

template <bool GRAD>
__global__ void __launch_bounds__(V_THREADS) vocab_tiles_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC,
                                                                VocabArgs p) {
  grid_wait();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const int A_BYTES = V_BM * 128, B_BYTES = p.bn * 128, STAGE_BYTES = A_BYTES + B_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + p.stages * STAGE_BYTES);
  uint64_t* empty = full + V_MAX_STAGES;
  uint64_t* acc_full = empty + V_MAX_STAGES;        // [2]
  uint64_t* acc_empty = acc_full + 2;               // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  uint8_t* stage_out = smem + p.stages * STAGE_BYTES + 1024;     // [8 warps][2 buffers][32 rows x 64 bytes]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tmA);
    ptx::prefetch_tensormap(&tmB);
    if (GRAD) ptx::prefetch_tensormap(&tmC);
    for (int s = 0; s < p.stages; ++s) { ptx::mbar_init(&full[s], 1); ptx::mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { ptx::mbar_init(&acc_full[a], 1); ptx::mbar_init(&acc_empty[a], 8); }   // eight epilogue warps release an accumulator
    ptx::fence_barrier_init();
  }
  if (warp == 1) { ptx::tmem_alloc(tmem_slot, 512); ptx::tmem_relinquish(); }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  auto decode = [&](int w, int& tm, int& tn) {
    const int per_group = p.group_m * p.tiles_n, g = w / per_group, r = w - g * per_group;
    const int gm = min(p.group_m, p.tiles_m - g * p.group_m);
    tn = r / gm;
    tm = g * p.group_m + r - tn * gm;
  };
  auto advance = [&](int& s, uint32_t& odd) { if (++s == p.stages) { s = 0; odd ^= 1; } };

  if (warp == 0) {
    if (ptx::elect_one()) {
      int s = 0;
      uint32_t odd = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < p.items && ok; w += gridDim.x) {
        int tm, tn;
        decode(w, tm, tn);
        for (int kb = 0; kb < p.total_kb; ++kb, advance(s, odd)) {
          if (!ptx::mbar_wait(&empty[s], odd ^ 1, 1u << 20)) { report_error(p.err, ERR_MMA_WAIT); ok = false; break; }
          uint8_t* a_dst = smem + s * STAGE_BYTES;
          ptx::mbar_expect_tx(&full[s], STAGE_BYTES);
          ptx::tma_load_3d(a_dst, &tmA, &full[s], kb * V_BK, tm * V_BM, 0);
          ptx::tma_load_3d(a_dst + A_BYTES, &tmB, &full[s], kb * V_BK, tn * p.bn, 0);
        }
      }
    }
  } else if (warp == 1) {
    if (ptx::elect_one()) {
      const uint32_t idesc = ptx::umma_idesc_bf16(V_BM, p.bn, false, false);
      int s = 0;
      uint32_t odd = 0, tile = 0;
      bool ok = true;
      for (int w = blockIdx.x; w < p.items && ok; w += gridDim.x, ++tile) {
        const int acc = tile & 1;
        if (!ptx::mbar_wait(&acc_empty[acc], ((tile >> 1) & 1) ^ 1, 1u << 22)) { report_error(p.err, ERR_EPILOGUE_WAIT); ok = false; break; }
        ptx::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * V_ACC_COLS;
        for (int kb = 0; kb < p.total_kb; ++kb, advance(s, odd)) {
          if (!ptx::mbar_wait(&full[s], odd, 1u << 20)) { report_error(p.err, ERR_TMA_WAIT); ok = false; break; }
          ptx::tc_fence_after();
          const uint32_t a_base = ptx::smem_u32(smem + s * STAGE_BYTES), b_base = a_base + A_BYTES;
#pragma unroll
          for (int j = 0; j < V_BK / 16; ++j)
            ptx::umma_f16(d_tmem, ptx::umma_smem_desc_sw128(a_base + j * 32, 0, 1024), ptx::umma_smem_desc_sw128(b_base + j * 32, 0, 1024), idesc, (kb | j) != 0);
          ptx::umma_commit(&empty[s]);
        }
        if (ok) ptx::umma_commit(&acc_full[acc]);
      }
    }
  } else {
    const int quarter = warp & 3, ew = warp - 2, group = ew >> 2;
    uint32_t tile = 0, chunk = 0;
    bool ok = true;
    const uint64_t l2e = pair2(V_LOG2E, V_LOG2E);
    for (int w = blockIdx.x; w < p.items && ok; w += gridDim.x, ++tile) {
      int tm, tn;
      decode(w, tm, tn);
      const int acc = tile & 1, row0 = tm * V_BM + quarter * 32, row = row0 + lane, n0 = tn * p.bn;
      const bool live = row < p.rows;
      // the row's values are on their way while the accumulator is
      const long long tgt = live ? p.target[row] : V_IGNORE;
      const long long rel = tgt - p.first_col - n0;                // column of the target in this tile, if it is there
      const bool inside = tgt >= 0 && tgt < p.vocab;
      const int hit = inside && rel >= 0 && rel < p.bn && rel < p.cols - n0 ? (int)rel : -1;
      float lse2 = 0.f, scale = 0.f;
      if (GRAD && inside) {
        lse2 = p.lse2[row];
        scale = p.upstream[(long long)row * p.upstream_step];
        if (p.count != nullptr) scale = __fdividef(scale, *p.count);
      }
      if (!ptx::mbar_wait_warp(&acc_full[acc], (tile >> 1) & 1, 1u << 22)) { report_error(p.err, ERR_EPILOGUE_WAIT); ok = false; break; }
      ptx::tc_fence_after();
      const uint32_t t_addr = tmem_base + acc * V_ACC_COLS + (uint32_t(quarter * 32) << 16);
      float k = -INFINITY, sum = 0.f, found = 0.f;
      auto reduce = [&](uint32_t (&r)[32], int c0) {
        if (n0 + c0 + 32 > p.cols) {                               // behind the last column
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (n0 + c0 + e >= p.cols) r[e] = 0xff800000u;
        }
        float m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = __uint_as_float(r[e]);
#pragma unroll
        for (int e = 4; e < 32; ++e) m[e & 3] = fmaxf(m[e & 3], __uint_as_float(r[e]));
        const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        const float kn = fmaxf(k, top * V_LOG2E), ref = kn == -INFINITY ? 0.f : kn;
        const uint64_t minus = pair2(-ref, -ref);
        uint64_t part[2] = {pair2(sum * exp2_approx(k - ref), 0.f), pair2(0.f, 0.f)};
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = unpair(fma2(pair2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), l2e, minus));
          part[(e >> 1) & 1] = add2(part[(e >> 1) & 1], pair2(exp2_approx(x.x), exp2_approx(x.y)));
        }
        const float2 s = unpair(add2(part[0], part[1]));
        sum = s.x + s.y;
        k = kn;
        if (__any_sync(0xffffffffu, hit >= c0 && hit < c0 + 32)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (hit == c0 + e) found = __uint_as_float(r[e]);
        }
      };
      auto emit = [&](uint32_t (&r)[32], int c0) {
        const uint64_t minus = pair2(-lse2, -lse2);
        const bool dead = scale == 0.f;                            // ignored, or no gradient: zeros whatever the logits are
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 x = unpair(fma2(pair2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), l2e, minus));
          v[e] = exp2_approx(x.x);
          v[e + 1] = exp2_approx(x.y);
        }
        if (__any_sync(0xffffffffu, hit >= c0 && hit < c0 + 32)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (hit == c0 + e) v[e] -= 1.f;
        }
        uint8_t* buf = stage_out + (ew * 2 + (chunk & 1)) * 2048;
        if (lane == 0) ptx::bulk_wait_read<1>();                   // the store issued two chunks ago has read this buffer
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t wd[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) wd[e] = dead ? 0u : bf16_pair(make_float2(v[q * 8 + 2 * e] * scale, v[q * 8 + 2 * e + 1] * scale));
          *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = make_uint4(wd[0], wd[1], wd[2], wd[3]);
        }
        ptx::fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          if (n0 + c0 < p.cols && row0 < p.rows) ptx::tma_store_3d(&tmC, buf, n0 + c0, row0, 0);
          ptx::bulk_commit();                                      // possibly empty: keeps the buffer accounting uniform
        }
        ++chunk;
      };
      auto use = [&](uint32_t (&r)[32], int c0) { if constexpr (GRAD) emit(r, c0); else reduce(r, c0); };
      uint32_t ra[32], rb[32];
      int c0 = 32 * group;
      ptx::tmem_ld_32x32b_x32(t_addr + c0, ra);                    // bn is a multiple of 64: every warp has a chunk
      for (; c0 < p.bn; c0 += 128) {                               // two chunks of this warpgroup per trip, the next one's read in flight
        ptx::tmem_ld_wait();
        if (c0 + 64 < p.bn) ptx::tmem_ld_32x32b_x32(t_addr + c0 + 64, rb);
        use(ra, c0);
        if (c0 + 64 < p.bn) {
          ptx::tmem_ld_wait();
          if (c0 + 128 < p.bn) ptx::tmem_ld_32x32b_x32(t_addr + c0 + 128, ra);
          use(rb, c0 + 64);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&acc_empty[acc]);
      if (!GRAD && live) {
        p.partial[(long long)(2 * tn + group) * p.rows + row] = make_float2(k, sum);
        if (hit >= 0 && ((hit >> 5) & 1) == group) p.target_logit[row] = found;
      }
    }
    if (GRAD && lane == 0) ptx::bulk_wait<0>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) ptx::tmem_dealloc(tmem_base, 512);
}

// lse2[row] = log2 of the row's sum and loss[row], from the tiles' pairs: 32 rows per CTA, eight threads per row in strides of eight pairs, joined in order.
// A target outside the vocabulary that is not the ignored one is an error: it is reported, and the row counts as ignored.
__global__ void __launch_bounds__(256) vocab_join_kernel(const float2* __restrict__ partial, int parts, int rows, int vocab, const long long* __restrict__ target,
                                                         const float* __restrict__ target_logit, float* __restrict__ lse2, float* __restrict__ loss, int* err) {
  grid_wait();
  __shared__ float2 part[8][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, row = blockIdx.x * 32 + x;
  auto join = [](float2 a, float2 b) {
    const float k = fmaxf(a.x, b.x), ref = k == -INFINITY ? 0.f : k;
    return make_float2(k, a.y * exp2_approx(a.x - ref) + b.y * exp2_approx(b.x - ref));
  };
  float2 v = make_float2(-INFINITY, 0.f);
  if (row < rows) {
    int i = y;
    for (; i + 24 < parts; i += 32) {
      const float2 a = partial[(long long)i * rows + row], b = partial[(long long)(i + 8) * rows + row], c = partial[(long long)(i + 16) * rows + row], d = partial[(long long)(i + 24) * rows + row];
      v = join(v, join(join(a, b), join(c, d)));
    }
    for (; i < parts; i += 8) v = join(v, partial[(long long)i * rows + row]);
  }
  part[y][x] = v;
  __syncthreads();
  if (y != 0 || row >= rows) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) v = join(v, part[q][x]);
  const double l2 = (double)v.x + log2((double)v.y);
  const long long tgt = target[row];
  const bool inside = tgt >= 0 && tgt < vocab;
  if (!inside && tgt != V_IGNORE) report_error(err, ERR_BOUNDS);
  lse2[row] = (float)l2;
  loss[row] = inside ? (float)(l2 * 0.69314718055994530942 - (double)target_logit[row]) : 0.f;
}

// Sum of all losses and number of rows that count, by one CTA in a fixed order: out[0] the sum or the mean over those rows, out[1] that number (at least 1).
__global__ void __launch_bounds__(1024) vocab_sum_kernel(const float* __restrict__ loss, const long long* __restrict__ target, int rows, int vocab, bool mean, float* out) {
  grid_wait();
  __shared__ double sums[32];
  __shared__ int counts[32];
  double s = 0.0;
  int n = 0;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    s += (double)loss[i];
    n += target[i] >= 0 && target[i] < vocab;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); n += __shfl_xor_sync(0xffffffffu, n, o); }
  if ((threadIdx.x & 31) == 0) { sums[threadIdx.x >> 5] = s; counts[threadIdx.x >> 5] = n; }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 32; ++w) { s += sums[w]; n += counts[w]; }
  n = max(n, 1);
  out[0] = (float)(mean ? s / n : s);
  out[1] = (float)n;
}

// out = sum of `slices` fp32 matrices [rows, cols] (rows of ldp elements), in order, as bf16 or fp32
__global__ void __launch_bounds__(256) vocab_slices_kernel(const float* __restrict__ part, int slices, long long slice, long long rows, int cols, int ldp, void* out, bool bf16) {
  grid_wait();
  const long long n = rows * cols;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / cols, at = r * ldp + (i - r * cols);
    float s = part[at];
    for (int k = 1; k < slices; ++k) s += part[k * slice + at];
    if (bf16) reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(s);
    else reinterpret_cast<float*>(out)[i] = s;
  }
}

namespace {

using at::Tensor;

// A 2-D bf16 tensor whose rows TMA accepts (contiguous, a multiple of 16 bytes apart, on 16 bytes); others are copied into padded rows
Tensor tma_rows(const Tensor& t) {
  const int64_t n = t.size(1);
  if (t.stride(1) == 1 && t.stride(0) >= n && t.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return t;
  auto view = at::empty({t.size(0), (n + 7) / 8 * 8}, t.options()).narrow(1, 0, n);
  view.copy_(t);
  return view;
}

// Tiles of 256 columns, narrower ones where there would not be one for every SM
int tile_width(int64_t rows, int64_t cols) {
  int bn = 256;
  while (bn > 64 && (rows + V_BM - 1) / V_BM * ((cols + bn - 1) / bn) < kNumSMs) bn /= 2;
  return bn;
}

template <bool GRAD>
void launch_tiles(const Tensor& h, const Tensor& w, int64_t first_col, int64_t cols, VocabArgs& p, const CUtensorMap* out, cudaStream_t stream) {
  p.rows = (int)h.size(0); p.K = (int)h.size(1); p.cols = (int)cols; p.first_col = (int)first_col; p.vocab = (int)w.size(0);
  p.tiles_m = (p.rows + V_BM - 1) / V_BM;
  p.bn = tile_width(p.rows, cols);
  p.tiles_n = (int)((cols + p.bn - 1) / p.bn);
  p.items = p.tiles_m * p.tiles_n;
  p.total_kb = (p.K + V_BK - 1) / V_BK;
  // Rows whose hidden states take 24 MB at most stay in L2 beside the columns in use
  p.group_m = (int)std::max<int64_t>(1, std::min<int64_t>(p.tiles_m, (24 << 20) / (V_BM * 2 * (int64_t)p.K)));
  const int stage = V_BM * 128 + p.bn * 128, fixed = 1024 + 1024 + (GRAD ? 8 * 2 * 2048 : 0);
  p.stages = std::min(V_MAX_STAGES, (227 * 1024 - fixed) / stage);
  const int smem = p.stages * stage + fixed;
  const CUtensorMap ta = make_tmap_box(h.data_ptr(), 2, p.K, p.rows, 1, h.stride(0), 0, V_BM, 128);
  const CUtensorMap tb = make_tmap_box(reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()) + first_col * w.stride(0), 2, p.K, cols, 1, w.stride(0), 0, p.bn, 128);
  auto kernel = vocab_tiles_kernel<GRAD>;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
  launch(kernel, (unsigned)std::min(p.items, kNumSMs), V_THREADS, smem, stream, ta, tb, out ? *out : ta, p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
}

void check(const Tensor& h, const Tensor& w, const Tensor& target) {
  TORCH_CHECK(h.is_cuda() && h.dim() == 2 && h.scalar_type() == at::kBFloat16 && w.device() == h.device() && w.dim() == 2 && w.scalar_type() == at::kBFloat16 && w.size(1) == h.size(1),
              "vocab_loss: bf16 hidden states [rows, hidden] and weight [vocabulary, hidden] on one CUDA device required");
  TORCH_CHECK(target.device() == h.device() && target.dim() == 1 && target.scalar_type() == at::kLong && target.is_contiguous() && target.size(0) == h.size(0),
              "vocab_loss: contiguous int64 targets, one per row, required");
  TORCH_CHECK(h.size(1) > 0 && w.size(0) > 0, "vocab_loss: a hidden size and a vocabulary of at least one required");
  // tiles are counted and columns addressed in 32 bits
  TORCH_CHECK(h.size(0) < (1ll << 24) && w.size(0) < (1ll << 24) && h.size(1) < (1ll << 24) && ((h.size(0) + 127) / 128) * ((w.size(0) + 63) / 64) < (1ll << 30), "vocab_loss: too many rows or columns");
}

}  // namespace

// reduction: 0 none, 1 sum, 2 mean over the rows that count.  Returns {loss ([rows] or 0-dim), lse2 [rows], count (one element; empty without a reduction)}.
std::vector<Tensor> vocab_loss_fwd(const Tensor& hidden, const Tensor& weight, const Tensor& target, int64_t reduction, const Tensor& err) {
  check(hidden, weight, target);
  const c10::cuda::CUDAGuard guard(hidden.device());
  const auto f32 = hidden.options().dtype(at::kFloat);
  const int64_t rows = hidden.size(0), vocab = weight.size(0);
  auto loss = at::empty({rows}, f32), lse2 = at::empty({rows}, f32);
  auto out = at::empty({reduction ? 2 : 0}, f32);
  auto stream = at::cuda::getCurrentCUDAStream();
  if (rows) {
    const Tensor h = tma_rows(hidden), w = tma_rows(weight);
    VocabArgs p{};
    const int bn = tile_width(rows, vocab);
    auto partial = at::empty({2 * ((vocab + bn - 1) / bn), rows, 2}, f32);
    auto logit = at::empty({rows}, f32);
    p.target = reinterpret_cast<const long long*>(target.data_ptr<int64_t>());
    p.partial = reinterpret_cast<float2*>(partial.data_ptr<float>());
    p.target_logit = logit.data_ptr<float>();
    p.err = err.data_ptr<int>();
    launch_tiles<false>(h, w, 0, vocab, p, nullptr, stream);
    launch(vocab_join_kernel, (unsigned)((rows + 31) / 32), 256, 0, stream, (const float2*)p.partial, 2 * p.tiles_n, (int)rows, (int)vocab, p.target, (const float*)p.target_logit,
           lse2.data_ptr<float>(), loss.data_ptr<float>(), p.err);
    count_launch();
  }
  if (reduction == 0) return {loss, lse2, out};
  launch(vocab_sum_kernel, 1, 1024, 0, stream, (const float*)loss.data_ptr<float>(), reinterpret_cast<const long long*>(target.data_ptr<int64_t>()), (int)rows, (int)vocab, reduction == 2,
         out.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
  return {out[0], lse2, out[1]};
}

// g: gradient of the loss ([rows] fp32 without a reduction, one element with one).  Returns {dh (bf16, or fp32 with `fp32_dh`), dW}: undefined where not wanted or, for dW,
// where it was added to `grad` (fp32 [vocabulary, hidden], contiguous).  `workspace`: bytes that dz of one piece may take.
std::vector<Tensor> vocab_loss_bwd(const Tensor& g, const Tensor& hidden, const Tensor& weight, const Tensor& target, const Tensor& lse2, const Tensor& count, int64_t reduction, bool want_dh,
                                   bool fp32_dh, bool want_dw, bool fp32_dw, const c10::optional<Tensor>& grad, int64_t workspace, const Tensor& err) {
  check(hidden, weight, target);
  TORCH_CHECK(g.device() == hidden.device() && g.scalar_type() == at::kFloat && g.is_contiguous() && g.numel() == (reduction ? 1 : hidden.size(0)) && lse2.numel() == hidden.size(0),
              "vocab_loss_bwd: bad gradient");
  const c10::cuda::CUDAGuard guard(hidden.device());
  const int64_t rows = hidden.size(0), K = hidden.size(1), vocab = weight.size(0), Kp = (K + 7) / 8 * 8;
  const auto f32 = hidden.options().dtype(at::kFloat);
  auto stream = at::cuda::getCurrentCUDAStream();
  Tensor dh, dw;
  if (rows == 0) {
    if (want_dh) dh = at::empty({0, K}, fp32_dh ? f32 : hidden.options());
    if (want_dw && !grad.has_value()) dw = at::zeros({vocab, K}, fp32_dw ? f32 : weight.options());
    return {dh, dw};
  }
  const Tensor h = tma_rows(hidden), w = tma_rows(weight);
  // Pieces: as few as the workspace allows, of equal width (whole tiles)
  const int64_t widest = std::max<int64_t>(256, workspace / (2 * rows) / 256 * 256), pieces = (vocab + widest - 1) / widest;
  const int64_t width = std::min((vocab + 7) / 8 * 8, ((vocab + pieces - 1) / pieces + 255) / 256 * 256);
  auto dz_all = at::empty({rows, width}, hidden.options());
  // dh: where its tiles are fewer than the SMs, slices of the piece side by side, added in order at the end
  const int64_t tiles = ((rows + 127) / 128) * ((Kp + 255) / 256);
  const int64_t slice_cols = std::max<int64_t>(256, (std::max<int64_t>(1, width * tiles / kNumSMs) + 63) / 64 * 64);
  const int64_t slices = std::max<int64_t>(1, std::min<int64_t>((width + slice_cols - 1) / slice_cols, kNumSMs));
  const bool direct = want_dh && slices == 1 && pieces == 1;
  Tensor part;
  if (want_dh && !direct) part = at::empty({slices, rows, Kp}, f32);
  if (direct) dh = at::empty({rows, Kp}, fp32_dh ? f32 : hidden.options());
  if (want_dw && !grad.has_value()) dw = at::empty({vocab, Kp}, fp32_dw ? f32 : weight.options());
  VocabArgs p{};
  p.target = reinterpret_cast<const long long*>(target.data_ptr<int64_t>());
  p.lse2 = lse2.data_ptr<float>(); p.upstream = g.data_ptr<float>(); p.upstream_step = reduction ? 0 : 1;
  p.count = reduction == 2 ? count.data_ptr<float>() : nullptr;
  p.err = err.data_ptr<int>();
  for (int64_t at = 0; at < vocab; at += width) {
    const int64_t cols = std::min(width, vocab - at);
    const bool first = at == 0;
    const CUtensorMap tc = make_tmap_box(dz_all.data_ptr(), 2, cols, rows, 1, width, 0, 32, 64);
    launch_tiles<true>(h, w, at, cols, p, &tc, stream);
    const Tensor dz = dz_all.narrow(1, 0, cols), wp = w.narrow(0, at, cols);
    if (direct) {
      gemm_bf16_persistent(dz, wp, dh.narrow(1, 0, K), false, true, 1.0, false, err, -1);
    } else if (want_dh) {
      const int64_t here = slices == 1 ? cols : slice_cols, whole = slices == 1 ? 1 : std::min(slices, cols / here), rest = cols - whole * here;
      if (whole)
        gemm_bf16_persistent(dz_all.as_strided({whole, rows, here}, {here, width, 1}), wp.as_strided({whole, here, K}, {here * w.stride(0), w.stride(0), 1}, wp.storage_offset()),
                             part.narrow(0, 0, whole).narrow(2, 0, K), false, true, 1.0, !first, err, -1);
      // the columns behind the last whole slice: a slice of their own in a first piece, added to the first slice's sum where there is none for them
      if (rest) {
        const bool own = whole < slices;
        gemm_bf16_persistent(dz.narrow(1, whole * here, rest), wp.narrow(0, whole * here, rest), part[own ? whole : 0].narrow(1, 0, K), false, true, 1.0, !(own && first), err, -1);
      }
    }
    if (want_dw) {
      if (grad.has_value()) gemm_bf16_persistent(dz, h, grad->narrow(0, at, cols), true, true, 1.0, true, err, -1);
      else gemm_bf16_persistent(dz, h, dw.narrow(0, at, cols).narrow(1, 0, K), true, true, 1.0, false, err, -1);
    }
  }
  if (want_dh && !direct) {
    dh = at::empty({rows, K}, fp32_dh ? f32 : hidden.options());
    launch(vocab_slices_kernel, (unsigned)std::min<int64_t>((rows * K + 255) / 256, kNumSMs * 8), 256, 0, stream, (const float*)part.data_ptr<float>(), (int)slices, (long long)(rows * Kp),
           (long long)rows, (int)K, (int)Kp, dh.data_ptr(), !fp32_dh);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launch();
  } else if (direct && Kp != K) dh = dh.narrow(1, 0, K).contiguous();
  if (dw.defined() && Kp != K) dw = dw.narrow(1, 0, K).contiguous();
  return {dh, dw};
}

}  // namespace q38
