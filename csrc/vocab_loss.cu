// Softmax cross entropy over a large vocabulary in pieces of the vocabulary, without keeping the logits.
//
//   z = h W^T,  lse_t = ln sum_v e^z_tv,  loss_t = lse_t - z_t,target;   dz = s_t (e^(z - lse) - onehot),  dh = dz W,  dW = dz^T h
//
// Forward: the product's tiles are reduced where they arise.  Each 128 x bn accumulator is read from tensor memory once, and leaves per row and half tile the
// pair (k, s) with sum = s 2^k and the target's logit; a small kernel joins the pairs.  Nothing of size rows x vocabulary is written.
// Backward: for one piece of the vocabulary after the other the same tiles are formed again, turned into dz (bf16, a workspace of one piece) and
// multiplied by W and h on the framework's GEMM.  The logits stay fp32 in tensor memory: storing them in bf16 (half a step of 2^-9 of a logit of ten) would put an
// error of 2 % into a probability.  dz is rounded to bf16 because the tensor cores take it so; its target entry is -1 + p, whose rounding is small, and a factor that all
// rows share is applied to the products in fp32.
//
// The kernel follows csrc/gemm_persistent.cu: one CTA per SM, warp 0 loads by TMA, one lane of warp 1 issues the MMAs into one of two accumulators, and eight
// warps (two warpgroups on alternate 32-column chunks) read the other.  Tiles are walked with the rows fastest, in groups of rows whose hidden states
// stay in L2: all SMs work on the same few columns of W, which so comes from memory once per group.
// On a B200, each kernel alone: 8192 x 50048 x 1024 forward 513 us (1.64 PFLOP/s, level with cuBLAS), dz 629 us (1.33), dh and dW 608 and 582 us; 4096 x 10112 x 576
// 38, 44, 43 and 48 us.  Bound by the tensor cores in the forward, by operand traffic (96 bytes per clock and SM, and the stores of dz) in the others.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "f32x2.cuh"
#include "ptx.cuh"
#include "host.h"
#include "launch.cuh"
#include "training.h"

namespace q38 {

void gemm_bf16_scaled(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c, bool a_mn_major, bool b_mn_major, const float* num, const float* den, bool accumulate,
                      int64_t slabs, const at::Tensor& err);     // gemm_persistent.cu
int64_t gemm_tiles(int64_t M, int64_t N);                        // gemm_persistent.cu

constexpr int V_BM = 128, V_BK = 64, V_MAX_STAGES = 8, V_THREADS = 320, V_ACC_COLS = 256;
constexpr float V_LOG2E = 1.44269504088896340736f;
constexpr long long V_IGNORE = -100;

struct VocabArgs {
  int rows, cols, K, bn;                       // cols: of this piece
  int tiles_m, tiles_n, group_m, total_kb, items, stages, first_col, vocab;
  const long long* target;
  float2* partial;                             // [2 tiles_n][rows]: (k, s) of a half tile
  float* target_logit;                         // [rows]
  const float *lse2, *upstream;                // backward: log2 of the row's sum; gradient of each row (null: one factor for all, which the products' epilogues apply)
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
        scale = p.upstream == nullptr ? 1.f : p.upstream[row];
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
      ptx::tmem_ld_32x32b_x32(t_addr + c0, ra);                    // bn is 64 at least: every warp has a chunk
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

// lse2[row] = log2 of the row's sum and loss[row], from the tiles' pairs: 32 rows per CTA, 32 threads per row in strides of 32 pairs, joined in order.
// A target outside the vocabulary that is not the ignored one is an error: it is reported, and the row counts as ignored.
__global__ void __launch_bounds__(1024) vocab_join_kernel(const float2* __restrict__ partial, int parts, int rows, int vocab, const long long* __restrict__ target,
                                                          const float* __restrict__ target_logit, float* __restrict__ lse2, float* __restrict__ loss, int* err) {
  grid_wait();
  __shared__ float2 part[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, row = blockIdx.x * 32 + x;
  auto join = [](float2 a, float2 b) {
    const float k = fmaxf(a.x, b.x), ref = k == -INFINITY ? 0.f : k;
    return make_float2(k, a.y * exp2_approx(a.x - ref) + b.y * exp2_approx(b.x - ref));
  };
  const float2 none = make_float2(-INFINITY, 0.f);
  float2 v = none;
  if (row < rows) {
    for (int i = y; i < parts; i += 128) {                       // four reads in flight
      float2 r[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) r[q] = i + 32 * q < parts ? partial[(long long)(i + 32 * q) * rows + row] : none;
      v = join(v, join(join(r[0], r[1]), join(r[2], r[3])));
    }
  }
  part[y][x] = v;
  __syncthreads();
  // a warp per row from here: lane q has the row's part q
  v = part[x][y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join(v, make_float2(__shfl_down_sync(0xffffffffu, v.x, o), __shfl_down_sync(0xffffffffu, v.y, o)));
  const int mine = blockIdx.x * 32 + y;
  if (x != 0 || mine >= rows) return;
  const double l2 = (double)v.x + log2((double)v.y);
  const long long tgt = target[mine];
  const bool inside = tgt >= 0 && tgt < vocab;
  if (!inside && tgt != V_IGNORE) report_error(err, ERR_BOUNDS);
  lse2[mine] = (float)l2;
  loss[mine] = inside ? (float)(l2 * 0.69314718055994530942 - (double)target_logit[mine]) : 0.f;
}

// Sum of all losses and number of rows that count, by one CTA in a fixed order: `total` the sum or the mean over those rows, `number` how many they are (at least 1).
__global__ void __launch_bounds__(1024) vocab_sum_kernel(const float* __restrict__ loss, const long long* __restrict__ target, int rows, int vocab, bool mean, float* total, float* number) {
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
  *total = (float)(mean ? s / n : s);
  *number = (float)n;
}

// out [rows, cols] = sum of `slabs` fp32 matrices (rows of ldp elements, a multiple of 4), in order, as bf16 or fp32: a warp per row, four columns per lane
template <bool BF16>
__global__ void __launch_bounds__(256) vocab_slabs_kernel(const float* __restrict__ part, int slabs, long long slab, int rows, int cols, int ldp, void* out) {
  grid_wait();
  const int lane = threadIdx.x & 31;
  const bool packs = cols % 4 == 0;
  for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.x * 8) {
    const float* in = part + r * ldp;
#pragma unroll 2
    for (int c = lane * 4; c < cols; c += 128) {                 // the last pack may end in a row's padding, which is read and not used
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k0 = 0; k0 < slabs; k0 += 4) {                     // four reads in flight
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = k0 + k < slabs ? *reinterpret_cast<const float4*>(in + (k0 + k) * slab + c) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) { s.x += v[k].x; s.y += v[k].y; s.z += v[k].z; s.w += v[k].w; }
      }
      const long long at = r * cols + c;
      if (packs) {
        if (BF16) *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(out) + at) = make_uint2(bf16_pair(make_float2(s.x, s.y)), bf16_pair(make_float2(s.z, s.w)));
        else *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = s;
      } else {
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < cols) {
            if (BF16) reinterpret_cast<__nv_bfloat16*>(out)[at + e] = __float2bfloat16_rn(v[e]);
            else reinterpret_cast<float*>(out)[at + e] = v[e];
          }
      }
    }
  }
}

// Rows of bf16 or fp32 into rows of another distance, a warp per row (hidden sizes that TMA does not take, into padded rows and back).
// 30011 x 711 to padded rows: torch's copy 46 us, this 18.
template <typename T>
__global__ void __launch_bounds__(256) vocab_rows_kernel(const T* __restrict__ in, long long ldi, long long step, T* __restrict__ out, long long ldo, int rows, int cols) {
  grid_wait();
  const int lane = threadIdx.x & 31;
  for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.x * 8) {
    const T* src = in + r * ldi;
    T* dst = out + r * ldo;
    for (int base = lane; base < cols; base += 256) {
      T v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) if (base + 32 * e < cols) v[e] = src[(base + 32 * e) * step];
#pragma unroll
      for (int e = 0; e < 8; ++e) if (base + 32 * e < cols) dst[base + 32 * e] = v[e];
    }
  }
}

namespace {

using at::Tensor;

void copy_rows(const Tensor& in, const Tensor& out, cudaStream_t stream) {
  const unsigned grid = (unsigned)std::min<int64_t>((in.size(0) + 7) / 8, kNumSMs * 16);
  if (in.element_size() == 2)
    launch(vocab_rows_kernel<uint16_t>, grid, 256, 0, stream, (const uint16_t*)in.data_ptr(), in.stride(0), in.stride(1), (uint16_t*)out.data_ptr(), out.stride(0), (int)in.size(0), (int)in.size(1));
  else
    launch(vocab_rows_kernel<uint32_t>, grid, 256, 0, stream, (const uint32_t*)in.data_ptr(), in.stride(0), in.stride(1), (uint32_t*)out.data_ptr(), out.stride(0), (int)in.size(0), (int)in.size(1));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
}

// The first n columns (views cost the host as much as launches: none where all are meant)
Tensor columns(const Tensor& t, int64_t n) { return t.size(-1) == n ? t : t.narrow(-1, 0, n); }

int64_t padded(int64_t n) { return (n + 63) / 64 * 64; }

// Parts of the reduction of dh = dz W side by side: rounds of tiles times K blocks (0.35 us each, six more for a tile's start), plus the sums' way through memory
int64_t pick_slabs(int64_t rows, int64_t K, int64_t cols) {
  const int64_t tiles = gemm_tiles(rows, K), blocks = (cols + 63) / 64;
  int64_t best = 1;
  double least = 1e30;
  for (int64_t s = 1; s <= std::max<int64_t>(8, kNumSMs / tiles) && blocks / s >= 4; ++s) {
    const int64_t per = (blocks + s - 1) / s;
    const double cost = double((tiles * s + kNumSMs - 1) / kNumSMs) * (per + 6) * 0.35e-6 + (s > 1 ? double(s) : 0.0) * rows * K * 8 / 6.5e12;
    if (cost < least * 0.98) { best = (blocks + per - 1) / per; least = cost; }
  }
  return best;
}

// Columns per tile: the fewest rounds of tiles times their width, where a tile's start is worth 32 columns
int tile_width(int64_t rows, int64_t cols) {
  int best = 256;
  int64_t least = INT64_MAX;
  for (int bn = 256; bn >= 64; bn -= 32) {
    const int64_t items = (rows + V_BM - 1) / V_BM * ((cols + bn - 1) / bn), cost = (items + kNumSMs - 1) / kNumSMs * (bn + 32);
    if (cost < least) { best = bn; least = cost; }
  }
  return best;
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
  allow_shared_memory((const void*)kernel, 227 * 1024);
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
  for (const Tensor* t : {&h, &w})
    TORCH_CHECK((t->stride(1) == 1 || t->size(1) == 1) && t->stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(t->data_ptr()) & 15) == 0, "vocab_loss: rows that TMA takes required");
  // tiles are counted and columns addressed in 32 bits
  TORCH_CHECK(h.size(0) < (1ll << 24) && w.size(0) < (1ll << 24) && h.size(1) < (1ll << 24) && ((h.size(0) + 127) / 128) * ((w.size(0) + 63) / 64) < (1ll << 30), "vocab_loss: too many rows or columns");
}

}  // namespace

// Copies go into rows of whole 128-byte lines: rows 16 bytes off a line cost two lines per box (2049 x 30011 x 711, the forward's tiles 109 -> 73 us).
Tensor vocab_rows(const Tensor& t) {
  const int64_t n = t.size(1);
  if ((t.stride(1) == 1 || n == 1) && t.stride(0) >= n && t.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return t;
  const c10::cuda::CUDAGuard guard(t.device());
  auto view = new_tensor({t.size(0), padded(n)}, t.scalar_type(), t.device()).narrow(1, 0, n);
  if (t.numel()) copy_rows(t, view, at::cuda::getCurrentCUDAStream());
  return view;
}

std::array<Tensor, 3> vocab_loss_fwd(const Tensor& hidden, const Tensor& weight, const Tensor& target, at::IntArrayRef shape, int64_t reduction, const Tensor& err) {
  check(hidden, weight, target);
  const auto device = hidden.device();
  const c10::cuda::CUDAGuard guard(device);
  const int64_t rows = hidden.size(0), vocab = weight.size(0);
  auto loss = new_tensor(reduction ? at::IntArrayRef(&rows, 1) : shape, at::kFloat, device), lse2 = new_tensor({rows}, at::kFloat, device);
  auto stream = at::cuda::getCurrentCUDAStream();
  if (rows) {
    // 65536 rows at a time bound the pairs' workspace: 16 bytes per row and tile of bn columns, so a sixteenth of a byte per score in wide tiles, a quarter in the narrowest
    for (int64_t at = 0; at < rows; at += 65536) {
      const int64_t n = std::min<int64_t>(65536, rows - at);
      const Tensor h = n == rows ? hidden : hidden.narrow(0, at, n);
      VocabArgs p{};
      const int bn = tile_width(n, vocab);
      auto partial = new_tensor({2 * ((vocab + bn - 1) / bn), n, 2}, at::kFloat, device), logit = new_tensor({n}, at::kFloat, device);
      p.target = reinterpret_cast<const long long*>(target.data_ptr<int64_t>()) + at;
      p.partial = reinterpret_cast<float2*>(partial.data_ptr<float>());
      p.target_logit = logit.data_ptr<float>();
      p.err = err.data_ptr<int>();
      launch_tiles<false>(h, weight, 0, vocab, p, nullptr, stream);
      launch(vocab_join_kernel, (unsigned)((n + 31) / 32), 1024, 0, stream, (const float2*)p.partial, 2 * p.tiles_n, (int)n, (int)vocab, p.target, (const float*)p.target_logit,
             lse2.data_ptr<float>() + at, loss.data_ptr<float>() + at, p.err);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      count_launch();
    }
  }
  if (reduction == 0) return {loss, lse2, Tensor()};
  auto total = new_tensor({}, at::kFloat, device), count = new_tensor({}, at::kFloat, device);
  launch(vocab_sum_kernel, 1, 1024, 0, stream, (const float*)loss.data_ptr<float>(), reinterpret_cast<const long long*>(target.data_ptr<int64_t>()), (int)rows, (int)vocab, reduction == 2,
         total.data_ptr<float>(), count.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launch();
  return {total, lse2, count};
}

std::pair<Tensor, Tensor> vocab_loss_bwd(const Tensor& g, const Tensor& h, const Tensor& w, const Tensor& target, const Tensor& lse2, const Tensor& count, int64_t reduction,
                                         bool want_dh, bool fp32_dh, bool want_dw, bool fp32_dw, const Tensor& grad, int64_t workspace, const Tensor& err) {
  check(h, w, target);
  TORCH_CHECK(g.device() == h.device() && g.scalar_type() == at::kFloat && g.is_contiguous() && g.numel() == (reduction ? 1 : h.size(0)) && lse2.numel() == h.size(0),
              "vocab_loss_bwd: bad gradient");
  const c10::cuda::CUDAGuard guard(h.device());
  const int64_t rows = h.size(0), K = h.size(1), vocab = w.size(0), Kp = K % 8 ? padded(K) : K;
  const auto device = h.device();
  const auto dh_type = fp32_dh ? at::kFloat : at::kBFloat16, dw_type = fp32_dw ? at::kFloat : at::kBFloat16;
  auto stream = at::cuda::getCurrentCUDAStream();
  Tensor dh, dw;
  if (rows == 0) {
    if (want_dh) dh = new_tensor({0, K}, dh_type, device);
    if (want_dw && !grad.defined()) dw = new_tensor({vocab, K}, dw_type, device).zero_();
    return {dh, dw};
  }
  // Pieces: as few as the workspace allows, of equal width (whole tiles); 256 columns at least, which is more than 256 MB beyond 524288 rows
  const int64_t widest = std::max<int64_t>(256, workspace / (2 * rows) / 256 * 256), pieces = (vocab + widest - 1) / widest;
  const int64_t width = std::min((vocab + 7) / 8 * 8, ((vocab + pieces - 1) / pieces + 255) / 256 * 256);
  auto dz_all = new_tensor({rows, width}, at::kBFloat16, device);
  // dh: where its tiles leave SMs without work, parts of the reduction side by side, added in order at the end
  const int64_t slabs = pick_slabs(rows, K, std::min(width, vocab));
  const bool direct = want_dh && slabs == 1 && pieces == 1;
  Tensor part;
  if (want_dh && !direct) part = new_tensor({slabs, rows, Kp}, at::kFloat, device);
  if (direct) dh = new_tensor({rows, Kp}, dh_type, device);
  if (want_dw && !grad.defined()) dw = new_tensor({vocab, Kp}, dw_type, device);
  VocabArgs p{};
  p.target = reinterpret_cast<const long long*>(target.data_ptr<int64_t>());
  p.lse2 = lse2.data_ptr<float>();
  p.upstream = reduction ? nullptr : g.data_ptr<float>();
  p.err = err.data_ptr<int>();
  // One factor for all rows stays out of dz: its rounding to bf16 would be the same for every row and not average out (8192 rows, 1/8028: 3.5e-3 instead of 1.8e-3 off)
  const float* num = reduction ? g.data_ptr<float>() : nullptr;
  const float* den = reduction == 2 ? count.data_ptr<float>() : nullptr;
  for (int64_t at = 0; at < vocab; at += width) {
    const int64_t cols = std::min(width, vocab - at);
    const bool first = at == 0;
    const CUtensorMap tc = make_tmap_box(dz_all.data_ptr(), 2, cols, rows, 1, width, 0, 32, 64);
    launch_tiles<true>(h, w, at, cols, p, &tc, stream);
    const Tensor dz = columns(dz_all, cols), wp = cols == vocab ? w : w.narrow(0, at, cols);
    if (direct) gemm_bf16_scaled(dz, wp, columns(dh, K), false, true, num, den, false, 0, err);
    else if (want_dh) gemm_bf16_scaled(dz, wp, columns(part, K), false, true, num, den, !first, slabs, err);
    if (want_dw) {
      if (grad.defined()) gemm_bf16_scaled(dz, h, cols == vocab ? grad : grad.narrow(0, at, cols), true, true, num, den, true, 0, err);
      else gemm_bf16_scaled(dz, h, columns(cols == vocab ? dw : dw.narrow(0, at, cols), K), true, true, num, den, false, 0, err);
    }
  }
  if (want_dh && !direct) {
    dh = new_tensor({rows, K}, dh_type, device);
    auto kernel = fp32_dh ? vocab_slabs_kernel<false> : vocab_slabs_kernel<true>;
    launch(kernel, (unsigned)std::min<int64_t>((rows + 7) / 8, kNumSMs * 8), 256, 0, stream, (const float*)part.data_ptr<float>(), (int)slabs, (long long)(rows * Kp), (int)rows, (int)K, (int)Kp,
           dh.data_ptr());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launch();
  } else if (direct && Kp != K) {
    const Tensor wide = dh.narrow(1, 0, K);
    dh = new_tensor({rows, K}, dh_type, device);
    copy_rows(wide, dh, stream);
  }
  if (dw.defined() && Kp != K) {
    const Tensor wide = dw.narrow(1, 0, K);
    dw = new_tensor({vocab, K}, dw_type, device);
    copy_rows(wide, dw, stream);
  }
  return {dh, dw};
}

}  // namespace q38
