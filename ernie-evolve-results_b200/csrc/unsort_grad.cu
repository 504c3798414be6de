// Gradients of the weighted way back (moe_rd_unsort_tokens_backward):
//   grad_y[pos(t,k),:] = w[t,k] * grad_out[t,:],    grad_w[t,k] = <grad_out[t,:], y[pos(t,k),:]>
//
// Walked token by token, so that grad_out is read once (row by row of y it would be read K times) while the rows of y
// are gathered and the rows of grad_y scattered, each once, whole: HBM bounds it.  1 to 8 warps of a block share a
// token, by the length of its row; a lane keeps one fp32 sum per slot over its vectors, in ascending order, the lanes
// are added by a fixed tree and the warps in ascending order, so grad_w does not depend on scheduling.
// Rows of y that no pair has get a zero gradient.  Without n_rows all of grad_y is cleared first.  With it the rows from
// *n_rows on are set to zero at the end, by all blocks; among those before it a caller may have taken pairs out of
// inverse_perm, and which rows that left without one is found by blocks of their own: each reads all of inverse_perm, marks
// in shared memory which of its rows (r = its number mod their number) a pair has, and clears the others, usually none.
// That runs beside the tokens: 16 tokens x 7168 bf16, K = 8, 6.1 us with and without, 2048 x 2048 21.0 / 20.1, 8192 x 7168
// 318 / 315, 32768 x 2048 366 / 363.  It shows where rows are short and many, because such a block reads 262144 pairs in
// 20 us: 32768 x 512 106 / 95 (all rows cleared beforehand: 134), 8192 x 128 12.6 / 9.4 (12.6), 16384 x 64 23.4 / 17.1 (20).
// 32, 64 and 128 of them: 8192 x 1024 45.9, 46.5, 48.0, 32768 x 512 108, 106, 112.
#include "row_types.cuh"

namespace moe_rd {

int device_sms();

namespace {

constexpr int kGradThreads = 256;
constexpr int kGradWarps = kGradThreads / 32;
constexpr int kGradBlocksPerSm = 16;
constexpr int kMarkBlocks = 64;    // so many blocks at most look for rows without a pair, or four times as many where
constexpr int kMarkRows = 32768;   // they had more rows than this otherwise, a byte in shared memory each
constexpr int kMarkLoads = 8;
constexpr int kShortRowPairs = 65536, kShortRow = 256;  // more pairs of rows of fewer bytes: all rows are cleared beforehand

struct UnsortGradArgs {
  const uint4* grad_out;
  const uint4* y;
  const int32_t* inverse_perm;
  const float* weights;   // or null: every weight is 1
  const int32_t* n_rows;  // device value: the rows from there on are nobody's; or null: all of grad_y was cleared before
  uint4* grad_y;          // or null
  float* grad_weights;
  int64_t T, y_rows;
  int nvec, K;
  int warps_per_token;    // 1, 2, 4 or 8
  int mark_blocks;        // so many blocks, a power of two, clear the rows before *n_rows that have no pair; 0: all are cleared
};

// *n_rows, or the rows of y where that is less.
__device__ __forceinline__ int64_t used_rows(const UnsortGradArgs& a) {
  if (a.n_rows == nullptr) return a.y_rows;
  const int64_t n = __ldg(a.n_rows);
  return n < 0 ? 0 : n < a.y_rows ? n : a.y_rows;
}

__device__ __forceinline__ void clear_row(const UnsortGradArgs& a, int64_t row, int lane) {
  for (int v = lane; v < a.nvec; v += 32) __stcs(a.grad_y + (size_t)row * a.nvec + v, make_uint4(0u, 0u, 0u, 0u));
}

// What a block that looks for rows without a pair does: those of the rows r = blockIdx.x mod mark_blocks.
__device__ __forceinline__ void clear_own_rows(const UnsortGradArgs& a, unsigned char* s_has) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned block = blockIdx.x, mask = (unsigned)a.mark_blocks - 1u, log = __popc(mask);
  const unsigned used = (unsigned)used_rows(a);  // needed at the end only
  auto rows_before = [&](unsigned r) { return block < r ? (r - block + mask) >> log : 0u; };
  const unsigned rows = rows_before((unsigned)a.y_rows);  // at most kMarkRows
  for (unsigned i = tid; i < rows; i += kGradThreads) s_has[i] = 0;
  __syncthreads();
  // row block + (i << log) -> i; rows of other blocks, and what is no row, -> past the end
  auto mark = [&](int r) {
    const unsigned i = __funnelshift_r((unsigned)r - block, (unsigned)r - block, log);
    if (i < rows) s_has[i] = 1;
  };
  const unsigned P = (unsigned)(a.T * a.K);  // below 2^31
  const unsigned vectors = (reinterpret_cast<uintptr_t>(a.inverse_perm) & 15) == 0 ? P >> 2 : 0u;
  const int4* inv4 = reinterpret_cast<const int4*>(a.inverse_perm);
  for (unsigned c = tid; c < vectors; c += kMarkLoads * kGradThreads) {
    int4 r[kMarkLoads];
#pragma unroll
    for (int i = 0; i < kMarkLoads; ++i) r[i] = c + i * kGradThreads < vectors ? __ldg(inv4 + c + i * kGradThreads) : make_int4(-1, -1, -1, -1);
#pragma unroll
    for (int i = 0; i < kMarkLoads; ++i) {
      mark(r[i].x);
      mark(r[i].y);
      mark(r[i].z);
      mark(r[i].w);
    }
  }
  for (unsigned p0 = 4 * vectors + tid; p0 < P; p0 += kMarkLoads * kGradThreads) {
    int r[kMarkLoads];
#pragma unroll
    for (int i = 0; i < kMarkLoads; ++i) r[i] = p0 + i * kGradThreads < P ? __ldg(a.inverse_perm + p0 + i * kGradThreads) : -1;
#pragma unroll
    for (int i = 0; i < kMarkLoads; ++i) mark(r[i]);
  }
  __syncthreads();
  const unsigned mine = rows_before(used);
  for (unsigned i0 = 32 * warp; i0 < mine; i0 += kGradThreads) {
    const bool without = i0 + lane < mine && s_has[i0 + lane] == 0;
    for (unsigned m = __ballot_sync(kFull, without); m != 0u; m &= m - 1u)
      clear_row(a, ((int64_t)(i0 + __ffs(m) - 1) << log) + block, lane);
  }
}

// KT slots at a time; NEED_W: grad_weights is wanted (and y is read).  The compiler left alone takes 128 registers for
// KT = 8, two blocks per SM; with 80 and three blocks 32768 tokens x 2048, K = 8 take 366 us (6.2 TB/s) instead of 381, and
// with eight warps a token instead of four 385.  KT = 2 is fastest left alone (110 us against 123 for 16384 x 4096).
template <int DT, int KT, bool NEED_W>
__global__ void __launch_bounds__(kGradThreads, KT == 8 ? 3 : KT == 4 ? 4 : 0) unsort_grad_kernel(const UnsortGradArgs a) {
  constexpr int NE = RowVec<DT>::N;
  __shared__ float s_part[kGradWarps][KT];
  extern __shared__ unsigned char s_has[];
  pdl_sync();
  if (blockIdx.x < a.mark_blocks) {
    clear_own_rows(a, s_has);
    return;
  }
  const unsigned used = (unsigned)used_rows(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wpt = a.warps_per_token;
  const int sub = warp & (wpt - 1);            // this warp's share of the token
  const int tokens = kGradWarps / wpt;         // tokens of a block at a time
  // every warp of the block makes the same number of trips: the barriers below are for all of them
  const int block = blockIdx.x - a.mark_blocks, blocks = gridDim.x - a.mark_blocks;
  for (int64_t base = (int64_t)block * tokens; base < a.T; base += (int64_t)blocks * tokens) {
    const int64_t t = base + warp / wpt;
    const bool live = t < a.T;
    for (int k0 = 0; k0 < a.K; k0 += KT) {
      int pos[KT];
      float w[KT], acc[KT];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        pos[k] = live && k0 + k < a.K ? __ldg(a.inverse_perm + (size_t)t * a.K + k0 + k) : -1;
        w[k] = live && k0 + k < a.K && a.weights != nullptr ? __ldg(a.weights + (size_t)t * a.K + k0 + k) : 1.0f;
        acc[k] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < KT; ++k)
        if ((unsigned)pos[k] >= used) pos[k] = -1;
      if (live) {
        for (int v = sub * 32 + lane; v < a.nvec; v += wpt * 32) {
          const uint4 gv = __ldg(a.grad_out + (size_t)t * a.nvec + v);
          uint4 yv[KT];
          if (NEED_W) {
#pragma unroll
            for (int k = 0; k < KT; ++k)
              if (pos[k] >= 0) yv[k] = __ldcs(a.y + (size_t)pos[k] * a.nvec + v);
          }
          float g[NE];
          RowVec<DT>::unpack(gv, g);
#pragma unroll
          for (int k = 0; k < KT; ++k) {
            if (pos[k] >= 0) {
              if (NEED_W) {
                float f[NE];
                RowVec<DT>::unpack(yv[k], f);
#pragma unroll
                for (int j = 0; j < NE; ++j) acc[k] = fmaf(g[j], f[j], acc[k]);
              }
              if (a.grad_y != nullptr) {
                float o[NE];
#pragma unroll
                for (int j = 0; j < NE; ++j) o[j] = __fmul_rn(w[k], g[j]);
                __stcs(a.grad_y + (size_t)pos[k] * a.nvec + v, RowVec<DT>::pack(o));
              }
            }
          }
        }
      }
      if (NEED_W) {
#pragma unroll
        for (int k = 0; k < KT; ++k) acc[k] = warp_tree_sum(acc[k]);
        if (lane == 0) {
#pragma unroll
          for (int k = 0; k < KT; ++k) s_part[warp][k] = acc[k];
        }
        __syncthreads();
        if (live && sub == 0 && lane < KT && k0 + lane < a.K) {
          float sum = s_part[warp][lane];
          for (int i = 1; i < wpt; ++i) sum = __fadd_rn(sum, s_part[warp + i][lane]);
          a.grad_weights[(size_t)t * a.K + k0 + lane] = sum;
        }
        __syncthreads();
      }
    }
  }
  if (a.grad_y != nullptr && a.mark_blocks > 0) {
    const int64_t first = (int64_t)block * kGradWarps + warp, step = (int64_t)blocks * kGradWarps;
    const int upr = (a.nvec + 31) >> 5;
    for (int64_t u = first; u < (a.y_rows - used) * upr; u += step) {
      const int64_t r = u / upr;
      const int v = (int)(u - r * upr) * 32 + lane;
      if (v < a.nvec) __stcs(a.grad_y + (size_t)(used + r) * a.nvec + v, make_uint4(0u, 0u, 0u, 0u));
    }
  }
}

template <int DT, bool NEED_W>
cudaError_t launch_typed(const UnsortGradArgs& a, dim3 grid, cudaStream_t s) {
  const size_t smem = a.mark_blocks > 0 ? (size_t)((a.y_rows + a.mark_blocks - 1) / a.mark_blocks) : 0;
  if (a.K <= 2) return launch_pdl(unsort_grad_kernel<DT, 2, NEED_W>, grid, dim3(kGradThreads), smem, s, a);
  if (a.K <= 4) return launch_pdl(unsort_grad_kernel<DT, 4, NEED_W>, grid, dim3(kGradThreads), smem, s, a);
  return launch_pdl(unsort_grad_kernel<DT, 8, NEED_W>, grid, dim3(kGradThreads), smem, s, a);
}

template <int DT>
cudaError_t launch_dtype(const UnsortGradArgs& a, dim3 grid, cudaStream_t s) {
  return a.grad_weights != nullptr ? launch_typed<DT, true>(a, grid, s) : launch_typed<DT, false>(a, grid, s);
}

}  // namespace
}  // namespace moe_rd

using namespace moe_rd;

extern "C" int moe_rd_unsort_tokens_backward(int64_t T, int32_t H, int32_t K, int32_t dtype, const void* grad_out,
                                             const void* y, int64_t y_rows, const int32_t* inverse_perm,
                                             const float* weights, const int32_t* n_rows, void* grad_y,
                                             float* grad_weights, void* stream) {
  const int rc = check_rows(T, H, K, dtype, y_rows);
  if (rc != MOE_RD_OK) return rc;
  if (grad_y == nullptr && grad_weights == nullptr)  // of an empty batch or of no rows there is nothing to write
    return T > 0 && y_rows > 0 ? MOE_RD_E_NULL : MOE_RD_OK;
  if (T > 0 && (grad_out == nullptr || inverse_perm == nullptr ||
                (grad_weights != nullptr && y == nullptr && y_rows > 0)))
    return MOE_RD_E_NULL;
  if ((reinterpret_cast<uintptr_t>(grad_out) | reinterpret_cast<uintptr_t>(y) |
       reinterpret_cast<uintptr_t>(grad_y)) & 15)
    return MOE_RD_E_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  // rows without a pair: cleared by blocks that look for them, or all rows beforehand
  const bool clear_rows = grad_y != nullptr && y_rows > 0 && T > 0 && n_rows != nullptr && y_rows <= (int64_t)4 * kMarkBlocks * kMarkRows &&
                          (T * K <= kShortRowPairs || H * (dtype == MOE_RD_T_F32 ? 4 : 2) >= kShortRow);
  if (grad_y != nullptr && y_rows > 0 && !clear_rows)
    e = cudaMemsetAsync(grad_y, 0, (size_t)y_rows * H * (dtype == MOE_RD_T_F32 ? 4 : 2), s);
  if (e == cudaSuccess && T > 0) {
    UnsortGradArgs a = {};
    a.grad_out = static_cast<const uint4*>(grad_out);
    a.y = static_cast<const uint4*>(y);
    a.inverse_perm = inverse_perm;
    a.weights = weights;
    a.n_rows = n_rows;
    a.grad_y = y_rows > 0 ? static_cast<uint4*>(grad_y) : nullptr;
    a.grad_weights = grad_weights;
    a.T = T;
    a.y_rows = y_rows;
    a.nvec = dtype == MOE_RD_T_F32 ? H / 4 : H / 8;
    a.K = K;
    // four warps a token at most, eight where there are too few tokens to fill the SMs
    a.warps_per_token = a.nvec > 128 && T <= 4 * device_sms() ? 8 : a.nvec > 64 ? 4 : a.nvec > 32 ? 2 : 1;
    const int tokens = kGradWarps / a.warps_per_token;
    const int64_t want = (T + tokens - 1) / tokens;
    const int64_t cap = (int64_t)device_sms() * kGradBlocksPerSm;
    dim3 grid((unsigned)(want < cap ? want : cap));  // cap: more than 4 * kMarkBlocks
    if (clear_rows) {
      // one for every 32 KB of rows
      int n = 1;
      while (2 * n <= kMarkBlocks && 2 * n <= y_rows * a.nvec / 2048) n *= 2;
      while (n < 4 * kMarkBlocks && (y_rows + n - 1) / n > kMarkRows) n *= 2;
      grid.x = (unsigned)(want < cap - n ? want : cap - n) + n;  // as many blocks as without them where that is the most
      a.mark_blocks = n;
    }
    if (dtype == MOE_RD_T_BF16)
      e = launch_dtype<MOE_RD_T_BF16>(a, grid, s);
    else if (dtype == MOE_RD_T_FP16)
      e = launch_dtype<MOE_RD_T_FP16>(a, grid, s);
    else
      e = launch_dtype<MOE_RD_T_F32>(a, grid, s);
    count_launch();
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return MOE_RD_E_CUDA;
  }
  return MOE_RD_OK;
}
