// Tokens sorted by expert for ids that the caller has (moe_rd_sort_tokens).
//
// The place of pair (t,k) is offsets[e] + (pairs of expert e before it in flat order), a stable counting sort whose
// output is the row copy rows[place] = x[t].  It needs x once and every row once: a copy of T rows to T*K places, so
// HBM bounds a batch and launch latency bounds a few tokens.  Two forms:
//
// * batch: sort_count_kernel counts the pairs per (tile of 64 tokens, expert) and per (group of 32 tiles, expert);
//   positions_kernel and scatter_kernel of the routing pipeline (scatter.cu) derive the places from those counts and
//   copy the rows, each token row read once and stored K times.
// * few pairs: one kernel.  Every block works out the places of ALL pairs from the ids in shared memory (the same
//   stable count) and copies its share of the rows, so a decode step pays one launch and needs no workspace.
#include "row_types.cuh"

namespace moe_rd {

int device_sms();
cudaError_t launch_sort_scatter(int64_t T, int H16, int E, int K, int64_t capacity, int64_t out_rows, const void* x,
                                const int32_t* ids, const int32_t* tile_counts, const int32_t* group_counts,
                                void* rows, int32_t* offsets, int32_t* inverse_perm, int32_t* row_token,
                                int32_t* counts, cudaStream_t s);

namespace {

constexpr int kCountThreads = 32 * kTileGroup;  // a warp per tile of the block's group

// Block g counts group g: one warp per tile, into its own shared row of E counters; the group's counts are the column
// sums.  Plain stores only, so nothing has to be cleared beforehand.
__global__ void __launch_bounds__(kCountThreads)
sort_count_kernel(const int32_t* __restrict__ ids, int64_t T, int E, int K, int ntiles, int32_t* __restrict__ tile_counts,
                  int32_t* __restrict__ group_counts) {
  extern __shared__ int s_cnt[];  // [kTileGroup][E]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kTileGroup * E; i += kCountThreads) s_cnt[i] = 0;
  __syncthreads();
  pdl_sync();
  const int tile = blockIdx.x * kTileGroup + warp;
  if (tile < ntiles) {
    int* mine = s_cnt + warp * E;
    const int64_t t0 = (int64_t)tile * kTile;
    const int P = (int)min((int64_t)kTile, T - t0) * K;
    const int32_t* src = ids + (size_t)t0 * K;
    for (int b = 0; b < P; b += 256) {
      int e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = b + 32 * i + lane < P ? __ldg(src + b + 32 * i + lane) : -1;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((unsigned)e[i] < (unsigned)E) atomicAdd(mine + e[i], 1);
    }
    __syncwarp();
    for (int e = lane; e < E; e += 32) tile_counts[(size_t)tile * E + e] = mine[e];
  }
  __syncthreads();
  for (int e = tid; e < E; e += kCountThreads) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kTileGroup; ++w) sum += s_cnt[w * E + e];
    group_counts[(size_t)blockIdx.x * E + e] = sum;
  }
}

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewPairs = 1024;
constexpr int kFewChunks = kFewPairs / 32 / kFewWarps;  // chunks of 32 pairs per warp
static_assert(kMaxE <= kFewThreads, "one expert per thread");

struct FewArgs {
  const uint4* x;
  const int32_t* ids;
  uint4* rows;
  int32_t* offsets;
  int32_t* inverse_perm;
  int32_t* row_token;
  int32_t* counts;
  int64_t capacity, out_rows;
  int T, E, K, nvec;
};

__global__ void __launch_bounds__(kFewThreads) sort_few_kernel(const FewArgs a) {
  extern __shared__ __align__(16) uint16_t s_cc[];  // [chunks][E] pairs per chunk and expert, then the pairs before it
  __shared__ int s_off[kMaxE], s_place[kFewPairs], s_w[kFewWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int P = a.T * a.K;
  const int nch = (P + 31) >> 5;
  for (int i = tid; i < (nch * a.E + 1) >> 1; i += kFewThreads) reinterpret_cast<uint32_t*>(s_cc)[i] = 0u;
  __syncthreads();
  pdl_sync();
  // the first unit of x is on its way while the places are worked out
  const int upr = (a.nvec + 31) >> 5;  // a unit: 32 vectors of a row
  const int units = a.T * upr;
  const int first = blockIdx.x * kFewWarps + warp;
  const int W = gridDim.x * kFewWarps;
  uint4 val = make_uint4(0u, 0u, 0u, 0u);
  if (first < units) {
    const int t = first / upr, v = (first - t * upr) * 32 + lane;
    if (v < a.nvec) val = __ldg(a.x + (size_t)t * a.nvec + v);
  }
  int e_reg[kFewChunks];
  unsigned before[kFewChunks];
#pragma unroll
  for (int i = 0; i < kFewChunks; ++i) {
    const int p = (i * kFewWarps + warp) * 32 + lane;
    const int e = p < P ? __ldg(a.ids + p) : -1;
    e_reg[i] = (unsigned)e < (unsigned)a.E ? e : -1;
  }
#pragma unroll
  for (int i = 0; i < kFewChunks; ++i) {
    const int c = i * kFewWarps + warp;
    if (c < nch) {
      const unsigned m = __match_any_sync(kFull, e_reg[i]);
      before[i] = __popc(m & ((1u << lane) - 1u));
      if (e_reg[i] >= 0 && before[i] == 0) s_cc[c * a.E + e_reg[i]] = (uint16_t)__popc(m);
    }
  }
  __syncthreads();
  int total = 0;
  if (tid < a.E) {
    for (int c = 0; c < nch; ++c) {
      const int v = s_cc[c * a.E + tid];
      s_cc[c * a.E + tid] = (uint16_t)total;
      total += v;
    }
  }
  const int kept = a.capacity > 0 && (int64_t)total > a.capacity ? (int)a.capacity : total;
  int incl = kept;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(kFull, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) s_w[warp] = incl;
  __syncthreads();
  int off = incl - kept, all = 0;
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    const int v = s_w[w];
    if (w < warp) off += v;
    all += v;
  }
  if (tid < a.E) s_off[tid] = off;
  if (blockIdx.x == 0) {
    if (tid < a.E) {
      a.offsets[tid] = off;
      if (a.counts != nullptr) a.counts[tid] = total;
    }
    if (tid == 0) a.offsets[a.E] = all;
    for (int64_t r = (int64_t)all + tid; r < a.out_rows; r += kFewThreads) a.row_token[r] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kFewChunks; ++i) {
    const int c = i * kFewWarps + warp, p = c * 32 + lane;
    if (p < P) {
      int place = -1;
      if (e_reg[i] >= 0) {
        const int rank = s_cc[c * a.E + e_reg[i]] + before[i];
        if (a.capacity == 0 || rank < a.capacity) place = s_off[e_reg[i]] + rank;
      }
      s_place[p] = place;
      if (blockIdx.x == 0) {
        a.inverse_perm[p] = place;
        if (place >= 0) a.row_token[place] = p / a.K;
      }
    }
  }
  __syncthreads();
  for (int u = first; u < units; u += W) {
    const int t = u / upr, v = (u - t * upr) * 32 + lane;
    if (v < a.nvec) {
      if (u != first) val = __ldg(a.x + (size_t)t * a.nvec + v);
      for (int k = 0; k < a.K; ++k) {
        const int place = s_place[t * a.K + k];
        if (place >= 0) __stcs(a.rows + (size_t)place * a.nvec + v, val);
      }
    }
  }
  const int64_t tail = (a.out_rows - all) * upr;
  for (int64_t u = first; u < tail; u += W) {
    const int64_t r = u / upr;
    const int v = (int)(u - r * upr) * 32 + lane;
    if (v < a.nvec) __stcs(a.rows + (size_t)(all + r) * a.nvec + v, make_uint4(0u, 0u, 0u, 0u));
  }
}

struct SortWorkspace {
  size_t tile_counts, group_counts, total;
};

SortWorkspace carve_sort(int64_t T, int32_t E) {
  const size_t ntiles = (size_t)((T + kTile - 1) / kTile), ngroups = (ntiles + kTileGroup - 1) / kTileGroup;
  SortWorkspace w;
  w.tile_counts = 0;
  w.group_counts = (ntiles * E * 4 + 255) & ~(size_t)255;
  w.total = w.group_counts + ((ngroups * E * 4 + 255) & ~(size_t)255);
  return w;
}

int check_experts(int64_t T, int32_t E) {
  if (E < 1 || E > kMaxE) return MOE_RD_E_SHAPE;
  if ((T + kTile - 1) / kTile * E > 0x7fffffff) return MOE_RD_E_TOO_LARGE;
  return MOE_RD_OK;
}

}  // namespace
}  // namespace moe_rd

using namespace moe_rd;

extern "C" int moe_rd_sort_workspace_bytes(int64_t T, int32_t E, int32_t K, size_t* bytes) {
  if (bytes == nullptr) return MOE_RD_E_NULL;
  int rc = check_rows(T, 8, K, MOE_RD_T_BF16, 0);
  if (rc == MOE_RD_OK) rc = check_experts(T, E);
  if (rc != MOE_RD_OK) return rc;
  *bytes = T * K <= kFewPairs ? 0 : carve_sort(T, E).total;
  return MOE_RD_OK;
}

extern "C" int moe_rd_sort_tokens(int64_t T, int32_t H, int32_t E, int32_t K, int32_t dtype, int64_t capacity,
                                  int64_t out_rows, const void* x, const int32_t* expert_ids, void* rows,
                                  int32_t* offsets, int32_t* inverse_perm, int32_t* row_token, int32_t* counts,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_rows(T, H, K, dtype, out_rows);
  if (rc == MOE_RD_OK) rc = check_experts(T, E);
  if (rc != MOE_RD_OK) return rc;
  if (capacity < 0 || (out_rows < T * K && (capacity == 0 || out_rows / E < capacity))) return MOE_RD_E_SHAPE;
  if (offsets == nullptr || (out_rows > 0 && (rows == nullptr || row_token == nullptr)) ||
      (T > 0 && (x == nullptr || expert_ids == nullptr || inverse_perm == nullptr)))
    return MOE_RD_E_NULL;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows)) & 15) return MOE_RD_E_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int H16 = dtype == MOE_RD_T_F32 ? 2 * H : H;
  cudaError_t e = cudaSuccess;
  if (T == 0) {
    e = cudaMemsetAsync(offsets, 0, (size_t)(E + 1) * 4, s);
    if (e == cudaSuccess && counts != nullptr) e = cudaMemsetAsync(counts, 0, (size_t)E * 4, s);
    if (e == cudaSuccess && out_rows > 0) e = cudaMemsetAsync(row_token, 0xff, (size_t)out_rows * 4, s);
    if (e == cudaSuccess && out_rows > 0) e = cudaMemsetAsync(rows, 0, (size_t)out_rows * H16 * 2, s);
  } else if (T * K <= kFewPairs) {
    FewArgs a = {};
    a.x = static_cast<const uint4*>(x);
    a.ids = expert_ids;
    a.rows = static_cast<uint4*>(rows);
    a.offsets = offsets;
    a.inverse_perm = inverse_perm;
    a.row_token = row_token;
    a.counts = counts;
    a.capacity = capacity;
    a.out_rows = out_rows;
    a.T = (int)T;
    a.E = E;
    a.K = K;
    a.nvec = H16 / 8;
    const int64_t want = (T * ((a.nvec + 31) / 32) + kFewWarps - 1) / kFewWarps;
    const int64_t cap = (int64_t)device_sms() * 2;
    const size_t smem = (size_t)((T * K + 31) / 32) * E * 2 + 16;
    e = launch_pdl(sort_few_kernel, dim3((unsigned)(want < cap ? want : cap)), dim3(kFewThreads), smem, s, a);
    count_launch();
  } else {
    const SortWorkspace w = carve_sort(T, E);
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255) || workspace_bytes < w.total)
      return MOE_RD_E_WORKSPACE;
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    int32_t* tile_counts = reinterpret_cast<int32_t*>(ws + w.tile_counts);
    int32_t* group_counts = reinterpret_cast<int32_t*>(ws + w.group_counts);
    const int ntiles = (int)((T + kTile - 1) / kTile);
    e = launch_pdl(sort_count_kernel, dim3((unsigned)((ntiles + kTileGroup - 1) / kTileGroup)), dim3(kCountThreads),
                   (size_t)kTileGroup * E * 4, s, expert_ids, T, (int)E, (int)K, ntiles, tile_counts, group_counts);
    count_launch();
    if (e == cudaSuccess)
      e = launch_sort_scatter(T, H16, E, K, capacity, out_rows, x, expert_ids, tile_counts, group_counts, rows,
                              offsets, inverse_perm, row_token, counts, s);
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return MOE_RD_E_CUDA;
  }
  return MOE_RD_OK;
}
