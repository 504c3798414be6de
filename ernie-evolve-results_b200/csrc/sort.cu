// Tokens sorted by expert for ids that the caller has (moe_rd_sort_tokens).
//
// The place of pair (t,k) is offsets[e] + (pairs of expert e before it in flat order), a stable counting sort whose
// output is the row copy rows[place] = x[t].  It needs x once and every row once: a copy of T rows to T*K places, so
// HBM bounds a batch and launch latency bounds a few tokens.  Two forms:
//
// * batch: sort_count_kernel counts the pairs per (tile of 64 tokens, expert) and per (group of 32 tiles, expert);
//   positions_kernel and scatter_kernel of the routing pipeline (scatter.cu) derive the places from those counts and
//   copy the rows, each token row read once and stored K times.
// * few pairs and few rows (in_one_kernel): one kernel.  Every block counts ALL pairs by itself (how many of every
//   expert there are, and how many before its own tokens), ranks its own pairs and copies their rows: the counting is
//   done once per SM or more, but from L2 and by blocks that would otherwise wait, and one launch does the work of
//   three.  No workspace.
// The counts are shared-memory atomics (their order does not matter); with __match_any_sync and one atomic per distinct
// expert 16384 pairs of 256 experts took 85 us instead of 13.
// Batch: 8192 tokens x 7168 bf16, K = 8: 172 us, 6.1 TB/s, of which about 8 us are the counts and places.
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

// The one-kernel form.  Every block counts all pairs, in shared memory: blocks of 1024 threads, one per SM, do that a quarter
// as often as four of 256 (8192 tokens, K = 2, H = 512: 8.3 us against 11.3; 2048 tokens, K = 8, H = 512: 7.8 / 12.8);
// of few pairs the copy is all there is, and small blocks start sooner (16 tokens, K = 8, H = 7168: 3.0 with 256 threads,
// 3.8 with 512, 5.0 with 1024; 256 such tokens 9.2 / 7.5 / 8.6).
constexpr int kOnceWarpsPerSm = 32;
constexpr int kSmallPairs = 1024, kMiddlePairs = 4096;  // the last of 256 and of 512 threads
// Where it ends: its blocks have equal numbers of tokens, whose rows they copy, and the batch form's even spread over the
// SMs counts for more than its two launches when there is much to copy, or much to count for little (us on the device, one
// kernel / batch form; the host needs 3 / 10 to enqueue them).  H = 7168, K = 8: 512 tokens 12.7 / 22.5, 1024 (132 MB
// read and written) 25.9 / 30.2, 2048 (264 MB) 51.3 / 51.3; K = 2, H = 7168, 4096 tokens (176 MB) 34.3 / 33.1; K = 1, H =
// 4096, 16000 tokens (262 MB) 49.9 / 44.4.  Of 32768 pairs: 1000 tokens, H = 256 9.8 / 21.6, 4096 tokens, H = 512 12.9 /
// 16.2, 8192 tokens 13.5 / 13.4, 16384 tokens 17.2 / 14.7.
constexpr int64_t kOnceBytes = 144 << 20;
constexpr int kOncePairs = 16384, kOnceFewTokens = 4096, kOncePairsOfFewTokens = 32768;
constexpr int kOwnPairs = 256;  // pairs of a block's tokens

struct OnceArgs {
  const uint4* x;
  const int32_t* ids;
  uint4* rows;
  int32_t* offsets;
  int32_t* inverse_perm;
  int32_t* row_token;
  int32_t* counts;
  int64_t capacity, out_rows;
  int T, E, K, nvec;
  int tokens;  // of a block; blockIdx.x: which tokens, blockIdx.y: which part of their rows
};

// A unit of the copy: 32 * UV vectors of a row, UV loads in flight per lane.
template <int NT, int UV>
__global__ void __launch_bounds__(NT, 32 * kOnceWarpsPerSm / NT) sort_once_kernel(const OnceArgs a) {
  static_assert(kMaxE <= NT && kOwnPairs <= NT, "one expert, one pair per thread");
  constexpr int kWarps = NT / 32;
  __shared__ int s_before[kMaxE], s_after[kMaxE];  // pairs per expert before the block's own, and from them on
  __shared__ int s_off[kMaxE], s_own[kOwnPairs], s_place[kOwnPairs], s_w[kMaxE / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kMaxE) s_before[tid] = s_after[tid] = 0;
  __syncthreads();
  pdl_sync();
  const int t0 = blockIdx.x * a.tokens, ntok = min(a.tokens, a.T - t0);
  const int P = a.T * a.K, p0 = t0 * a.K, own = ntok * a.K;
  // the first unit of x is on its way while the places are worked out
  const int upr = (a.nvec + 32 * UV - 1) / (32 * UV);
  const int units = ntok * upr;
  const int first = blockIdx.y * kWarps + warp, W = gridDim.y * kWarps;
  const uint4* x = a.x + (size_t)t0 * a.nvec;
  uint4 val[UV];
  auto load = [&](int u) {
    const int t = u / upr, v = (u - t * upr) * 32 * UV + lane;
#pragma unroll
    for (int i = 0; i < UV; ++i)
      if (v + 32 * i < a.nvec) val[i] = __ldg(x + (size_t)t * a.nvec + v + 32 * i);
  };
  if (first < units) load(first);
  for (int c0 = tid; c0 < P; c0 += 8 * NT) {
    int e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c0 + i * NT < P ? __ldg(a.ids + c0 + i * NT) : -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = c0 + i * NT;
      if ((unsigned)e[i] < (unsigned)a.E) atomicAdd((p < p0 ? s_before : s_after) + e[i], 1);
      if ((unsigned)(p - p0) < (unsigned)own) s_own[p - p0] = e[i];
    }
  }
  __syncthreads();
  const int total = tid < kMaxE ? s_before[tid] + s_after[tid] : 0;
  const int kept = a.capacity > 0 && (int64_t)total > a.capacity ? (int)a.capacity : total;
  int incl = kept;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(kFull, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31 && tid < kMaxE) s_w[warp] = incl;
  __syncthreads();
  int off = incl - kept, all = 0;
#pragma unroll
  for (int w = 0; w < kMaxE / 32; ++w) {
    const int v = s_w[w];
    if (w < warp) off += v;
    all += v;
  }
  if (tid < kMaxE) s_off[tid] = off;
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    if (tid < a.E) {
      a.offsets[tid] = off;
      if (a.counts != nullptr) a.counts[tid] = total;
    }
    if (tid == 0) a.offsets[a.E] = all;
  }
  __syncthreads();
  // a pair's rank among its expert's: those before the block's own, and those before it among these
  if (tid < own) {
    const int e = s_own[tid];
    int place = -1;
    if ((unsigned)e < (unsigned)a.E) {
      int rank = s_before[e];
      for (int q = 0; q < tid; ++q) rank += s_own[q] == e;
      if (a.capacity == 0 || rank < a.capacity) place = s_off[e] + rank;
    }
    s_place[tid] = place;
    if (blockIdx.y == 0) {
      a.inverse_perm[p0 + tid] = place;
      if (place >= 0) a.row_token[place] = t0 + tid / a.K;
    }
  }
  __syncthreads();
  for (int u = first; u < units; u += W) {
    const int t = u / upr, v = (u - t * upr) * 32 * UV + lane;
    if (u != first) load(u);
    for (int k = 0; k < a.K; ++k) {
      const int place = s_place[t * a.K + k];
      if (place < 0) continue;
      uint4* to = a.rows + (size_t)place * a.nvec + v;
#pragma unroll
      for (int i = 0; i < UV; ++i)
        if (v + 32 * i < a.nvec) __stcs(to + 32 * i, val[i]);
    }
  }
  // rows of nobody
  const int64_t block = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, blocks = (int64_t)gridDim.x * gridDim.y;
  for (int64_t r = (int64_t)all + block * NT + tid; r < a.out_rows; r += blocks * NT) a.row_token[r] = -1;
  for (int64_t k = ((int64_t)all * a.nvec) + block * NT + tid; k < a.out_rows * a.nvec; k += blocks * NT)
    __stcs(a.rows + k, make_uint4(0u, 0u, 0u, 0u));
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

template <int NT>
cudaError_t launch_once(OnceArgs& a, cudaStream_t s) {
  constexpr int kWarps = NT / 32;
  // as many blocks as are resident at once, each with the same number of tokens (at most kOwnPairs pairs); few tokens
  // share their rows' columns out among blocks
  const int most = device_sms() * (kOnceWarpsPerSm / kWarps);
  a.tokens = (a.T + most - 1) / most;
  while (a.tokens > 1 && a.tokens * a.K > kOwnPairs) --a.tokens;
  const int bx = (a.T + a.tokens - 1) / a.tokens;
  const int units = (a.nvec + 31) / 32;
  int by = (a.tokens * units + kWarps - 1) / kWarps;
  if (by > most / bx) by = most / bx > 1 ? most / bx : 1;
  // more units than resident warps: fewer and larger ones
  const dim3 grid((unsigned)bx, (unsigned)by);
  return (int64_t)a.T * units > (int64_t)most * kWarps * 2 ? launch_pdl(sort_once_kernel<NT, 4>, grid, dim3(NT), 0, s, a)
                                                           : launch_pdl(sort_once_kernel<NT, 1>, grid, dim3(NT), 0, s, a);
}

bool in_one_kernel(int64_t T, int32_t H16, int32_t K) {
  return T * K <= (T <= kOnceFewTokens ? kOncePairsOfFewTokens : kOncePairs) && T * (K + 1) * H16 * 2 <= kOnceBytes;
}

int check_experts(int64_t T, int32_t E) {
  if (E < 1 || E > kMaxE) return MOE_RD_E_SHAPE;
  if ((T + kTile - 1) / kTile * E > 0x7fffffff) return MOE_RD_E_TOO_LARGE;
  return MOE_RD_OK;
}

}  // namespace
}  // namespace moe_rd

using namespace moe_rd;

extern "C" int moe_rd_sort_workspace_bytes(int64_t T, int32_t H, int32_t E, int32_t K, int32_t dtype, size_t* bytes) {
  if (bytes == nullptr) return MOE_RD_E_NULL;
  int rc = check_rows(T, H, K, dtype, 0);
  if (rc == MOE_RD_OK) rc = check_experts(T, E);
  if (rc != MOE_RD_OK) return rc;
  *bytes = T == 0 || in_one_kernel(T, dtype == MOE_RD_T_F32 ? 2 * H : H, K) ? 0 : carve_sort(T, E).total;
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
  } else if (in_one_kernel(T, H16, K)) {
    OnceArgs a = {};
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
    e = T * K > kMiddlePairs ? launch_once<1024>(a, s) : T * K > kSmallPairs ? launch_once<512>(a, s) : launch_once<256>(a, s);
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
