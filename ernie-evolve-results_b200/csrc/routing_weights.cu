// The combine weights of chosen experts from the router's logits, and their gradient.
//
// With z the (biased) logits of a token, s = softmax(z) or sigmoid(z), u_k = s[id_k] (+ bias), S = sum_k u_k and
// c = routed_scale:  w_k = c u_k / max(S, m)  (renorm) or  c u_k.  For g_k = dL/dw_k:
//   h_k = c (g_k - [S >= m] sum_j g_j u_j / S) / max(S, m)   (renorm) or  c g_k       (dL/du_k)
//   softmax:  dL/dz_e = s_e (H_e - D),  H_e = sum_{k: id_k = e} h_k,  D = sum_e s_e H_e
//   sigmoid:  dL/dz_e = s_e (1 - s_e) H_e
// A router that is sure of itself has one u_k / S (one s_e) next to 1, where those differences cancel.  They are
// computed without it, from differences of the g and h themselves:
//   g_k - sum_j g_j u_j / S = sum_j (u_j / S) (g_k - g_j)                        (the u_j / S add up to 1)
//   H_e - D = sum_{chosen f} s_f (H_e - H_f) + H_e * (sum of s over the experts that were not chosen)
// Where u = s, renormalised and S >= m, D is zero identically (w does not change when every logit moves by the same
// amount) and is left out.  1 - s of the sigmoid is exp(-z) s, not a subtraction.
//
// One warp per token.  The softmax needs every logit of the token, the sigmoid only those of the chosen experts; the
// gradient row is put together in shared memory (background -s_e D, then the chosen experts) and stored whole.
// Reading logits and writing gradients once is all the memory traffic there is: HBM bounds a batch.
#include "common.cuh"

namespace moe_rd {

int device_sms();

namespace {

constexpr int kRwThreads = 256;
constexpr int kRwWarps = kRwThreads / 32;

struct RwArgs {
  const float* logits;
  const int32_t* ids;
  const float* logit_bias;    // or null
  const float* select_bias;   // added to the chosen scores, or null
  const float* grad_weights;  // backward
  float* out;                 // weights [T,K], or grad_logits [T,E]
  int64_t T;
  int E, K, renorm;
  float routed_scale, norm_min;
};

template <bool SOFTMAX, bool BACKWARD>
__global__ void __launch_bounds__(kRwThreads) routing_weights_kernel(const RwArgs a) {
  constexpr int kPer = kMaxE / 32;
  __shared__ float s_row[BACKWARD ? kRwWarps : 1][BACKWARD ? kMaxE : 1];
  pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t t = (int64_t)blockIdx.x * kRwWarps + warp; t < a.T; t += (int64_t)gridDim.x * kRwWarps) {
    const float* row = a.logits + (size_t)t * a.E;
    const int id = lane < a.K ? __ldg(a.ids + (size_t)t * a.K + lane) : -1;
    const bool valid = (unsigned)id < (unsigned)a.E;
    const float gw = BACKWARD && valid ? __ldg(a.grad_weights + (size_t)t * a.K + lane) : 0.0f;
    const float zb = valid && a.logit_bias != nullptr ? __ldg(a.logit_bias + id) : 0.0f;
    const float zk = valid ? __fadd_rn(__ldg(row + id), zb) : 0.0f;
    const float kb = valid && a.select_bias != nullptr ? __ldg(a.select_bias + id) : 0.0f;
    const bool any = __any_sync(kFull, valid);

    float p[SOFTMAX ? kPer : 1];
    float sk = 0.0f;    // score of this lane's slot
    float dsk = 0.0f;   // sigmoid: its derivative
    float inv = 0.0f;   // softmax: 1 / sum
    if (SOFTMAX) {
      float m = -__int_as_float(0x7f800000);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        p[i] = e < a.E ? __ldg(row + e) : -__int_as_float(0x7f800000);
        if (a.logit_bias != nullptr && e < a.E) p[i] = __fadd_rn(p[i], __ldg(a.logit_bias + e));
        m = fmaxf(m, p[i]);
      }
      m = warp_max(m);
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        p[i] = lane + 32 * i < a.E ? expf(__fsub_rn(p[i], m)) : 0.0f;
        sum = __fadd_rn(sum, p[i]);
      }
      inv = __fdiv_rn(1.0f, warp_tree_sum(sum));
      sk = valid ? __fmul_rn(expf(__fsub_rn(zk, m)), inv) : 0.0f;
    } else if (valid) {
      const float q = expf(-fabsf(zk));
      const float r = __fdiv_rn(1.0f, __fadd_rn(1.0f, q));
      sk = zk >= 0.0f ? r : __fmul_rn(q, r);
      if (zk != zk) sk = zk;
      dsk = __fmul_rn(__fmul_rn(q, r), r);
    }
    const float u = valid ? __fadd_rn(sk, kb) : 0.0f;
    float total = 0.0f;
    if (a.renorm) total = warp_tree_sum(u);

    if (!BACKWARD) {
      if (lane < a.K) {
        const float w = a.renorm ? __fdiv_rn(u, fmaxf(total, a.norm_min)) : u;
        a.out[(size_t)t * a.K + lane] = valid ? __fmul_rn(w, a.routed_scale) : 0.0f;
      }
      continue;
    }

    float h = __fmul_rn(a.routed_scale, gw);
    bool no_background = !SOFTMAX;
    if (a.renorm) {
      const bool moving = total >= a.norm_min;
      if (moving) {
        const float part = __fdiv_rn(u, total);
        float diff = 0.0f;
        for (int k = 0; k < a.K; ++k) {
          const float other = __shfl_sync(kFull, h, k), share = __shfl_sync(kFull, part, k);
          if (share != 0.0f) diff = fmaf(share, __fsub_rn(h, other), diff);
        }
        h = diff;
        if (a.select_bias == nullptr) no_background = true;
      }
      h = valid ? __fdiv_rn(h, moving ? total : a.norm_min) : 0.0f;
    }
    // slots with the same expert are added by the first of them, in slot order
    const unsigned same = __match_any_sync(kFull, valid ? id : -1 - lane);
    const bool leader = valid && (same & ((1u << lane) - 1u)) == 0u;
    if (__any_sync(kFull, valid && (same & (same - 1u)) != 0u)) {
      float sum = 0.0f;
      for (int k = 0; k < a.K; ++k) {
        const float other = __shfl_sync(kFull, h, k);
        if ((same >> k) & 1u) sum = __fadd_rn(sum, other);
      }
      h = sum;
    }
    float mine = leader ? __fmul_rn(SOFTMAX ? sk : dsk, h) : 0.0f;
    float back = 0.0f;
    if (SOFTMAX && !no_background) {
      back = warp_tree_sum(mine);
      float diff = 0.0f;
      unsigned chosen = 0u;  // of this lane's experts
      for (int k = 0; k < a.K; ++k) {
        const float other = __shfl_sync(kFull, h, k), score = __shfl_sync(kFull, leader ? sk : 0.0f, k);
        const int e = __shfl_sync(kFull, valid ? id : -1, k);
        if (score != 0.0f) diff = fmaf(score, __fsub_rn(h, other), diff);
        if (e >= 0 && (e & 31) == lane) chosen |= 1u << (e >> 5);
      }
      float rest = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (!((chosen >> i) & 1u)) rest = __fadd_rn(rest, p[SOFTMAX ? i : 0]);
      rest = __fmul_rn(warp_tree_sum(rest), inv);
      mine = __fmul_rn(sk, fmaf(h, rest, diff));
    }
    float* s = s_row[warp];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < a.E) s[e] = SOFTMAX && any && !no_background ? -__fmul_rn(__fmul_rn(p[SOFTMAX ? i : 0], inv), back) : 0.0f;
    }
    __syncwarp();
    if (leader) s[id] = mine;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i;
      if (e < a.E) __stcs(a.out + (size_t)t * a.E + e, s[e]);
    }
    __syncwarp();
  }
}

int check(int64_t T, int32_t E, int32_t K, int32_t score_fn) {
  if (E < 1 || E > kMaxE || K < 1 || K > kMaxK || T < 0 || T > ((int64_t)1 << 31) / K - 1) return MOE_RD_E_SHAPE;
  if (score_fn != MOE_RD_SCORE_SOFTMAX && score_fn != MOE_RD_SCORE_SIGMOID) return MOE_RD_E_ENUM;
  return MOE_RD_OK;
}

template <bool BACKWARD>
int launch(const RwArgs& a, int32_t score_fn, void* stream) {
  const int64_t want = (a.T + kRwWarps - 1) / kRwWarps;
  const int64_t cap = (int64_t)device_sms() * 32;
  const dim3 grid((unsigned)(want < cap ? want : cap));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = score_fn == MOE_RD_SCORE_SOFTMAX
                            ? launch_pdl(routing_weights_kernel<true, BACKWARD>, grid, dim3(kRwThreads), 0, s, a)
                            : launch_pdl(routing_weights_kernel<false, BACKWARD>, grid, dim3(kRwThreads), 0, s, a);
  count_launch();
  if (e != cudaSuccess) set_last_cuda_error(e);
  return e == cudaSuccess ? MOE_RD_OK : MOE_RD_E_CUDA;
}

}  // namespace
}  // namespace moe_rd

using namespace moe_rd;

extern "C" int moe_rd_routing_weights(int64_t T, int32_t E, int32_t K, int32_t score_fn, int32_t renorm,
                                      float routed_scale, float norm_min, const float* logits,
                                      const int32_t* expert_ids, const float* logit_bias, const float* select_bias,
                                      float* weights, void* stream) {
  const int rc = check(T, E, K, score_fn);
  if (rc != MOE_RD_OK) return rc;
  if (T == 0) return MOE_RD_OK;
  if (logits == nullptr || expert_ids == nullptr || weights == nullptr) return MOE_RD_E_NULL;
  const RwArgs a = {logits, expert_ids, logit_bias, select_bias, nullptr, weights, T, E, K, renorm, routed_scale, norm_min};
  return launch<false>(a, score_fn, stream);
}

extern "C" int moe_rd_routing_weights_backward(int64_t T, int32_t E, int32_t K, int32_t score_fn, int32_t renorm,
                                               float routed_scale, float norm_min, const float* logits,
                                               const int32_t* expert_ids, const float* logit_bias,
                                               const float* select_bias, const float* grad_weights,
                                               float* grad_logits, void* stream) {
  const int rc = check(T, E, K, score_fn);
  if (rc != MOE_RD_OK) return rc;
  if (T == 0) return MOE_RD_OK;
  if (logits == nullptr || expert_ids == nullptr || grad_weights == nullptr || grad_logits == nullptr)
    return MOE_RD_E_NULL;
  const RwArgs a = {logits, expert_ids, logit_bias, select_bias, grad_weights, grad_logits, T, E, K, renorm, routed_scale, norm_min};
  return launch<true>(a, score_fn, stream);
}
