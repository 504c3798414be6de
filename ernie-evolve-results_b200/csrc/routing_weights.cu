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
// Reading logits and writing gradients once is all the memory traffic there is, so HBM should bound a batch; what has to
// be kept small is the number of instructions per token.  W = 4, 8, 16 or 32 lanes (the fewest that K slots fit in) share a
// token, so that a warp works on 8, 4, 2 or 1 at a time: the slots, the reductions and the sums over pairs of slots cost a
// warp the same whether its lanes belong to one token or to four.  The softmax needs every logit of the token (16-byte
// loads where E and the address allow it), the sigmoid only those of the chosen experts.  The gradient row is put together
// in shared memory (background -s_e D, then the chosen experts) and stored whole.
// 32768 tokens, 128 experts, K = 8, softmax: 10.1 us, against 27 us with a warp per token.  Of 4 lanes and 8 (gradient): 32768
// tokens, 64 experts, K = 4 6.3 / 8.4 us, 16 experts 3.3 / 7.0; 8192 tokens, 64 experts 4.9 / 4.5, which is why few
// tokens keep 8 there: the logits of a token are then more lanes' work, and the SMs are not full.
#include "common.cuh"

namespace moe_rd {

int device_sms();

namespace {

constexpr int kRwThreads = 256;
constexpr int kManyTokens = 16384;

struct RwArgs {
  const float* logits;
  const int32_t* ids;
  const float* logit_bias;    // or null
  const float* select_bias;   // added to the chosen scores, or null
  const float* grad_weights;  // backward
  float* out;                 // weights [T,K], or grad_logits [T,E]
  int64_t T;
  int E, K, renorm;
  int vec;                    // rows of logits (and of their gradient) are whole 16-byte vectors
  float routed_scale, norm_min;
};

// Over the W lanes of a token, by the tree v[l] += v[l ^ off].
template <int W>
__device__ __forceinline__ float token_sum(float v) {
#pragma unroll
  for (int o = W / 2; o; o >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// Each lane holds up to LOGITS of them (E <= W * LOGITS).
template <int W, int LOGITS, bool SOFTMAX, bool BACKWARD>
__global__ void __launch_bounds__(kRwThreads, LOGITS <= 16 ? 4 : 3) routing_weights_kernel(const RwArgs a) {
  constexpr int kPer = SOFTMAX ? LOGITS : 1;
  constexpr int kTokens = kRwThreads / W;        // of a block
  constexpr float kInf = __builtin_huge_valf();
  extern __shared__ __align__(16) float s_rows[];  // BACKWARD: [kTokens][E rounded up to 4]
  pdl_sync();
  const int lane = threadIdx.x & 31, slot = lane & (W - 1), in_block = threadIdx.x / W;
  const int E4 = (a.E + 3) & ~3;
  float* s_row = BACKWARD ? s_rows + in_block * E4 : nullptr;
  // all lanes of a warp stay in the loop for its last token
  for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < a.T; t0 += (int64_t)gridDim.x * kTokens) {
    const int64_t t = t0 + in_block;
    const bool live = t < a.T;
    const float* row = a.logits + (size_t)(live ? t : 0) * a.E;
    const int id = live && slot < a.K ? __ldg(a.ids + (size_t)t * a.K + slot) : -1;
    const bool valid = (unsigned)id < (unsigned)a.E;

    float p[kPer];
    if (SOFTMAX) {
      if (a.vec) {
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i) {
          const int e = 4 * (slot + W * i);
          float4 v = make_float4(-kInf, -kInf, -kInf, -kInf);
          if (e < a.E) v = __ldg(reinterpret_cast<const float4*>(row + e));
          p[4 * i] = v.x;
          p[4 * i + 1] = v.y;
          p[4 * i + 2] = v.z;
          p[4 * i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int e = 4 * (slot + W * (i / 4)) + i % 4;
          p[i] = e < a.E ? __ldg(row + e) : -kInf;
        }
      }
    }
    const float gw = BACKWARD && valid ? __ldg(a.grad_weights + (size_t)t * a.K + slot) : 0.0f;
    const float zb = valid && a.logit_bias != nullptr ? __ldg(a.logit_bias + id) : 0.0f;
    const float zk = valid ? __fadd_rn(__ldg(row + id), zb) : 0.0f;
    const float kb = valid && a.select_bias != nullptr ? __ldg(a.select_bias + id) : 0.0f;

    float sk = 0.0f;   // score of this lane's slot
    float dsk = 0.0f;  // sigmoid: its derivative
    float inv = 0.0f;  // softmax: 1 / sum
    if (SOFTMAX) {
      if (a.logit_bias != nullptr) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int e = 4 * (slot + W * (i / 4)) + i % 4;
          if (e < a.E) p[i] = __fadd_rn(p[i], __ldg(a.logit_bias + e));
        }
      }
      float m = -kInf;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (4 * W * (i / 4) < a.E) m = fmaxf(m, p[i]);
#pragma unroll
      for (int o = W / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (4 * W * (i / 4) < a.E) {  // the same for all lanes
          const bool mine = 4 * (slot + W * (i / 4)) + i % 4 < a.E;
          p[i] = mine ? expf(__fsub_rn(p[i], m)) : 0.0f;
          sum = __fadd_rn(sum, p[i]);
        }
      }
      inv = __fdiv_rn(1.0f, token_sum<W>(sum));
      sk = valid ? __fmul_rn(expf(__fsub_rn(zk, m)), inv) : 0.0f;
    } else if (valid) {
      const float q = expf(-fabsf(zk));
      const float r = __fdiv_rn(1.0f, __fadd_rn(1.0f, q));
      sk = zk >= 0.0f ? r : __fmul_rn(q, r);
      if (zk != zk) sk = zk;
      dsk = __fmul_rn(__fmul_rn(q, r), r);
    }
    const float u = valid ? __fadd_rn(sk, kb) : 0.0f;
    float total = 1.0f, divisor = 1.0f;
    if (a.renorm) {
      total = token_sum<W>(u);
      divisor = total < a.norm_min ? a.norm_min : total;  // a sum that is no number stays one
    }

    if (!BACKWARD) {
      if (live && slot < a.K) {
        const float w = a.renorm ? __fdiv_rn(u, divisor) : u;
        a.out[(size_t)t * a.K + slot] = valid ? __fmul_rn(w, a.routed_scale) : 0.0f;
      }
      continue;
    }

    float h = __fmul_rn(a.routed_scale, gw);
    bool flat = !SOFTMAX;  // D = 0: no gradient but that of the chosen experts
    if (a.renorm) {
      const bool moving = !(total < a.norm_min);
      const float part = __fdiv_rn(u, total);
      float diff = 0.0f;
      for (int k = 0; k < a.K; ++k) {
        const float other = __shfl_sync(kFull, h, k, W), share = __shfl_sync(kFull, part, k, W);
        if (share != 0.0f) diff = fmaf(share, __fsub_rn(h, other), diff);
      }
      if (moving) {
        h = diff;
        if (a.select_bias == nullptr) flat = true;
      }
      h = valid ? __fdiv_rn(h, divisor) : 0.0f;
    }
    // slots with the same expert are added by the first of them, in slot order
    const unsigned group = W == 32 ? kFull : (((1u << W) - 1u) << (lane & ~(W - 1)));
    const unsigned same = __match_any_sync(kFull, valid ? id : -1 - lane) & group;
    const bool leader = valid && (same & ((1u << lane) - 1u)) == 0u;
    if (__any_sync(kFull, valid && (same & (same - 1u)) != 0u)) {
      float sum = 0.0f;
      for (int k = 0; k < a.K; ++k) {
        const float other = __shfl_sync(kFull, h, k, W);
        if ((same >> ((lane & ~(W - 1)) + k)) & 1u) sum = __fadd_rn(sum, other);
      }
      h = sum;
    }
    float mine = leader ? __fmul_rn(SOFTMAX ? sk : dsk, h) : 0.0f;
    float back = 0.0f;
    const bool any = (__ballot_sync(kFull, valid) & group) != 0u;
    if (SOFTMAX && __any_sync(kFull, !flat)) {
      back = token_sum<W>(mine);
      float diff = 0.0f;
      unsigned chosen = 0u;  // of this lane's experts
      for (int k = 0; k < a.K; ++k) {
        const float other = __shfl_sync(kFull, h, k, W), score = __shfl_sync(kFull, leader ? sk : 0.0f, k, W);
        const int e = __shfl_sync(kFull, valid ? id : -1, k, W);
        if (score != 0.0f) diff = fmaf(score, __fsub_rn(h, other), diff);
        if (e >= 0 && ((e >> 2) & (W - 1)) == slot) chosen |= 1u << ((e >> 2) / W * 4 + (e & 3));
      }
      float rest = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (4 * W * (i / 4) < a.E && !((chosen >> i) & 1u)) rest = __fadd_rn(rest, p[i]);
      rest = __fmul_rn(token_sum<W>(rest), inv);
      if (!flat && leader) mine = __fmul_rn(sk, fmaf(h, rest, diff));
    }
    const bool plain = flat || !any;  // a token without a valid id gets zeros whatever its logits are
    const float down = __fmul_rn(-inv, back);
    if (a.vec) {
      for (int i = 0; 4 * W * i < a.E; ++i) {
        const int e = 4 * (slot + W * i);
        if (e < a.E) *reinterpret_cast<float4*>(s_row + e) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      if (SOFTMAX && !plain) {
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i) {
          const int e = 4 * (slot + W * i);
          if (e < a.E)
            *reinterpret_cast<float4*>(s_row + e) = make_float4(__fmul_rn(p[SOFTMAX ? 4 * i : 0], down), __fmul_rn(p[SOFTMAX ? 4 * i + 1 : 0], down),
                                                                __fmul_rn(p[SOFTMAX ? 4 * i + 2 : 0], down), __fmul_rn(p[SOFTMAX ? 4 * i + 3 : 0], down));
        }
      }
    } else {
      for (int e = slot; e < a.E; e += W) s_row[e] = 0.0f;
      __syncwarp();
      if (SOFTMAX && !plain) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int e = 4 * (slot + W * (i / 4)) + i % 4;
          if (e < a.E) s_row[e] = __fmul_rn(p[i], down);
        }
      }
    }
    __syncwarp();
    if (leader) s_row[id] = mine;
    __syncwarp();
    if (live) {
      float* out = a.out + (size_t)t * a.E;
      if (a.vec) {
        for (int e = 4 * slot; e < a.E; e += 4 * W) __stcs(reinterpret_cast<float4*>(out + e), *reinterpret_cast<const float4*>(s_row + e));
      } else {
        for (int e = slot; e < a.E; e += W) __stcs(out + e, s_row[e]);
      }
    }
    __syncwarp();
  }
}

int check(int64_t T, int32_t E, int32_t K, int32_t score_fn) {
  if (E < 1 || E > kMaxE || K < 1 || K > kMaxK || T < 0 || T > ((int64_t)1 << 31) / K - 1) return MOE_RD_E_SHAPE;
  if (score_fn != MOE_RD_SCORE_SOFTMAX && score_fn != MOE_RD_SCORE_SIGMOID) return MOE_RD_E_ENUM;
  return MOE_RD_OK;
}

template <int W, int LOGITS, bool BACKWARD>
cudaError_t launch_wide(const RwArgs& a, int32_t score_fn, cudaStream_t s) {
  constexpr int kTokens = kRwThreads / W;
  const int64_t want = (a.T + kTokens - 1) / kTokens;
  const int64_t cap = (int64_t)device_sms() * 32;
  const dim3 grid((unsigned)(want < cap ? want : cap));
  const size_t smem = BACKWARD ? (size_t)kTokens * ((a.E + 3) & ~3) * 4 : 0;  // at most 32 KB
  return score_fn == MOE_RD_SCORE_SOFTMAX
             ? launch_pdl(routing_weights_kernel<W, LOGITS, true, BACKWARD>, grid, dim3(kRwThreads), smem, s, a)
             : launch_pdl(routing_weights_kernel<W, LOGITS, false, BACKWARD>, grid, dim3(kRwThreads), smem, s, a);
}

template <bool BACKWARD>
int launch(RwArgs a, int32_t score_fn, void* stream) {
  a.vec = a.E % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.logits) | (BACKWARD ? reinterpret_cast<uintptr_t>(a.out) : 0)) & 15) == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.K <= 4 && a.E <= 16                     ? launch_wide<4, 4, BACKWARD>(a, score_fn, s)
                        : a.K <= 4 && a.E <= 64 && a.T > kManyTokens ? launch_wide<4, 16, BACKWARD>(a, score_fn, s)
                        : a.K <= 8 && a.E <= 128                     ? launch_wide<8, 16, BACKWARD>(a, score_fn, s)
                        : a.K <= 8                                   ? launch_wide<8, 32, BACKWARD>(a, score_fn, s)
                        : a.K <= 16                                  ? launch_wide<16, 16, BACKWARD>(a, score_fn, s)
                                                                     : launch_wide<32, 8, BACKWARD>(a, score_fn, s);
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
  const RwArgs a = {logits, expert_ids, logit_bias, select_bias, nullptr, weights, T, E, K, renorm, 0, routed_scale, norm_min};
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
  const RwArgs a = {logits, expert_ids, logit_bias, select_bias, grad_weights, grad_logits, T, E, K, renorm, 0, routed_scale, norm_min};
  return launch<true>(a, score_fn, stream);
}
