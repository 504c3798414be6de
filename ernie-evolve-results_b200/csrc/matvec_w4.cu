// Products of few rows with 4-bit expert weights (moe_rd_expert_matvec_w4):
//   out[r,n] = sum_groups scale[n,group] * sum_{k in group} x[r,k] * (q[n,k] - zero[n,group])
//
// Reading the weights (half a byte each) of the experts that have rows is nearly all the traffic, so HBM is the floor.
// A product on the CUDA cores would need one FMA per weight and row; from three rows on that is slower than the
// memory.  So the weights go through the warp's matrix instruction (mma m16n8k16: 16 outputs x 16 inputs times 8
// rows of x): q - zero is an integer in -15..15, exact in bf16 and fp16, and the group's scale multiplies the fp32 sum
// of the group afterwards, so nothing is rounded below 32 bits before the result is.
//
// The weight tile of 16 outputs x 128 inputs is 1 KB, stored so that a lane's two 16-byte loads are its operand
// fragments: word i holds the eight inputs 32i + 8j.. of one output, the pair (2p, 2p+1) in nibbles p of its two
// halves, so that (w >> 4p) & 0x000f000f is a pair of integers; with the exponent bits of 128 (bf16) or 1024 (fp16)
// or'ed in it is a pair of floats 128 + q (1024 + q), from which 128 + zero (1024 + zero) is subtracted exactly.
// Every 16 inputs of one instruction lie inside one block of 32, so groups of 32, 64, 96, ... inputs work alike.
//
// A unit of work is 16 outputs of one expert; the warps of a block split its inputs (tiles warp, warp + 8, ...) and
// their fp32 sums are added in warp order.  Only experts that have rows get units: every block lists them from the
// offsets.
#include "row_types.cuh"

namespace moe_rd {

int device_sms();

namespace {

constexpr int kW4Threads = 256;
constexpr int kW4Warps = kW4Threads / 32;
constexpr int kW4BlocksPerSm = 2;

struct W4Args {
  const unsigned char* x;
  const unsigned char* weight;
  const unsigned char* scales;
  const uint8_t* zeros;
  const int32_t* offsets;
  unsigned char* out;
  int64_t rows;
  int N, K, E, G, group;
  int chunks;  // tiles of 128 inputs
  int nblocks; // tiles of 16 outputs
};

template <int DT>
struct W4Type;

template <>
struct W4Type<MOE_RD_T_BF16> {
  static constexpr uint32_t kBase = 0x43004300u;  // 128 in both halves; the last mantissa bit is worth 1
  static constexpr int kOffset = 128;
  static __device__ __forceinline__ float scale(const unsigned char* p, size_t i) {
    return __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + i) << 16);
  }
  static __device__ __forceinline__ uint32_t both(int v) {
    const __nv_bfloat162 b = __bfloat162bfloat162(__int2bfloat16_rn(v));
    return *reinterpret_cast<const uint32_t*>(&b);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint16_t round(float v) {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    return *reinterpret_cast<const uint16_t*>(&b);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

template <>
struct W4Type<MOE_RD_T_FP16> {
  static constexpr uint32_t kBase = 0x64006400u;  // 1024 in both halves; the last mantissa bit is worth 1
  static constexpr int kOffset = 1024;
  static __device__ __forceinline__ float scale(const unsigned char* p, size_t i) {
    return __half2float(__ushort_as_half(__ldg(reinterpret_cast<const uint16_t*>(p) + i)));
  }
  static __device__ __forceinline__ uint32_t both(int v) {
    const __half2 b = __half2half2(__int2half_rn(v));
    return *reinterpret_cast<const uint32_t*>(&b);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint16_t round(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

template <int DT>
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int p, uint32_t zero) {
  return W4Type<DT>::sub(((word >> (4 * p)) & 0x000f000fu) | W4Type<DT>::kBase, zero);
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int DT, bool ZEROS>
__global__ void __launch_bounds__(kW4Threads, kW4BlocksPerSm) w4_kernel(const W4Args a) {
  using Ty = W4Type<DT>;
  __shared__ int s_expert[kMaxE], s_lo[kMaxE], s_n[kMaxE], s_w[kW4Warps];
  __shared__ float s_sum[kW4Warps][16 * 8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, j = lane & 3;
  pdl_sync();

  // experts that have rows, in order
  int lo = 0, n = 0;
  int64_t first_row = 0, last_row = a.rows;
  if (a.offsets == nullptr) {
    n = tid == 0 ? (int)a.rows : 0;
  } else {
    if (tid < a.E) {
      lo = max(__ldg(a.offsets + tid), 0);
      n = min((int64_t)__ldg(a.offsets + tid + 1), a.rows) - lo;
    }
    first_row = max(__ldg(a.offsets), 0);
    last_row = __ldg(a.offsets + a.E);
  }
  const unsigned busy = __ballot_sync(kFull, n > 0);
  if (lane == 0) s_w[warp] = __popc(busy);
  __syncthreads();
  int at = __popc(busy & ((1u << lane) - 1u)), experts = 0;
#pragma unroll
  for (int w = 0; w < kW4Warps; ++w) {
    if (w < warp) at += s_w[w];
    experts += s_w[w];
  }
  if (n > 0) {
    s_expert[at] = tid;
    s_lo[at] = lo;
    s_n[at] = n;
  }
  __syncthreads();

  const int64_t units = (int64_t)experts * a.nblocks;
  const int64_t u_end = units * (blockIdx.x + 1) / gridDim.x;
  for (int64_t u = units * blockIdx.x / gridDim.x; u < u_end; ++u) {
    const int i = (int)(u / a.nblocks), nb = (int)(u - (int64_t)i * a.nblocks);
    const int e = s_expert[i], rows_e = s_n[i];
    const size_t block = (size_t)e * a.nblocks + nb;
    const unsigned char* wp = a.weight + block * a.chunks * 1024 + lane * 16;
    const size_t sp = block * a.G * 16 + g;
    for (int r0 = 0; r0 < rows_e; r0 += 8) {
      const unsigned char* xp = a.x + ((size_t)(s_lo[i] + r0 + g) * a.K + 8 * j) * 2;
      const bool has = r0 + g < rows_e;
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int c = warp; c < a.chunks; c += kW4Warps) {
        const uint4 wa = ld_stream(wp + (size_t)c * 1024), wb = ld_stream(wp + (size_t)c * 1024 + 512);
        uint4 xv[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          xv[q] = has && 128 * c + 32 * q < a.K ? __ldg(reinterpret_cast<const uint4*>(xp + (size_t)(128 * c + 32 * q) * 2))
                                                : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t ua[4] = {wa.x, wa.y, wa.z, wa.w}, ub[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int gr = min((128 * c + 32 * q) / a.group, a.G - 1);
          const float sa = Ty::scale(a.scales, sp + (size_t)gr * 16), sb = Ty::scale(a.scales, sp + (size_t)gr * 16 + 8);
          const uint32_t za = Ty::both(Ty::kOffset + (ZEROS ? (int)__ldg(a.zeros + sp + (size_t)gr * 16) : 8));
          const uint32_t zb = Ty::both(Ty::kOffset + (ZEROS ? (int)__ldg(a.zeros + sp + (size_t)gr * 16 + 8) : 8));
          float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          Ty::mma(part, w4_pair<DT>(ua[q], 0, za), w4_pair<DT>(ub[q], 0, zb), w4_pair<DT>(ua[q], 1, za),
                  w4_pair<DT>(ub[q], 1, zb), xv[q].x, xv[q].y);
          Ty::mma(part, w4_pair<DT>(ua[q], 2, za), w4_pair<DT>(ub[q], 2, zb), w4_pair<DT>(ua[q], 3, za),
                  w4_pair<DT>(ub[q], 3, zb), xv[q].z, xv[q].w);
          acc[0] = fmaf(sa, part[0], acc[0]);
          acc[1] = fmaf(sa, part[1], acc[1]);
          acc[2] = fmaf(sb, part[2], acc[2]);
          acc[3] = fmaf(sb, part[3], acc[3]);
        }
      }
      // [row of x][output]
      s_sum[warp][(2 * j) * 16 + g] = acc[0];
      s_sum[warp][(2 * j + 1) * 16 + g] = acc[1];
      s_sum[warp][(2 * j) * 16 + g + 8] = acc[2];
      s_sum[warp][(2 * j + 1) * 16 + g + 8] = acc[3];
      __syncthreads();
      if (tid < 128) {
        float sum = s_sum[0][tid];
#pragma unroll
        for (int w = 1; w < kW4Warps; ++w) sum = __fadd_rn(sum, s_sum[w][tid]);
        const int r = r0 + (tid >> 4), col = nb * 16 + (tid & 15);
        if (r < rows_e && col < a.N)
          reinterpret_cast<uint16_t*>(a.out)[(size_t)(s_lo[i] + r) * a.N + col] = Ty::round(sum);
      }
      __syncthreads();
    }
  }

  // rows of no expert
  if (first_row > a.rows) first_row = a.rows;
  if (last_row < first_row) last_row = first_row;
  const int64_t before = first_row * a.N;
  const int64_t idle = before + (last_row < a.rows ? (a.rows - last_row) * a.N : 0);
  for (int64_t k = (int64_t)blockIdx.x * kW4Threads + tid; k < idle; k += (int64_t)gridDim.x * kW4Threads)
    reinterpret_cast<uint16_t*>(a.out)[k < before ? k : last_row * a.N + (k - before)] = 0;
}

}  // namespace
}  // namespace moe_rd

using namespace moe_rd;

extern "C" int moe_rd_expert_matvec_w4(int64_t rows, int32_t N, int32_t K, int32_t E, int32_t group, int32_t dtype,
                                       const void* x, const void* weight, const void* scales, const uint8_t* zeros,
                                       const int32_t* offsets, void* out, void* stream) {
  if (dtype == MOE_RD_T_F32) return MOE_RD_E_UNSUPPORTED;
  if (dtype != MOE_RD_T_BF16 && dtype != MOE_RD_T_FP16) return MOE_RD_E_ENUM;
  if (rows < 0 || rows > 0x7fffffff || N < 1 || N > (1 << 24) || K < 32 || K > (1 << 20) || E < 1 || E > kMaxE ||
      group < 32 || group % 32 != 0 || K % group != 0 || (offsets == nullptr && E != 1))
    return MOE_RD_E_SHAPE;
  if (rows == 0) return MOE_RD_OK;
  if (x == nullptr || weight == nullptr || scales == nullptr || out == nullptr) return MOE_RD_E_NULL;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(weight)) & 15 ||
      (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scales)) & 1)
    return MOE_RD_E_ALIGN;
  W4Args a = {};
  a.x = static_cast<const unsigned char*>(x);
  a.weight = static_cast<const unsigned char*>(weight);
  a.scales = static_cast<const unsigned char*>(scales);
  a.zeros = zeros;
  a.offsets = offsets;
  a.out = static_cast<unsigned char*>(out);
  a.rows = rows;
  a.N = N;
  a.K = K;
  a.E = E;
  a.group = group;
  a.G = K / group;
  a.chunks = (K + 127) / 128;
  a.nblocks = (N + 15) / 16;
  const dim3 grid((unsigned)(device_sms() * kW4BlocksPerSm));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == MOE_RD_T_BF16)
    e = zeros != nullptr ? launch_pdl(w4_kernel<MOE_RD_T_BF16, true>, grid, dim3(kW4Threads), 0, s, a)
                         : launch_pdl(w4_kernel<MOE_RD_T_BF16, false>, grid, dim3(kW4Threads), 0, s, a);
  else
    e = zeros != nullptr ? launch_pdl(w4_kernel<MOE_RD_T_FP16, true>, grid, dim3(kW4Threads), 0, s, a)
                         : launch_pdl(w4_kernel<MOE_RD_T_FP16, false>, grid, dim3(kW4Threads), 0, s, a);
  count_launch();
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return MOE_RD_E_CUDA;
  }
  return MOE_RD_OK;
}
