// Rows of any element type (moe_rd_sort_tokens, moe_rd_unsort_tokens and their gradients): a 16-byte vector of a row
// as fp32 values and back.  Every conversion to fp32 is exact; pack rounds each value once, to nearest even.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace moe_rd {

// Argument checks shared by the entry points that take such rows.
inline int check_rows(int64_t T, int32_t H, int32_t K, int32_t dtype, int64_t rows) {
  if (dtype != MOE_RD_T_BF16 && dtype != MOE_RD_T_FP16 && dtype != MOE_RD_T_F32) return MOE_RD_E_ENUM;
  const int per_vec = dtype == MOE_RD_T_F32 ? 4 : 8;
  if (K < 1 || K > kMaxK || T < 0 || T > ((int64_t)1 << 31) / K - 1) return MOE_RD_E_SHAPE;
  if (H < per_vec || H % per_vec != 0 || H > (1 << 20)) return MOE_RD_E_SHAPE;
  if (rows < 0 || rows > 0x7fffffff) return MOE_RD_E_SHAPE;
  return MOE_RD_OK;
}

#ifdef __CUDACC__

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t pack_fp16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int DT>
struct RowVec;

template <>
struct RowVec<MOE_RD_T_BF16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) { unpack8(v, f); }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};

template <>
struct RowVec<MOE_RD_T_FP16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_fp16x2(f[0], f[1]), pack_fp16x2(f[2], f[3]), pack_fp16x2(f[4], f[5]),
                      pack_fp16x2(f[6], f[7]));
  }
};

template <>
struct RowVec<MOE_RD_T_F32> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

#endif  // __CUDACC__

}  // namespace moe_rd
