// What the attention kernels on the 5th-generation tensor cores share: packed fp32 arithmetic, the base-2
// exponential, TMA boxes and the tensor maps behind them.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "tcgen05.cuh"

namespace inq {

__device__ __forceinline__ void pf_arrive(unsigned mbar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mbar) : "memory");
}
__device__ __forceinline__ float pf_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 values in one 64-bit register, for the packed units
__device__ __forceinline__ unsigned long long pf_pair(float lo, float hi) {
  unsigned long long d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void pf_unpair(unsigned long long d, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d));
}
__device__ __forceinline__ unsigned long long pf_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long pf_add2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x of a pair on the FMA units, beside the exponential unit that bounds kernels of many exponentials: x = n + f with
// n the nearest integer (it falls into the low bits of x + 3 2^22) and |f| <= 1/2, 2^f by a polynomial, n added to its
// exponent.  The polynomials are minimax fits of the relative error on that interval (Remez exchange), in fp32 off by at
// most 7.5e-5, 2.7e-6 and 2.2e-7 for degrees 3, 4 and 5.  x is at most 126 and counts as -126 below that, so that 2^-126
// stands for anything smaller, zero included; a NaN stays one.
template <int DEGREE>
__device__ __forceinline__ void pf_exp2_fma(unsigned long long x2, float& e0, float& e1) {
  static_assert(DEGREE >= 3 && DEGREE <= 5, "a polynomial of these");
  constexpr float kFit[3][6] = {{0.9999280571937561f, 0.6932609677314758f, 0.2426111251115799f, 0.0551716685295105f, 0.f, 0.f},
                                {0.9999992847442627f, 0.6931217908859253f, 0.240247443318367f, 0.05591785907745361f, 0.009570102207362652f, 0.f},
                                {1.0000001192092896f, 0.6931469440460205f, 0.24022120237350464f, 0.05550713092088699f, 0.009675540961325169f,
                                 0.0013276472454890609f}};
  constexpr float kShift = 12582912.f;
  float x0, x1;
  pf_unpair(x2, x0, x1);
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x0) : "f"(x0), "f"(-126.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x1) : "f"(x1), "f"(-126.f));
  x2 = pf_pair(x0, x1);
  const unsigned long long t2 = pf_add2(x2, pf_pair(kShift, kShift)), n2 = pf_add2(t2, pf_pair(-kShift, -kShift));
  const unsigned long long f2 = pf_fma2(n2, pf_pair(-1.f, -1.f), x2);
  unsigned long long p2 = pf_pair(kFit[DEGREE - 3][DEGREE], kFit[DEGREE - 3][DEGREE]);
#pragma unroll
  for (int k = DEGREE - 1; k >= 0; --k) p2 = pf_fma2(p2, f2, pf_pair(kFit[DEGREE - 3][k], kFit[DEGREE - 3][k]));
  float t0, t1, p0, p1;
  pf_unpair(t2, t0, t1);
  pf_unpair(p2, p0, p1);
  e0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  e1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}
template <typename QT>
__device__ __forceinline__ unsigned pf_pack2(float lo, float hi) {
  if (std::is_same<QT, __half>::value) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&h);
  }
  __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<unsigned*>(&b);
}

// One TMA box: 64 columns (128 bytes) x `rows` rows of head `z`, starting at column x and row y, into
// a swizzled slab; rows beyond the tensor are zero-filled by the hardware.
__device__ __forceinline__ void pf_tma(unsigned dst, const CUtensorMap* map, int x, int y, int z, unsigned mbar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(mbar) : "memory");
}
__device__ __forceinline__ void pf_expect(unsigned mbar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mbar), "r"(bytes) : "memory");
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &result) == cudaSuccess &&
        result == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  }
  return fn;
}
// [heads][tokens][dim] tensor of 2-byte elements, boxes of 64 columns x `box_rows` rows, 128-byte swizzle
inline bool make_map(CUtensorMap* map, const void* base, int dtype, int dim, long long tokens, long long heads, long long stride_t,
                     long long stride_h, int box_rows) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  if (heads == 1) stride_h = tokens * stride_t;   // unused, but must be a valid stride
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)tokens, (cuuint64_t)heads};
  const cuuint64_t strides[2] = {(cuuint64_t)stride_t * 2, (cuuint64_t)stride_h * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, dtype == INQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)base, dims,
            strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace inq
