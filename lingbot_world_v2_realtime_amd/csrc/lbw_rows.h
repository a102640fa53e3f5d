// Row access shared by the block operators: 8 consecutive values of a row in registers as fp32, in any of the three
// element formats, and sums over a wave.
#pragma once

#include "lbw_block.h"
#include "lbw_common.h"

namespace lbw {

// Workgroups in any number below 2^32, which group_id() counts in 32 bits (the entry points take 2^30 at most): a grid
// dimension holds fewer than 2^32 threads, so past 2^20 workgroups there is a second one, whose last part may have
// workgroups past the end.
constexpr unsigned GRID_X = 1u << 20;
inline dim3 grid_of(int64_t n) {
  return dim3((unsigned)(n < GRID_X ? n : GRID_X), (unsigned)((n + GRID_X - 1) / GRID_X));
}
__device__ __forceinline__ uint32_t group_id() { return blockIdx.x + blockIdx.y * GRID_X; }

constexpr int elem_size(int dt) { return dt == LBW_DTYPE_FP32 ? 4 : 2; }

// One value.
template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == LBW_DTYPE_FP32) return ((const float*)p)[i];
  else if constexpr (DT == LBW_DTYPE_FP16) return __half2float(((const __half*)p)[i]);
  else return bf16_to_f32(((const uint16_t*)p)[i]);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (DT == LBW_DTYPE_FP32) ((float*)p)[i] = v;
  else if constexpr (DT == LBW_DTYPE_FP16) ((__half*)p)[i] = __float2half_rn(v);
  else ((__bf16*)p)[i] = (__bf16)v;
}

// Two fp32 values rounded to a word of the 16-bit format (ties to even; NaN stays NaN).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == LBW_DTYPE_FP16) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// The 8 values p[i .. i + 8) as they lie in memory. VEC: i is a multiple of 8 and p 16-byte aligned (two loads of 16
// bytes for fp32); else value by value, those at or past `end` read as zero.
template <int DT, bool VEC>
struct Raw8 {
  v4i w[DT == LBW_DTYPE_FP32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t i, int64_t end) {
    if constexpr (VEC) {
      const v4i* q = (const v4i*)((const char*)p + i * elem_size(DT));
      w[0] = q[0];
      if constexpr (DT == LBW_DTYPE_FP32) w[1] = q[1];
    } else if constexpr (DT == LBW_DTYPE_FP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e >> 2][e & 3] = i + e < end ? ((const int*)p)[i + e] : 0;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t a = i + 2 * e < end ? ((const uint16_t*)p)[i + 2 * e] : 0u;
        const uint32_t b = i + 2 * e + 1 < end ? ((const uint16_t*)p)[i + 2 * e + 1] : 0u;
        w[0][e] = (int)(a | b << 16);
      }
    }
  }
  __device__ __forceinline__ void zero() {
    w[0] = v4i{0, 0, 0, 0};
    if constexpr (DT == LBW_DTYPE_FP32) w[1] = v4i{0, 0, 0, 0};
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (DT == LBW_DTYPE_FP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __int_as_float(w[e >> 2][e & 3]);
    } else {
      unpack8t<DT == LBW_DTYPE_FP16>(w[0], f);
    }
  }
};

template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* p, int64_t i, int64_t end, const float* f) {
  if constexpr (!VEC) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < end) store1<DT>(p, i + e, f[e]);
  } else if constexpr (DT == LBW_DTYPE_FP32) {
    v4i* q = (v4i*)((float*)p + i);
    q[0] = v4i{__float_as_int(f[0]), __float_as_int(f[1]), __float_as_int(f[2]), __float_as_int(f[3])};
    q[1] = v4i{__float_as_int(f[4]), __float_as_int(f[5]), __float_as_int(f[6]), __float_as_int(f[7])};
  } else {
    *(v4i*)((uint16_t*)p + i) = v4i{(int)pack2<DT>(f[0], f[1]), (int)pack2<DT>(f[2], f[3]),
                                    (int)pack2<DT>(f[4], f[5]), (int)pack2<DT>(f[6], f[7])};
  }
}

// Sum over the wave's 64 lanes, the same bits in every lane.
__device__ __forceinline__ float wave_sum(float x) {
  x = row16_sum(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

}  // namespace lbw
