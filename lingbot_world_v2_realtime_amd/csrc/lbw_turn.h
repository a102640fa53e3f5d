// What the kernels that turn q and k by their positions share: units of consecutive values, and the sine and cosine of a
// position's angle.
#pragma once

#include <type_traits>

#include "lbw_rows.h"

namespace lbw {

// N consecutive values: 16 bytes, 8, or one value; as they lie in memory, too, for loads that run ahead
template <int DT, int N>
struct Unit {
  static constexpr int WORDS = N * elem_size(DT) / 4;
  struct One {
    float v;
    __device__ __forceinline__ One() {}
    __device__ __forceinline__ One(int x) : v((float)x) {}
  };
  typedef int vec __attribute__((ext_vector_type(WORDS > 0 ? WORDS : 1)));
  typedef std::conditional_t<N == 1, One, vec> Raw;
  float f[N];
  static __device__ __forceinline__ Raw raw(const void* p, int64_t i) {
    if constexpr (N == 1) {
      One r;
      r.v = load1<DT>(p, i);
      return r;
    } else {
      return *(const vec*)((const char*)p + i * elem_size(DT));
    }
  }
  __device__ __forceinline__ void load(const void* p, int64_t i) { set(raw(p, i)); }
  __device__ __forceinline__ void set(const Raw w) {
    if constexpr (N == 1) {
      f[0] = w.v;
    } else {
#pragma unroll
      for (int e = 0; e < WORDS; ++e) {
        if constexpr (DT == LBW_DTYPE_FP32) {
          f[e] = __int_as_float(w[e]);
        } else {
          f[2 * e] = lo16<DT == LBW_DTYPE_FP16>((uint32_t)w[e]);
          f[2 * e + 1] = hi16<DT == LBW_DTYPE_FP16>((uint32_t)w[e]);
        }
      }
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    if constexpr (N == 1) {
      store1<DT>(p, i, f[0]);
    } else {
      vec w;
#pragma unroll
      for (int e = 0; e < WORDS; ++e) {
        if constexpr (DT == LBW_DTYPE_FP32) w[e] = __float_as_int(f[e]);
        else w[e] = (int)pack2<DT>(f[2 * e], f[2 * e + 1]);
      }
      *(vec*)((char*)p + i * elem_size(DT)) = w;
    }
  }
};

// The angle in 64 bits, reduced to (-1/2, 1/2] turns there; its sine and cosine in fp32, for fp32 values moved by what the
// rounding of the reduced angle took off.
template <int DT>
__device__ __forceinline__ void turn_of(int64_t pos, double freq, float& s, float& c) {
  const double turns = (double)pos * freq * 0.15915494309189533577;   // 1 / (2 pi)
  const double half = 2.0 * (turns - rint(turns));
  const float near = (float)half;
  sincospif(near, &s, &c);
  if constexpr (DT == LBW_DTYPE_FP32) {
    const float rest = (float)(half - near) * 3.14159265358979f, s0 = s;
    s = fmaf(c, rest, s);
    c = fmaf(-s0, rest, c);
  }
}

}  // namespace lbw
