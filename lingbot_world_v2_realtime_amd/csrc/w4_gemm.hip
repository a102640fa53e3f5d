// Linears with 4-bit weights (include/lbw_block.h): their quantisation, and x w^T with codes that become matrix-core
// operands in registers.
//
// A code enters the products exactly. fp4 converts by the hardware's own instruction. An integer code c becomes 1 + c / 16 in
// the 16-bit format: its four bits placed in the mantissa of 1, a shift and a mask for two codes (converting to the signed integer
// instead takes three more operations a pair). With v = c - z the group's sum is then
//   sum x v = 16 sum x (1 + c / 16) - (16 + z) sum x,
// sum x from one more matrix instruction a step (x times ones) whose result stands where the products' do. Group sums are
// scaled in fp32: out += s (...) for every group, so neither scale nor zero is ever rounded into a 16-bit weight.
#include "lbw_rows.h"

namespace lbw {
namespace {

constexpr int TN = 16, TK = 128;      // a tile of the stored weights
constexpr int TILE_BYTES = TN * TK / 2;

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- quantisation

template <int DPP>
__device__ __forceinline__ void dpp_max_min(float& hi, float& lo) {
  hi = fmaxf(hi, dpp<DPP>(hi));
  lo = fminf(lo, dpp<DPP>(lo));
}

// A workgroup makes one tile: 16 lanes a row, each 8 columns in a row; a group's extremes by DPP within its lanes.
template <bool F32>
__global__ __launch_bounds__(256) void quant_w4_kernel(const void* w, int64_t n, int64_t k, int64_t s_row, int fmt,
                                                       int group, uint8_t* w4, uint16_t* scale, uint8_t* zero) {
#pragma clang fp contract(off)   // a product and a sum rounded each, as written: a fused one moves ties to other codes
  const int r = threadIdx.x >> 4, c8 = threadIdx.x & 15;
  const int64_t kt = blockIdx.x, nt = blockIdx.y, tile = nt * gridDim.x + kt;
  const int64_t row = nt * TN + r, col = kt * TK + 8 * c8;
  float v[8];
  float hi = 0.f, lo = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = row < n && col + e < k ? load1<F32 ? LBW_DTYPE_FP32 : LBW_DTYPE_BF16>(w, row * s_row + col + e) : 0.f;
    hi = fmaxf(hi, v[e]);
    lo = fminf(lo, v[e]);
  }
  dpp_max_min<DPP_XOR1>(hi, lo);
  dpp_max_min<DPP_XOR2>(hi, lo);
  if (group >= 64) dpp_max_min<DPP_HALF_MIRROR>(hi, lo);
  if (group >= 128) dpp_max_min<DPP_MIRROR>(hi, lo);
  const float amax = fmaxf(hi, -lo);
  const float want = __fdiv_rn(fmt == LBW_W4_FP4 || !zero ? amax : hi - lo, fmt == LBW_W4_FP4 ? 6.f : zero ? 15.f : 7.f);
  float s = bf16_round(want);
  if (!(s >= 1.17549435e-38f)) s = 0.f;   // below the normal numbers: the group counts as zeros
  const float inv = s > 0.f ? __fdiv_rn(1.f, s) : 0.f;
  const float z = zero ? fminf(fmaxf(rintf(-lo * inv), 0.f), 15.f) : 8.f;
  uint32_t code[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (fmt == LBW_W4_FP4) {
      const float u = s > 0.f ? __fdiv_rn(v[e], s) : 0.f, m = fabsf(u);
      code[e] = (m > 0.25f) + (m > 0.75f) + (m > 1.25f) + (m > 1.75f) + (m > 2.5f) + (m > 3.5f) + (m > 5.f) +
                (u < 0.f ? 8u : 0u);
    } else {
      code[e] = (uint32_t)fminf(fmaxf(rintf(v[e] * inv + z), 0.f), 15.f);
    }
  }
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) word |= code[i] << 4 * (fmt == LBW_W4_FP4 ? i : (i >> 1) + 4 * (i & 1));
  ((uint32_t*)(w4 + tile * TILE_BYTES))[4 * (TN * (c8 & 3) + r) + (c8 >> 2)] = word;
  const int lanes = group / 8, per = TK / group;
  if (c8 % lanes == 0) {
    const int64_t at = tile * TN * per + r * per + c8 / lanes;
    scale[at] = f32_to_bf16_bits(s);
    if (zero) zero[at] = (uint8_t)z;
  }
}

// ---------------------------------------------------------------- products

template <int DT>
__device__ __forceinline__ v4f mfma(v4i a, v4i b, v4f c) {
  if constexpr (DT == LBW_DTYPE_FP16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

template <int DT>
constexpr uint32_t ONES = DT == LBW_DTYPE_FP16 ? 0x3C003C00u : 0x3F803F80u;

// The 8 codes of a word as 16-bit operands: integer codes as 1 + c / 16, fp4 codes as their values.
template <int DT, bool FP4>
__device__ __forceinline__ v4i operand(uint32_t w) {
  v4i r;
  if constexpr (FP4) {
    if constexpr (DT == LBW_DTYPE_FP16) {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 0));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 1));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 2));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 3));
    } else {
      r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0));
      r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1));
      r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 2));
      r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 3));
    }
  } else {
    // nibbles t and t + 4 (codes 2 t and 2 t + 1) into the top mantissa bits of a pair of ones
    constexpr int S = DT == LBW_DTYPE_FP16 ? 6 : 3;
    constexpr uint32_t M = 0x000F000Fu << S;
#pragma unroll
    for (int t = 0; t < 4; ++t) r[t] = (int)(((4 * t < S ? w << (S - 4 * t) : w >> (4 * t - S)) & M) | ONES<DT>);
  }
  return r;
}

struct GemmArgs {
  const void* x;
  int64_t m, k, x_s_row;
  const uint8_t* w4;
  const uint16_t* scale;
  const uint8_t* zero;
  int64_t n, kt;                    // kt: tiles along K
  const void* bias;
  void* out;
};

// x[row][col .. col + 8), zero past K; rows past M read row M - 1 (their results are dropped)
template <bool VEC>
__device__ __forceinline__ v4i load_x(const GemmArgs& a, int64_t row, int64_t col) {
  const uint16_t* p = (const uint16_t*)a.x + row * a.x_s_row;
  if constexpr (VEC) {
    return col < a.k ? *(const v4i*)(p + col) : v4i{0, 0, 0, 0};
  } else {
    v4i r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = col + 2 * e < a.k ? p[col + 2 * e] : 0u, hi = col + 2 * e + 1 < a.k ? p[col + 2 * e + 1] : 0u;
      r[e] = (int)(lo | hi << 16);
    }
    return r;
  }
}

// 16 columns of the output and 16 MT rows a workgroup; its waves take the K tiles in turn and add their sums through LDS.
template <int DT, bool FP4, int GROUP, int MT, bool VEC>
__global__ __launch_bounds__(512) void w4_rows_kernel(GemmArgs a) {
  constexpr int PER = TK / GROUP, STEPS = GROUP / 32;
  extern __shared__ float part[];   // [waves][MT][256]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int64_t nt = blockIdx.x, m0 = (int64_t)blockIdx.y * 16 * MT;
  int64_t row[MT];
  v4f out[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    row[i] = min(m0 + 16 * i + r, a.m - 1);
    out[i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  const v4i ones = {(int)ONES<DT>, (int)ONES<DT>, (int)ONES<DT>, (int)ONES<DT>};
  for (int64_t t = wave; t < a.kt; t += waves) {
    const int64_t tile = nt * a.kt + t;
    const v4i w = *(const v4i*)(a.w4 + tile * TILE_BYTES + 16 * lane);
    float s[PER], z[PER];
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      s[g] = bf16_to_f32(a.scale[(tile * TN + r) * PER + g]);
      z[g] = !FP4 && a.zero ? (float)a.zero[(tile * TN + r) * PER + g] : 8.f;
    }
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      v4f acc[MT], sum[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = sum[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const int st = g * STEPS + j;
        const v4i b = operand<DT, FP4>((uint32_t)w[st]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const v4i x = load_x<VEC>(a, row[i], t * TK + 32 * st + 8 * q);
          acc[i] = mfma<DT>(x, b, acc[i]);
          if constexpr (!FP4) sum[i] = mfma<DT>(x, ones, sum[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (FP4) out[i][e] = fmaf(s[g], acc[i][e], out[i][e]);
          else out[i][e] = fmaf(16.f * s[g], acc[i][e], fmaf(-s[g] * (16.f + z[g]), sum[i][e], out[i][e]));
        }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[(wave * MT + i) * 256 + (4 * q + e) * 16 + r] = out[i][e];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += blockDim.x) {
    const int64_t m = m0 + (i >> 4), n = nt * TN + (i & 15);
    if (m >= a.m || n >= a.n) continue;
    float y = 0.f;
    for (int w = 0; w < waves; ++w) y += part[w * MT * 256 + i];
    if (a.bias) y += load1<DT>(a.bias, n);
    store1<DT>(a.out, m * a.n + n, y);
  }
}

template <int DT, bool FP4, int GROUP, int MT, bool VEC>
void launch_rows(const GemmArgs& a, hipStream_t stream) {
  const int waves = a.kt < 8 ? (int)a.kt : 8;
  const dim3 grid((unsigned)((a.n + TN - 1) / TN), (unsigned)((a.m + 16 * MT - 1) / (16 * MT)));
  w4_rows_kernel<DT, FP4, GROUP, MT, VEC><<<grid, 64 * waves, waves * MT * 256 * sizeof(float), stream>>>(a);
}

template <int DT, bool FP4, int GROUP>
void launch_group(const GemmArgs& a, bool vec, hipStream_t stream) {
  if (!vec) launch_rows<DT, FP4, GROUP, 2, false>(a, stream);
  else if (a.m <= 16) launch_rows<DT, FP4, GROUP, 1, true>(a, stream);
  else if (a.m <= 32) launch_rows<DT, FP4, GROUP, 2, true>(a, stream);
  else launch_rows<DT, FP4, GROUP, 4, true>(a, stream);
}

template <int DT, bool FP4>
void launch_format(const GemmArgs& a, int64_t group, bool vec, hipStream_t stream) {
  if (group == 32) launch_group<DT, FP4, 32>(a, vec, stream);
  else if (group == 64) launch_group<DT, FP4, 64>(a, vec, stream);
  else launch_group<DT, FP4, 128>(a, vec, stream);
}

bool sizes_ok(int64_t n, int64_t k, int fmt, int64_t group) {
  // (tiles along K and N are grid dimensions of at most 65535)
  return n >= 1 && k >= 1 && n <= (1 << 20) && k <= (1 << 20) && (fmt == LBW_W4_INT4 || fmt == LBW_W4_FP4) &&
         (group == 32 || group == 64 || group == 128);
}

}  // namespace
}  // namespace lbw

using namespace lbw;

extern "C" int lbw_quant_w4(const void* w, int w_is_fp32, int64_t n, int64_t k, int64_t s_row, int fmt, int64_t group,
                            uint8_t* w4, uint16_t* scale, uint8_t* zero, void* stream) {
  if (!w || !w4 || !scale) return LBW_E_NULL;
  if (!sizes_ok(n, k, fmt, group) || (zero && fmt == LBW_W4_FP4)) return LBW_E_SHAPE;
  if ((uintptr_t)w % (w_is_fp32 ? 4 : 2) || (uintptr_t)w4 % 16 || (uintptr_t)scale % 2) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const dim3 grid((unsigned)((k + TK - 1) / TK), (unsigned)((n + TN - 1) / TN));
  if (grid.y > 65535) return LBW_E_SHAPE;
  if (w_is_fp32) quant_w4_kernel<true><<<grid, 256, 0, (hipStream_t)stream>>>(w, n, k, s_row, fmt, (int)group, w4, scale, zero);
  else quant_w4_kernel<false><<<grid, 256, 0, (hipStream_t)stream>>>(w, n, k, s_row, fmt, (int)group, w4, scale, zero);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

extern "C" int lbw_gemm_w4(const void* x, int dtype, int64_t m, int64_t k, int64_t x_s_row, const uint8_t* w4,
                           const uint16_t* scale, const uint8_t* zero, int fmt, int64_t group, int64_t n,
                           const void* bias, void* out, void* stream) {
  if (!x || !w4 || !scale || !out) return LBW_E_NULL;
  if (!sizes_ok(n, k, fmt, group) || (zero && fmt == LBW_W4_FP4) || m < 1 || m > (1 << 20) ||
      (dtype != LBW_DTYPE_BF16 && dtype != LBW_DTYPE_FP16))
    return LBW_E_SHAPE;
  if ((uintptr_t)x % 2 || (uintptr_t)w4 % 16 || (uintptr_t)scale % 2 || (uintptr_t)bias % 2 || (uintptr_t)out % 2)
    return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const GemmArgs a = {x, m, k, x_s_row, w4, scale, zero, n, (k + TK - 1) / TK, bias, out};
  const bool vec = k % 8 == 0 && x_s_row % 8 == 0 && (uintptr_t)x % 16 == 0;
  const bool fp4 = fmt == LBW_W4_FP4, half = dtype == LBW_DTYPE_FP16;
  hipStream_t s = (hipStream_t)stream;
  if (half) fp4 ? launch_format<LBW_DTYPE_FP16, true>(a, group, vec, s) : launch_format<LBW_DTYPE_FP16, false>(a, group, vec, s);
  else fp4 ? launch_format<LBW_DTYPE_BF16, true>(a, group, vec, s) : launch_format<LBW_DTYPE_BF16, false>(a, group, vec, s);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
