// Linears with 4-bit weights (include/lbw_block.h): their quantisation, and x w^T with codes that become matrix-core
// operands in registers.
//
// A code enters the products exactly. fp4 converts by the hardware's own instruction. An integer code c becomes 1 + c
// / 16 in the 16-bit format: its four bits placed in the mantissa of 1, a shift and a mask for two codes (converting
// to the signed integer instead takes three more operations a pair). With v = c - z the group's sum is then
//   sum x v = 16 (sum x (1 + c / 16) - (1 + z / 16) sum x),
// sum x from one more matrix instruction a step (x times ones) whose result stands where the products' do. Group sums
// are scaled in fp32: out += s (...) for every group, so neither scale nor zero is ever rounded into a 16-bit weight.
#include "lbw_rows.h"

namespace lbw {
namespace {

constexpr int TN = 16, TK = 128;      // a tile of the stored weights
constexpr int TILE_BYTES = TN * TK / 2;
enum Form { INT4, INT4_ZEROS, FP4 };   // of the stored codes (the zeros' form apart: a load less, and no branch around it)

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- quantisation

template <int DPP>
__device__ __forceinline__ void dpp_max_min(float& hi, float& lo) {
  hi = fmaxf(hi, dpp<DPP>(hi));
  lo = fminf(lo, dpp<DPP>(lo));
}

// A workgroup makes one tile: 16 lanes a row, each 8 columns in a row; a group's extremes by DPP within its lanes. Runs
// once, at load, and reads value by value: 8960 x 1536 from bf16 in 18.6 us (1.9 TB/s), fp4 22.4, from fp32 27.
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

// Those in a vector register: mask and ones then enter one instruction (which takes a single scalar or literal), not
// two. With the factor of 16 left to the end a K tile takes 357 vector instructions beside its 68 products, not 437
// (2048 x 8192 x 6144 with zeros: 238 -> 229 us).
template <int DT>
__device__ __forceinline__ uint32_t vector_ones() {
  uint32_t r;
  asm("v_mov_b32 %0, %1" : "=v"(r) : "i"(ONES<DT>));
  return r;
}

// The 8 codes of a word as 16-bit operands: integer codes as 1 + c / 16, fp4 codes as their values.
template <int DT, Form F>
__device__ __forceinline__ v4i operand(uint32_t w, uint32_t ones) {
  v4i r;
  if constexpr (F == FP4) {
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
    for (int t = 0; t < 4; ++t) r[t] = (int)(((4 * t < S ? w << (S - 4 * t) : w >> (4 * t - S)) & M) | ones);
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
  bool bias_fp32;
  void* out;
};

// x from row m0 on, read 8 columns at a time. VEC: by buffer loads, a base for the workgroup and 32 bits of offset a
// lane (64-bit addresses of 16 rows took 32 registers, spills, and more clocks than the products); what lies past the
// last row or past K reads as zero by the buffer's bounds. Else value by value. Zero past K is needed: the tiles hold
// anything there.
template <bool VEC>
struct RowsOfX {
  __amdgpu_buffer_rsrc_t rsrc;
  const uint16_t* p;
  int64_t rows, k, stride;
  __device__ __forceinline__ RowsOfX(const GemmArgs& a, int64_t m0) {
    rows = a.m - m0;
    k = a.k;
    stride = a.x_s_row;
    p = (const uint16_t*)a.x + m0 * stride;
    // (a workgroup reads 64 rows at most: 2^30 bytes)
    const int64_t bytes = 2 * ((min(rows, (int64_t)64) - 1) * stride + k);
    if constexpr (VEC) rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)(uint32_t)bytes, 0x00020000);
  }
  // the offset of a lane that reads from row `row`: what load takes, with its column
  __device__ __forceinline__ uint32_t offset(int row) const { return (uint32_t)(row * stride) * 2u; }
  __device__ __forceinline__ v4i load(int row, uint32_t off, int64_t col) const {
    if constexpr (VEC) {
      const uint32_t at = col < k ? off + 2u * (uint32_t)col : 0xFFFFFFF0u;
      return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, 0));
    } else {
      v4i r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = row < rows;
        const uint32_t lo = in && col + 2 * e < k ? p[row * stride + col + 2 * e] : 0u;
        const uint32_t hi = in && col + 2 * e + 1 < k ? p[row * stride + col + 2 * e + 1] : 0u;
        r[e] = (int)(lo | hi << 16);
      }
      return r;
    }
  }
};

// The bias of four columns of the output from n on in each of N tiles, from its own format (the output's, or fp32): one
// branch for all, and none around a load (past the last column the last is read again), so that they are in flight
// together. The fp32 form stands out of the way: in line it cost the 16-bit one 1 % (61 x 8960 x 1536 9.70 -> 9.80 us).
template <int DT, int N>
struct Bias {
  v4f tile[N];
  __device__ __forceinline__ Bias(const GemmArgs& a, int64_t n) {
#pragma unroll
    for (int t = 0; t < N; ++t) tile[t] = v4f{0.f, 0.f, 0.f, 0.f};
    if (!a.bias) return;
    if (__builtin_expect(a.bias_fp32, 0)) load<LBW_DTYPE_FP32>(a, n);
    else load<DT>(a, n);
  }
  template <int BT>
  __device__ __forceinline__ void load(const GemmArgs& a, int64_t n) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[t][e] = load1<BT>(a.bias, min(n + TN * t + e, a.n - 1));
  }
};

// Sums of four columns with their bias. Integer codes were taken as sixteenths.
template <Form F>
__device__ __forceinline__ v4f finished(v4f y, v4f bias) {
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = fmaf(F == FP4 ? 1.f : 16.f, y[e], bias[e]);
  return y;
}

// Four columns of the output from n on (a multiple of 4), 8 bytes at once where the output's rows allow it.
template <int DT, Form F>
__device__ __forceinline__ void store_out(const GemmArgs& a, int64_t m, int64_t n, v4f y, v4f bias) {
  y = finished<F>(y, bias);
  if (a.n % 4 == 0) {
    *(v2i*)((uint16_t*)a.out + m * a.n + n) = v2i{(int)pack2<DT>(y[0], y[1]), (int)pack2<DT>(y[2], y[3])};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.n) store1<DT>(a.out, m * a.n + n + e, y[e]);
  }
}

// The scales (bf16) and zeros of a tile's rows 4 q .. 4 q + 3, the ones whose products a lane holds: 4 PER of each.
template <Form F, int PER>
struct Scales {
  uint32_t s[2 * PER], z[PER];
  template <int N>
  static __device__ __forceinline__ void words(uint32_t* to, const void* p) {
    if constexpr (N == 1) {
      to[0] = *(const uint32_t*)p;
    } else if constexpr (N == 2) {
      const uint2 v = *(const uint2*)p;
      to[0] = v.x;
      to[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint4 v = ((const uint4*)p)[i / 4];
        to[i] = v.x;
        to[i + 1] = v.y;
        to[i + 2] = v.z;
        to[i + 3] = v.w;
      }
    }
  }
  // row: 16 times the tile's number and 4 q
  __device__ __forceinline__ void load(const uint16_t* scale, const uint8_t* zero, int64_t row) {
    words<2 * PER>(s, scale + PER * row);
    if constexpr (F == INT4_ZEROS) words<PER>(z, zero + PER * row);
  }
  // what the sums of group g are multiplied by
  __device__ __forceinline__ v4f scale_of(int g) const {
    v4f r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = PER * e + g;
      r[e] = __uint_as_float(i & 1 ? s[i >> 1] & 0xFFFF0000u : s[i >> 1] << 16);
    }
    return r;
  }
  // where they start, from the sum of x: the codes' offset -(16 + z) / 16 comes off (for z = 8 it has already been
  // multiplied in, once for all columns)
  __device__ __forceinline__ v4f start(int g, float sum) const {
    v4f r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = PER * e + g;
      r[e] = F == INT4_ZEROS ? sum * (-1.f - 0.0625f * (float)(z[i >> 2] >> 8 * (i & 3) & 0xFFu)) : sum;
    }
    return r;
  }
};

// The sum of each of 16 rows of x over a group, from its operands (ones times them: every row of the result is the
// sums), as Scales::start takes it.
template <int DT, Form F, int STEPS>
__device__ __forceinline__ float group_sum(const v4i* x) {
  if constexpr (F == FP4) return 0.f;
  v4f sum = {0.f, 0.f, 0.f, 0.f};
  const v4i ones = {(int)ONES<DT>, (int)ONES<DT>, (int)ONES<DT>, (int)ONES<DT>};
#pragma unroll
  for (int j = 0; j < STEPS; ++j) sum = mfma<DT>(ones, x[j], sum);
  return F == INT4 ? -1.5f * sum[0] : sum[0];
}

// Both kernels multiply weights by x transposed: a lane then holds 4 neighbouring columns of a row of the output,
// which it stores at once, and one sum of x for them.

// Few rows: 16 MT rows and 16 NT columns a workgroup. Its waves share out the K tiles (so that the few workgroups of
// a narrow output still have loads in flight on every SIMD) and add their sums through LDS at the end. x comes in
// rows of 256 bytes, four a load, and is turned into operands through LDS, each wave in a part of its own (no
// barrier): loads in the operands' own order, 16 rows of 64 bytes each, took 120 clocks apiece, all rows in one bank
// of the cache's tags. A row's 16-byte pieces are exchanged by its number, so that 16 rows' pieces lie in all banks.
// The next tile's x and codes are in flight while a tile is multiplied. Latency bounds it: 5 x 1536 x 8960 in fp4 6.8
// us, 61 x 8960 x 1536 in int4 with zeros 9.7, one row x 9216 x 1536 5.0, where the weights' bytes take 1.4 to 1.7.
template <int DT, Form F, int GROUP, int MT, int NT, int MOST, bool VEC>
__global__ __launch_bounds__(64 * MOST) void w4_rows_kernel(GemmArgs a) {
  constexpr int PER = TK / GROUP, STEPS = GROUP / 32, ROWS = 16 * MT, COLS = TN * NT;
  extern __shared__ __align__(16) char lds[];   // x: [waves][ROWS][256]; afterwards the sums: [waves][ROWS][COLS] fp32
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * ROWS, nt0 = (int64_t)blockIdx.y * NT, nts = (a.n + TN - 1) / TN;
  char* mine = lds + wave * (ROWS * 256);
  const RowsOfX<VEC> rows(a, m0);
  const uint32_t off0 = rows.offset(q), four = rows.offset(4);
  int64_t tile[NT];
  v4f out[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    tile[n] = min(nt0 + n, nts - 1) * a.kt;   // (a tile past the last: read the last again, its results are dropped)
#pragma unroll
    for (int i = 0; i < MT; ++i) out[n][i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t one = vector_ones<DT>();
  v4i w[NT], x[4 * MT];
  Scales<F, PER> sc[NT];
  const auto load = [&](int64_t t) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      w[n] = *(const v4i*)(a.w4 + (tile[n] + t) * TILE_BYTES + 16 * lane);
      sc[n].load(a.scale, a.zero, (tile[n] + t) * TN + 4 * q);
    }
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i) x[i] = rows.load(4 * i + q, off0 + i * four, t * TK + 8 * r);   // row 4 i + q
  };
  load(wave);   // (there are no more waves than tiles)
  for (int64_t t = wave; t < a.kt; t += waves) {
#pragma unroll
    for (int i = 0; i < 4 * MT; ++i)
      *(v4i*)(mine + (4 * i + q) * 256 + ((r ^ (4 * i + q) & 15) << 4)) = x[i];
    v4i wc[NT];
    Scales<F, PER> cc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      wc[n] = w[n];
      cc[n] = sc[n];
    }
    __builtin_amdgcn_wave_barrier();
    if (t + waves < a.kt) load(t + waves);
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      v4i xo[MT][STEPS];
      float sum[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < STEPS; ++j)
          xo[i][j] = *(const v4i*)(mine + (16 * i + r) * 256 + (((4 * (g * STEPS + j) + q) ^ r) << 4));
        sum[i] = group_sum<DT, F, STEPS>(xo[i]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const v4f s = cc[n].scale_of(g);
        v4f acc[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = cc[n].start(g, sum[i]);
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          const v4i b = operand<DT, F>((uint32_t)wc[n][g * STEPS + j], one);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i] = mfma<DT>(b, xo[i][j], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[n][i][e] = fmaf(s[e], acc[i][e], out[n][i][e]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();   // every wave has read its x
  float* part = (float*)lds;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i) *(v4f*)(part + (wave * ROWS + 16 * i + r) * COLS + TN * n + 4 * q) = out[n][i];
  __syncthreads();
  for (int i = 4 * threadIdx.x; i < ROWS * COLS; i += 4 * blockDim.x) {
    const int64_t m = m0 + i / COLS, n = nt0 * TN + i % COLS;
    if (m >= a.m || n >= a.n) continue;
    v4f y = *(const v4f*)(part + i);
    for (int w = 1; w < waves; ++w) y += *(const v4f*)(part + w * (ROWS * COLS) + i);
    store_out<DT, F>(a, m, n, y, Bias<DT, 1>(a, n).tile[0]);
  }
}

// Many rows: 64 rows x 256 columns a workgroup, four waves of 64 x 64, two workgroups a CU, which drift apart, so
// that one's matrix work runs under the other's conversions (eight such waves in step on 128 rows took 62.7 us where
// this took 57.5, before the steps that made it 51). With a bias, groups of 128, bf16, int4 / int4 with zeros / fp4:
//   1508 x 8960 x 1536    51.1 us (813 TFLOP/s) / 56.6 (733) / 47.2 (879); 64 columns a group with zeros 66.9
//   2048 x 8192 x 6144   195.2   (1056)         / 216.0 (954) / 184.2 (1119); the grid fills whole rounds
// x passes through LDS, a K tile at a time in two buffers (rows and pieces as above): wave w
// loads rows 16 w .. 16 w + 15 in the operands' own order, forms their sums over each group while they are in
// registers, and leaves both there. Codes go from memory to registers, a tile ahead. The output leaves through LDS,
// so that a store holds whole rows of 128 bytes (1508 x 8960 x 1536, zeros and bias, at that step: 68.1 -> 64.9 us;
// with no store at all 61.2). The conversions bound it: each wave makes its columns' operands for its own 64 rows, and
// vector instructions take about 1.3 times the matrix core's cycles, which two waves a SIMD overlap in part.
constexpr int GM = 64, GN = 256;
constexpr int X_TILE = GM * TK * 2;   // bytes

template <int DT, Form F, int GROUP>
__global__ __launch_bounds__(256, 2) void w4_gemm_kernel(GemmArgs a, int m_tiles) {
  constexpr int PER = TK / GROUP, STEPS = GROUP / 32;
  __shared__ __align__(16) char xs[2][X_TILE];   // (afterwards the output, GM * 128 bytes a wave)
  __shared__ float sums[2][PER][GM];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = lane & 15, q = lane >> 4;
  // an XCD takes workgroups that follow each other down the rows: they read the same weights
  const int total = gridDim.x, per_xcd = (total + 7) / 8;
  const int id = (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  if (id >= m_tiles * (int)((a.n + GN - 1) / GN)) return;
  const int64_t m0 = (int64_t)(id % m_tiles) * GM, nt0 = (int64_t)(id / m_tiles) * (GN / TN) + 4 * wave;
  const int64_t nts = (a.n + TN - 1) / TN;
  const RowsOfX<true> rows(a, m0);
  const uint32_t off = rows.offset(16 * wave + r);
  int64_t tile[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) tile[n] = min(nt0 + n, nts - 1) * a.kt;
  v4f out[4][4];
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) out[n][i] = v4f{0.f, 0.f, 0.f, 0.f};

  const uint32_t one = vector_ones<DT>();
  v4i xr[4], w[4];
  Scales<F, PER> sc[4];
  const auto load = [&](int64_t t) {
#pragma unroll
    for (int st = 0; st < 4; ++st) xr[st] = rows.load(16 * wave + r, off, t * TK + 32 * st + 8 * q);
  };
  const auto load_w = [&](int n, int64_t t) {
    w[n] = *(const v4i*)(a.w4 + (tile[n] + t) * TILE_BYTES + 16 * lane);
    sc[n].load(a.scale, a.zero, (tile[n] + t) * TN + 4 * q);
  };
  // this wave's 16 rows of x and their sums into buffer `to` (the four quarters of a wave hold the same sums)
  const auto leave = [&](int to) {
#pragma unroll
    for (int st = 0; st < 4; ++st)
      *(v4i*)(xs[to] + (16 * wave + r) * 256 + (((4 * st + q) ^ r) << 4)) = xr[st];
    if constexpr (F != FP4) {
#pragma unroll
      for (int g = 0; g < PER; ++g) sums[to][g][16 * wave + r] = group_sum<DT, F, STEPS>(&xr[g * STEPS]);
    }
  };
  load(0);
#pragma unroll
  for (int n = 0; n < 4; ++n) load_w(n, 0);
  leave(0);
  __syncthreads();
  for (int64_t t = 0; t < a.kt; ++t) {
    const int buf = (int)(t & 1);
    const int64_t next = min(t + 1, a.kt - 1);   // (the last tile again at the end: no branch in the loop)
#pragma unroll
    for (int g = 0; g < PER; ++g) {
      v4i x[4][STEPS];
      float sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < STEPS; ++j)
          x[i][j] = *(const v4i*)(xs[buf] + (16 * i + r) * 256 + (((4 * (g * STEPS + j) + q) ^ r) << 4));
        sum[i] = F == FP4 ? 0.f : sums[buf][g][16 * i + r];
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const v4f s = sc[n].scale_of(g);
        v4f acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = sc[n].start(g, sum[i]);
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          const v4i b = operand<DT, F>((uint32_t)w[n][g * STEPS + j], one);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = mfma<DT>(b, x[i][j], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[n][i][e] = fmaf(s[e], acc[i][e], out[n][i][e]);
        if (g == PER - 1) load_w(n, next);   // into the registers just read: no second set
        if (g == 0 && n == 0) {
          // (not earlier, for its registers; and held here: the scheduler moves the loads down to where they are
          // waited for)
          __builtin_amdgcn_sched_barrier(0);
          load(next);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);     // (or the groups' operands are all loaded at once, and spilled)
    }
    // the other buffer was last read before the barrier that ended the previous tile
    leave(buf ^ 1);
    __syncthreads();
  }
  const int64_t col0 = nt0 * TN + 4 * q;
  const Bias<DT, 4> bias(a, col0);
  if (a.n % 8 == 0 && (uintptr_t)a.out % 16 == 0) {
    char* mine = xs[0] + wave * (GM * 128);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const v4f y = finished<F>(out[n][i], bias.tile[n]);
        *(v2i*)(mine + (16 * i + r) * 128 + (((2 * n + (q >> 1)) ^ (r & 7)) << 4) + 8 * (q & 1)) =
            v2i{(int)pack2<DT>(y[0], y[1]), (int)pack2<DT>(y[2], y[3])};
      }
    __builtin_amdgcn_wave_barrier();
    const int piece = lane & 7;
    const int64_t col = nt0 * TN + 8 * piece;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 8 * i + (lane >> 3);
      const v4i y = *(const v4i*)(mine + row * 128 + ((piece ^ (row & 7)) << 4));
      if (m0 + row < a.m && col < a.n) *(v4i*)((uint16_t*)a.out + (m0 + row) * a.n + col) = y;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 16 * i + r;
    if (m >= a.m) continue;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t col = col0 + n * TN;
      if (col < a.n) store_out<DT, F>(a, m, col, out[n][i], bias.tile[n]);
    }
  }
}

// `most` (at most MOST) waves
template <int DT, Form F, int GROUP, int MT, int NT, int MOST, bool VEC>
void launch_rows(const GemmArgs& a, int most, hipStream_t stream) {
  // the fewest rounds of K tiles that `most` waves allow, in as few waves
  const int64_t rounds = (a.kt + most - 1) / most;
  const int waves = (int)((a.kt + rounds - 1) / rounds);
  const dim3 grid((unsigned)((a.m + 16 * MT - 1) / (16 * MT)), (unsigned)((a.n + TN * NT - 1) / (TN * NT)));
  const int each = MT * (NT > 4 ? NT : 4) * 1024;   // bytes of LDS a wave needs
  w4_rows_kernel<DT, F, GROUP, MT, NT, MOST, VEC><<<grid, 64 * waves, waves * each, stream>>>(a);
}

// Which kernel. Few rows are a matter of latency: the smallest tile whose workgroups all run at once, one a CU, since
// a second round costs more than a larger tile, and a larger tile more than a part of the first round left empty
// (bf16, groups of 128, int4 / groups of 64, int4 with zeros; rows x columns x K, us in graphs):
//                        16 x 16 tiles   16 x 32         16 x 48         32 x 48
//   24 x  1536 x 8960     6.9 /  7.8      9.4 / 11.6     11.3 / 14.8     17.0 / 21.0
//   77 x  1536 x 1536     4.5 /  4.9      4.3 /  4.8      4.8 /  5.7      5.9 /  6.8
//    1 x  9216 x 1536     5.3 /  5.9      5.6 /  6.5      4.7 /  5.6      5.9 /  6.8
//   32 x  8960 x 1536     7.8 /  8.5      7.9 /  9.1      7.1 /  9.6      6.1 /  7.0
//    5 x 20480 x 8960    29.9 / 32.9     23.3 / 28.6     21.7 / 28.7     27.3 / 34.0
// (the last: up to 16 rows never fill two row blocks). A CU with a single 16 x 16 tile has 12 waves, against 8 (5 x
// 1536 x 8960: fp4 7.15 -> 7.05, int4 with zeros 7.95 -> 7.55; 16 waves 7.45 and 7.9). With 32 x 48 tiles past one
// round two workgroups of four waves share a CU better than one of six (512 x 1536 x 8960: 28.6 against 34.4). Whole
// tiles of 64 x 256 win from about half a tile a CU on: 256 x 8960 x 1536 (140 tiles) 18.0 against 20.9, 1508 x 1536
// x 1536 (144) 17.8 against 19.8, 512 x 8960 x 1536 (280) 26.3 against 36.5, about even for 1508 x 1536 x 8960 (144)
// 84 against 81; but 1024 x 1536 x 1536 (96) 17.4 against 14.5, and half empty ones never: 32 x 40960 x 1536 (160)
// 17.5 against 15.4.
template <int DT, Form F, int GROUP>
void launch_group(const GemmArgs& a, bool vec, hipStream_t stream) {
  const auto grid = [&](int rows, int cols) { return ((a.m + rows - 1) / rows) * ((a.n + cols - 1) / cols); };
  constexpr int CUS = 256;
  if (!vec) launch_rows<DT, F, GROUP, 2, 1, 8, false>(a, 8, stream);
  else if (grid(16, 16) <= CUS) launch_rows<DT, F, GROUP, 1, 1, 12, true>(a, 12, stream);
  else if (grid(16, 32) <= CUS) launch_rows<DT, F, GROUP, 1, 2, 8, true>(a, 8, stream);
  else if (grid(16, 48) <= CUS) launch_rows<DT, F, GROUP, 1, 3, 8, true>(a, 8, stream);
  else if (a.m <= 16) launch_rows<DT, F, GROUP, 1, 2, 8, true>(a, 8, stream);
  else if (a.m <= 32 || grid(GM, GN) < CUS / 2)
    launch_rows<DT, F, GROUP, 2, 3, 6, true>(a, grid(32, 48) <= CUS ? 6 : 4, stream);
  else w4_gemm_kernel<DT, F, GROUP><<<(unsigned)((grid(GM, GN) + 7) / 8 * 8), 4 * GM, 0, stream>>>(a, (int)grid(GM, 1 << 30));
}

template <int DT, Form F>
void launch_format(const GemmArgs& a, int64_t group, bool vec, hipStream_t stream) {
  if (group == 32) launch_group<DT, F, 32>(a, vec, stream);
  else if (group == 64) launch_group<DT, F, 64>(a, vec, stream);
  else launch_group<DT, F, 128>(a, vec, stream);
}

constexpr int64_t MAX_N = 65535 * TN;   // (column tiles are a second grid dimension)

bool sizes_ok(int64_t n, int64_t k, int fmt, int64_t group) {
  return n >= 1 && k >= 1 && n <= MAX_N && k <= (1 << 20) && (fmt == LBW_W4_INT4 || fmt == LBW_W4_FP4) &&
         (group == 32 || group == 64 || group == 128);
}

}  // namespace
}  // namespace lbw

using namespace lbw;

extern "C" int lbw_quant_w4(const void* w, int w_is_fp32, int64_t n, int64_t k, int64_t s_row, int fmt, int64_t group,
                            uint8_t* w4, uint16_t* scale, uint8_t* zero, void* stream) {
  if (!w || !w4 || !scale) return LBW_E_NULL;
  if (!sizes_ok(n, k, fmt, group) || (zero && fmt == LBW_W4_FP4)) return LBW_E_SHAPE;
  if ((uintptr_t)w % (w_is_fp32 ? 4 : 2) || (uintptr_t)w4 % 16 || (uintptr_t)scale % 16 || (uintptr_t)zero % 16)
    return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const dim3 grid((unsigned)((k + TK - 1) / TK), (unsigned)((n + TN - 1) / TN));
  if (w_is_fp32) quant_w4_kernel<true><<<grid, 256, 0, (hipStream_t)stream>>>(w, n, k, s_row, fmt, (int)group, w4, scale, zero);
  else quant_w4_kernel<false><<<grid, 256, 0, (hipStream_t)stream>>>(w, n, k, s_row, fmt, (int)group, w4, scale, zero);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

extern "C" int lbw_gemm_w4(const void* x, int dtype, int64_t m, int64_t k, int64_t x_s_row, const uint8_t* w4,
                           const uint16_t* scale, const uint8_t* zero, int fmt, int64_t group, int64_t n,
                           const void* bias, void* out, void* stream) {
  if (!x || !w4 || !scale || !out) return LBW_E_NULL;
  const bool bias_fp32 = (dtype & LBW_W4_BIAS_FP32) != 0;
  dtype &= ~LBW_W4_BIAS_FP32;
  if (!sizes_ok(n, k, fmt, group) || (zero && fmt == LBW_W4_FP4) || m < 1 || m > (1 << 24) ||
      (dtype != LBW_DTYPE_BF16 && dtype != LBW_DTYPE_FP16))
    return LBW_E_SHAPE;
  if ((uintptr_t)x % 2 || (uintptr_t)w4 % 16 || (uintptr_t)scale % 16 || (uintptr_t)zero % 16 ||
      (uintptr_t)bias % (bias_fp32 ? 4 : 2) || (uintptr_t)out % 8)
    return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const GemmArgs a = {x, m, k, x_s_row, w4, scale, zero, n, (k + TK - 1) / TK, bias, bias_fp32, out};
  // (a workgroup's rows have to lie within the 32 bits of a buffer's offsets)
  const bool vec = k % 8 == 0 && x_s_row % 8 == 0 && x_s_row >= 0 && x_s_row < (1 << 23) && (uintptr_t)x % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  const auto by_form = [&](auto dt) {
    if (fmt == LBW_W4_FP4) launch_format<dt.value, FP4>(a, group, vec, s);
    else if (zero) launch_format<dt.value, INT4_ZEROS>(a, group, vec, s);
    else launch_format<dt.value, INT4>(a, group, vec, s);
  };
  if (dtype == LBW_DTYPE_FP16) by_form(std::integral_constant<int, LBW_DTYPE_FP16>{});
  else by_form(std::integral_constant<int, LBW_DTYPE_BF16>{});
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
