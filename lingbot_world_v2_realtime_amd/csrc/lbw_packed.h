// What the kernels of packed attention share: the sequences of a call found from their starts, tiles of rows in LDS,
// and the fragments of matrix products read from them.
//
// A tile is rows of DH 16-bit channels as they lie in memory, brought in by buffer loads that write to LDS (rows past a
// sequence's end are outside the resource and come in as zeros, so no neighbour's value, however odd, meets a weight of
// zero). A 16-byte piece c of row r lies at piece c ^ swizzle(r): 16 rows of one piece cover all banks, and so do 4 rows
// of 4 neighbouring pieces, so that the rows are read without conflicts as they are (16 bytes a lane, 8 channels of a
// row) and turned (ds_read_b64_tr_b16: 4 rows of 16 channels for 16 lanes, a lane receiving one channel of the 4 rows).
#pragma once

#include <type_traits>

#include "lbw_spans.h"

namespace lbw {
namespace packed {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;

template <int N>
using ic = std::integral_constant<int, N>;

// Stands in a branch that a whole wave takes or not: the compiler would take both sides and select, for every tile what the
// last ones need.
__device__ __forceinline__ void branch_here() { asm volatile(""); }

template <bool F16>
__device__ __forceinline__ v16f mfma(const v4i a, const v4i b, const v16f c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(hf8, a), __builtin_bit_cast(hf8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack(float a, float b) { return pack2<F16 ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16>(a, b); }

// The weights of a softmax are 1 at most. fp16 holds them times 2^LIFT, so that those below 2^-14 of the largest, of which
// a long row has many, are not held in fewer bits yet; the sum of the row has the same factor.
template <bool F16>
constexpr float LIFT = F16 ? 10.f : 0.f;

__device__ __forceinline__ v16f zeros16() {
  v16f z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

__device__ __forceinline__ float sum_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The head and tile of a workgroup, numbered so that one XCD (a workgroup's number mod 8) has as few heads of k and v as it
// can: with c the greatest common divisor of those heads and 8, XCD x takes the heads x mod c, + c, .. and every (8 / c)-th
// tile of theirs, the heads of q that share one behind each other.
inline uint32_t xcd_common(int64_t k_heads) { return k_heads % 8 == 0 ? 8 : k_heads % 4 == 0 ? 4 : k_heads % 2 == 0 ? 2 : 1; }
inline int64_t xcd_groups(int64_t tiles, int64_t k_heads, int64_t group) {
  const int64_t c = xcd_common(k_heads), each = 8 / c;
  return (tiles + each - 1) / each * (k_heads / c) * group * 8;
}
__device__ __forceinline__ void head_tile(uint32_t id, uint32_t k_heads, uint32_t group, uint32_t common, uint32_t& head, uint32_t& tile) {
  const uint32_t x = id & 7, r = id >> 3, per = k_heads / common, rest = r / group, g = r - rest * group;
  const uint32_t t = rest / per, j = rest - t * per;
  head = (x % common + common * j) * group + g;
  tile = t * (8 / common) + x / common;
}

template <int DH>
constexpr int row_bytes = 2 * DH;

template <int DH>
__device__ __forceinline__ int swizzle(int r) {
  if constexpr (DH == 128) return (r & 3) << 2 | (r >> 2 & 3);
  else return (r >> 1 & 1) << 2 | (r >> 2 & 3);   // (two rows share 256 bytes)
}

// 16 bytes a lane from the buffer `rs` at byte off[i] to LDS at dst + 1024 i + 16 lane. Inline asm, for the builtin is taken to
// touch any LDS, so that every LDS wait would wait for it too; it has no result register. One block for all of a wave's
// loads: m0, which says where they go, is the compiler's before and after.
template <int N>
__device__ __forceinline__ void dma16(const v4i rs, const uint32_t (&off)[N], uint8_t* lds) {
  static_assert(N == 2 || N == 4 || N == 8, "loads of a wave");
  uint32_t keep;
  const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)lds);
#define LBW_NEXT "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
#define LBW_LOAD(i) "buffer_load_dwordx4 %" #i ", %1, 0 offen lds\n\t"
  if constexpr (N == 2) {
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t" LBW_LOAD(3) LBW_NEXT LBW_LOAD(4) "s_mov_b32 m0, %0"
                 : "=&s"(keep) : "s"(rs), "s"(dst), "v"(off[0]), "v"(off[1]) : "memory", "scc");
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t" LBW_LOAD(3) LBW_NEXT LBW_LOAD(4) LBW_NEXT LBW_LOAD(5)
                   LBW_NEXT LBW_LOAD(6) "s_mov_b32 m0, %0"
                   : "=&s"(keep)
                   : "s"(rs), "s"(dst + i * 1024), "v"(off[i]), "v"(off[i + 1]), "v"(off[i + 2]), "v"(off[i + 3])
                   : "memory", "scc");
  }
#undef LBW_NEXT
#undef LBW_LOAD
}
__device__ __forceinline__ void wait_dma() { __builtin_amdgcn_s_waitcnt(0x0F70); }   // vmcnt(0) alone
// Until all but the last `ahead` (0 .. 2) tiles' loads are done, of PER loads each (memory reads return in order).
template <int PER>
__device__ __forceinline__ void wait_dma_but(int ahead) {
  constexpr auto imm = [](int n) { return 0x0F70 | (n & 15) | (n >> 4) << 14; };
  static_assert(2 * PER < 64, "vmcnt counts to 63");
  if (ahead >= 2) __builtin_amdgcn_s_waitcnt(imm(2 * PER));
  else if (ahead == 1) __builtin_amdgcn_s_waitcnt(imm(PER));
  else __builtin_amdgcn_s_waitcnt(imm(0));
}

// Rows of a tensor's head from `base` on, a row every `stride` elements, `left` of them: the resource of one tile of R rows
// ends with the last row that there is.
template <int DH>
__device__ __forceinline__ v4i rows_buffer(const uint16_t* base, int64_t stride, int left, int R) {
  const int n = min(left, R);
  const uint64_t a = (uint64_t)base;
  const uint32_t bytes = n > 0 ? (uint32_t)(n - 1) * (uint32_t)stride * 2 + row_bytes<DH> : 0;
  return v4i{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(a >> 32 & 0xFFFF)),
             __builtin_amdgcn_readfirstlane((int)bytes), 0x00027000};
}

// A tile of R rows by W waves: piece i of a wave is 1 KB of the tile. Byte offsets of a lane's piece in memory.
template <int DH, int R, int W>
struct Loader {
  static constexpr int PER = 1024 / row_bytes<DH>;   // rows of 1 KB
  static constexpr int N = R / PER / W;              // pieces of a wave
  static_assert(N * PER * W == R, "whole pieces");
  uint32_t off[N];
  __device__ __forceinline__ void init(int w, int lane, int64_t stride) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (w * N + i) * PER + lane * 16 / row_bytes<DH>, p = lane & (row_bytes<DH> / 16 - 1);
      off[i] = (uint32_t)r * (uint32_t)stride * 2 + ((p ^ swizzle<DH>(r)) << 4);
    }
  }
  __device__ __forceinline__ void issue(const v4i rs, int w, uint8_t* lds) const {
    dma16<N>(rs, off, lds + w * N * 1024);
  }
};

// Where a lane reads its part of 32 rows x 16 channels (rows as they are: 8 channels of row lane & 31): piece 2 st +
// (lane >> 5) for the 16 channels from 16 st on. Further 32 rows follow at 32 row_bytes.
template <int DH>
struct RowReads {
  int at[DH / 16];
  __device__ __forceinline__ void init(int lane) {
    const int r = lane & 31, hf = lane >> 5;
#pragma unroll
    for (int st = 0; st < DH / 16; ++st) at[st] = r * row_bytes<DH> + (((2 * st + hf) ^ swizzle<DH>(r)) << 4);
  }
  __device__ __forceinline__ v4i get(const uint8_t* tile, int rows32, int st) const {
    return *(const v4i*)(tile + rows32 * 32 * row_bytes<DH> + at[st]);
  }
};

// The same rows turned: lane l receives channel 32 mt + (l & 31) of the 8 rows 16 u + 4 (l >> 5) + {0 .. 3, 8 .. 11}, the
// order in which a lane holds the rows of a 32 x 32 product's result (its column being l & 31).
template <int DH>
struct TurnedReads {
  int at[DH / 32][2];
  __device__ __forceinline__ void init(int lane) {
    const int l = lane & 15, b = lane >> 4 & 1, hf = lane >> 5;
#pragma unroll
    for (int mt = 0; mt < DH / 32; ++mt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * x + 4 * hf + (l >> 2), c = 4 * mt + 2 * b + (l >> 1 & 1);
        at[mt][x] = r * row_bytes<DH> + ((c ^ swizzle<DH>(r)) << 4) + ((l & 1) << 3);
      }
  }
  __device__ __forceinline__ v4i get(const uint8_t* tile, int u, int mt) const {
    typedef __attribute__((address_space(3))) s4 lds4;
    const uint8_t* p = tile + u * 16 * row_bytes<DH>;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + at[mt][0]));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + at[mt][1]));
    const int2 a = __builtin_bit_cast(int2, lo), c = __builtin_bit_cast(int2, hi);
    return v4i{a.x, a.y, c.x, c.y};
  }
};

// An infinity or NaN of a row that a column does not see must not reach it, but its weight of zero times either is NaN. So a
// workgroup whose sums are not finite at its end (and whose columns do not all see the same) goes over its tiles once more,
// and where a tile is partly seen takes such values out of the products (clean) and adds them, as they are, to the sums of
// the columns that see them (add_odd). No other call pays for it, but for the look at the sums.
__device__ __forceinline__ bool is_odd(float x) { return !(fabsf(x) < INFINITY); }
template <int MT>
__device__ __forceinline__ bool any_odd(const v16f (&o)[MT]) {
  float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i & 3] = fmaf(o[mt][i], 0.f, z[i & 3]);
  return __any(is_odd((z[0] + z[1]) + (z[2] + z[3])));
}
template <bool F16>
__device__ __forceinline__ v4i clean(v4i f) {
  constexpr uint32_t e = F16 ? 0x7C00 : 0x7F80;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = f[i];
    f[i] = (w & e) == e ? w & 0xFFFF0000u : w;
    f[i] = (w >> 16 & e) == e ? f[i] & 0xFFFF : f[i];
  }
  return f;
}
// Rows 32 x .. + 32 of a tile; sees(j): whether the lane's column sees row j of them. NAN_ALL: NaN for each such value, where
// its weight can be zero, or NaN, but nothing else.
template <int DH, bool F16, bool NAN_ALL = false, class Sees>
__device__ __forceinline__ void add_odd(v16f (&o)[DH / 32], const uint8_t* tile, int x, int hf, const Sees& sees) {
#pragma unroll 1
  for (int j = 0; j < 32; ++j) {
    const uint8_t* row = tile + (32 * x + j) * row_bytes<DH>;
    const bool s = sees(j);
#pragma unroll
    for (int mt = 0; mt < DH / 32; ++mt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint2 w = *(const uint2*)(row + (((4 * mt + c) ^ swizzle<DH>(j)) << 4) + 8 * hf);
        const float v[4] = {lo16<F16>(w.x), hi16<F16>(w.x), lo16<F16>(w.y), hi16<F16>(w.y)};
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][4 * c + e] += s && is_odd(v[e]) ? (NAN_ALL ? __builtin_nanf("") : v[e]) : 0.f;
        __builtin_amdgcn_sched_barrier(0);   // (few registers rather than speed)
      }
  }
}

// 32 rows of one wave straight into the lanes that a product's other operand wants them in: lane l, piece st holds the
// channels 16 st + 8 (l >> 5) .. + 8 of row l & 31; rows that are not there are zero.
template <int DH>
__device__ __forceinline__ void load_rows(const uint16_t* base, int64_t stride, int left, int lane, v4i (&f)[DH / 16]) {
  const int r = lane & 31, hf = lane >> 5;
  const uint16_t* p = base + (int64_t)r * stride + 8 * hf;
#pragma unroll
  for (int st = 0; st < DH / 16; ++st) f[st] = r < left ? *(const v4i*)(p + 16 * st) : v4i{0, 0, 0, 0};
}

// The values are there from here on: used in a loop that waits for its own loads by count, they must not be waited for again.
template <int N>
__device__ __forceinline__ void arrived(v4i (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// The 32 columns that a wave holds of a result turned (lane l: column l & 31, values i of channel tile mt are channels
// 32 mt + 8 (i >> 2) + 4 (l >> 5) + (i & 3)), times `scale`, as rows of the 16-bit type: through the wave's own part of LDS
// (32 rows of 16 bytes more than a row) to whole rows in memory. Rows from `left` on are not written. REST: what the rounding
// to the type takes off, instead.
template <int DH, bool F16, bool REST = false>
__device__ __forceinline__ void store_turned(const v16f (&o)[DH / 32], float scale, uint8_t* lds, int lane, uint16_t* base,
                                             int64_t stride, int left) {
  constexpr int ROW = row_bytes<DH> + 16, LANES = row_bytes<DH> / 16, PER = 64 / LANES;
  const int c = lane & 31, hf = lane >> 5;
  const auto two = [&](float a, float b) {
    const uint32_t w = pack<F16>(a * scale, b * scale);
    return REST ? pack<F16>(a * scale - lo16<F16>(w), b * scale - hi16<F16>(w)) : w;
  };
#pragma unroll
  for (int mt = 0; mt < DH / 32; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *(uint2*)(lds + c * ROW + (32 * mt + 8 * i + 4 * hf) * 2) =
          make_uint2(two(o[mt][4 * i], o[mt][4 * i + 1]), two(o[mt][4 * i + 2], o[mt][4 * i + 3]));
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): the wave's rows are in LDS (it reads only its own)
  __builtin_amdgcn_wave_barrier();
  const int piece = lane & (LANES - 1);
#pragma unroll
  for (int j = 0; j < 32 / PER; ++j) {
    const int r = j * PER + lane / LANES;
    const v4i x = *(const v4i*)(lds + r * ROW + piece * 16);
    if (r < left) *(v4i*)(base + (int64_t)r * stride + piece * 8) = x;
  }
}
template <int DH>
constexpr int STAGING = 32 * (row_bytes<DH> + 16);   // LDS bytes of a wave

// 64 fp32 values from p on, `left` of them there (zeros behind), to LDS, a value a lane.
__device__ __forceinline__ void dma4(const float* p, int left, uint32_t off, uint8_t* lds) {
  uint32_t keep;
  const uint32_t dst = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)lds);
  const v4i rs = {__builtin_amdgcn_readfirstlane((int)(uint32_t)(uint64_t)p), __builtin_amdgcn_readfirstlane((int)((uint64_t)p >> 32 & 0xFFFF)),
                  __builtin_amdgcn_readfirstlane(max(0, min(left, 64)) * 4), 0x00027000};
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(off), "s"(rs), "s"(dst) : "memory");
}

struct Shape {
  int64_t seqs, q_rows, k_rows;
  int q_heads, k_heads, group, common;   // common: xcd_common
  const int32_t *starts, *k_starts;
  int causal;
  float scale, sl2;   // sm_scale, and times log2(e)
};

}  // namespace packed
}  // namespace lbw
