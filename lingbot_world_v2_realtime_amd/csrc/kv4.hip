// A cache of K and V in 4 bits, in pages of 64 tokens (include/lbw_causal.h): tokens written, read back, and attended.
//
// Codes are e2m1 with a power of two for each 32 channels of a token: a value is exact in bf16, and v_cvt_scalef32_pk_bf16_fp4
// makes two of them, scale and all, in one instruction, so the products are bf16 matrix products with nothing to correct.
// The layouts are those of the products' operands: a lane's 16 bytes of K are its key's channels in the four steps of
// 32; its 16 bytes of V are 8 keys at 4 channels, in the order in which S^T leaves their weights in registers.
//
// All of it is bound by memory, or by a launch's latency where there is little. 6914 tokens of 8 heads of 128 written 9.5 us, read
// back 9.5 (3.8 TB/s each); 64 sequences' single tokens 5.1 and 4.8, with starts (by blocks) 5.2 and 4.1. One query of 32 heads over 8 for each of 61 sequences of up to
// 6032: 50 us and 5 to join the segments (204 MB: 3.7 TB/s in all); 5 tokens of 12 heads in fp16 over 7 sequences of up to
// 24128: 44 and 5 (159 MB: 3.2); one sequence of 1508: 8 and 3.
#include "lbw_spans.h"

namespace lbw {
namespace {

constexpr int PAGE = LBW_KV4_PAGE, THREADS = 256;
constexpr float LOG2E = 1.4426950408889634f;

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct Pages {
  uint8_t *k4, *ks, *v4, *vs;
  int64_t heads, pages, width, t_s_seq, seqs, rows;
  const int32_t *starts, *lens, *table;
};

// The page of a sequence's token, or -1.
__device__ __forceinline__ int64_t page_of(const Pages& c, int64_t seq, int64_t pos) {
  if (seq < 0 || pos < 0 || pos / PAGE >= c.width) return -1;
  const int64_t p = c.table[seq * c.t_s_seq + pos / PAGE];
  return p >= 0 && p < c.pages ? p : -1;
}

// Byte of a token's V codes for channel n of 16 in group g of 32, and of its scale.
__device__ __forceinline__ int v_part(int t) { return t >> 2 & 3; }
__device__ __forceinline__ int v_slot(int t) { return (t >> 4 & 1) * 4 + (t & 3); }
template <int DH>
__device__ __forceinline__ int v_code_at(int t, int g, int n) {
  return (((((t >> 5) * (DH / 64) + (g >> 1)) * 4 + v_part(t)) * 16 + n) * 2 + (g & 1)) * 8 + v_slot(t);
}
template <int DH>
__device__ __forceinline__ int v_scale_at(int t, int g) { return (((t >> 5) * 4 + v_part(t)) * (DH / 32) + g) * 8 + v_slot(t); }

// 8 values of a group's 32 (four neighbouring lanes hold it) -> their codes, two a byte in order, and the group's scale.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t& scale) {
  float m = 0.f;
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    m = fmaxf(m, fabsf(x[e]));
    odd = odd || !(fabsf(x[e]) < INFINITY);
  }
  if (odd) m = INFINITY;
  m = fmaxf(m, dpp<DPP_XOR1>(m));
  m = fmaxf(m, dpp<DPP_XOR2>(m));
  const uint32_t b = __float_as_uint(m);
  // m = 1.f 2^E: 2^(E - 2) holds it up to 1.5, else 2^(E - 1)
  const int e = max((int)(b >> 23) - 2 + ((b & 0x7FFFFF) > 0x400000), 2);
  scale = b >= 0x7F800000u ? 255 : e;
  const float s = __uint_as_float((uint32_t)min(e, 253) << 23), most = 0x1.8p127f;   // 3 * 2^126
  uint32_t w = 0;
#define LBW_PAIR(i) w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, __builtin_amdgcn_fmed3f(x[2 * i], -most, most), __builtin_amdgcn_fmed3f(x[2 * i + 1], -most, most), s, i);
  LBW_PAIR(0) LBW_PAIR(1) LBW_PAIR(2) LBW_PAIR(3)
#undef LBW_PAIR
  return w;
}

// ---- one token for each sequence, without starts: 16 (8) lanes a head of K or V, all heads at once, so that a call is one load and one store long

struct Lane {
  int64_t seq, tile;   // tile: of the token's page and the head; seq < 0: nothing to do, tile < 0: in no page
  int64_t head;
  int t;
  bool is_k;
};
template <int LANES>
__device__ __forceinline__ Lane lane_of(const Pages& c) {
  const int64_t i = ((int64_t)group_id() * THREADS + threadIdx.x) / LANES, seq = i / (2 * c.heads), h2 = i - seq * 2 * c.heads;
  if (seq >= c.seqs) return {-1, -1, 0, 0, false};
  const int64_t pos = (int64_t)c.lens[seq] - 1, page = page_of(c, seq, pos), head = h2 < c.heads ? h2 : h2 - c.heads;
  return {seq, page < 0 ? -1 : page * c.heads + head, head, (int)(pos & (PAGE - 1)), h2 < c.heads};
}

template <int DH, bool F16>
__global__ __launch_bounds__(THREADS) void kv4_write_kernel(Pages c, const uint16_t* k, const uint16_t* v, int64_t k_tok, int64_t k_head,
                                                            int64_t v_tok, int64_t v_head) {
  constexpr int LANES = DH / 8;
  const Lane at = lane_of<LANES>(c);
  if (at.tile < 0) return;   // (the lanes of a head together)
  const int t = at.t, c8 = threadIdx.x % LANES, g = c8 >> 2, p = c8 & 3;
  float x[8];
  unpack8t<F16>(*(const v4i*)((at.is_k ? k + at.seq * k_tok + at.head * k_head : v + at.seq * v_tok + at.head * v_head) + 8 * c8), x);
  uint32_t scale;
  const uint32_t w = encode8(x, scale), other = dpp_u32<DPP_XOR2>(w);
  if (at.is_k) {
    *(uint32_t*)(c.k4 + (at.tile * PAGE + t) * (DH / 2) + p * (DH / 8) + g * 4) = w;
    if (p == 0) c.ks[(at.tile * PAGE + t) * (DH / 32) + g] = (uint8_t)scale;
  } else {
    // channels 8 (p & 1) + .. of the low (p < 2) or the high 16: the first four bytes by the one, the others by the other
    uint8_t* to = c.v4 + at.tile * (PAGE * DH / 2);
    const uint32_t lo = p < 2 ? w : other, hi = p < 2 ? other : w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = (p < 2 ? 0 : 4) + e;
      to[v_code_at<DH>(t, g, 8 * (p & 1) + n)] = (uint8_t)((lo >> 4 * n & 15) | (hi >> 4 * n & 15) << 4);
    }
    if (p == 0) c.vs[at.tile * (PAGE * DH / 32) + v_scale_at<DH>(t, g)] = (uint8_t)scale;
  }
}

// 8 codes, two a byte -> bf16. The instruction takes the exponent of its scale operand alone; 255 gives NaN.
__device__ __forceinline__ v4i decode8(uint32_t w, float scale) {
  return v4i{(int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
             (int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
             (int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
             (int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}
// Byte i of a word as that operand: its exponent bits, and whatever falls around them.
__device__ __forceinline__ float scale_at(uint32_t w, int i) { return __uint_as_float(i < 3 ? w << (23 - 8 * i) : w >> 1); }

template <int DH>
__global__ __launch_bounds__(THREADS) void kv4_read_kernel(Pages c, uint16_t* k, uint16_t* v) {
  constexpr int LANES = DH / 8;
  const Lane at = lane_of<LANES>(c);
  if (at.seq < 0) return;
  const int t = at.t, c8 = threadIdx.x % LANES, g = c8 >> 2, p = c8 & 3;
  v4i x = {0, 0, 0, 0};
  if (at.tile >= 0 && at.is_k) {
    x = decode8(*(const uint32_t*)(c.k4 + (at.tile * PAGE + t) * (DH / 2) + p * (DH / 8) + g * 4), scale_at(c.ks[(at.tile * PAGE + t) * (DH / 32) + g], 0));
  } else if (at.tile >= 0) {
    const uint8_t* from = c.v4 + at.tile * (PAGE * DH / 2);
    uint32_t w = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) w |= (uint32_t)(from[v_code_at<DH>(t, g, 8 * (p & 1) + n)] >> (p < 2 ? 0 : 4) & 15) << 4 * n;
    x = decode8(w, scale_at(c.vs[at.tile * (PAGE * DH / 32) + v_scale_at<DH>(t, g)], 0));
  }
  *(v4i*)((at.is_k ? k : v) + (at.seq * c.heads + at.head) * DH + 8 * c8) = x;
}

// ---- with starts: a workgroup a head's 32 tokens between two multiples of 32, whose V codes are neighbours in memory (also where
// there are few: a wave for each token instead took 9.2 us for 7.6 at one token, 26.9 for 20.4 at 64 sequences of 128)

constexpr int BLOCK = 32;

// The tokens of a call in blocks: where sequence s holds positions [from, to), the blocks from / 32 to (to - 1) / 32, numbered
// from starts[s] / 32 + 2 s on (n tokens lie in n / 32 + 2 blocks at most).
struct Block {
  int64_t seq, row;   // row: of the block's first token, were it one of the call
  int64_t pos;        // its position
  int first, end;     // tokens of the block that are the call's
};
inline int64_t blocks_of(int64_t rows, int64_t seqs) { return rows / BLOCK + 2 * seqs; }
__device__ __forceinline__ Block block_of(const Pages& c, int64_t want) {
  const int64_t s = last_of(c.seqs, want, [&](int64_t i) { return min(max((int64_t)c.starts[i], (int64_t)0), c.rows) / BLOCK + 2 * i; });
  if (s < 0) return {-1, 0, 0, 0, 0};
  const Span of = span(c.starts, s, c.rows);
  const int64_t from = (int64_t)c.lens[s] - of.n, to = c.lens[s];   // (from below zero: tokens before the first, in no page)
  const int64_t base = min(max((int64_t)c.starts[s], (int64_t)0), c.rows) / BLOCK + 2 * s;
  const int64_t pos = ((from >> 5) + want - base) * BLOCK;
  static_assert(BLOCK == 1 << 5, "the shift rounds down below zero too");
  if (of.n == 0 || want < base || pos >= to) return {-1, 0, 0, 0, 0};   // (starts that fall: a sequence behind the number)
  return {s, of.first + pos - from, pos, (int)max(from - pos, (int64_t)0), (int)min(to - pos, (int64_t)BLOCK)};
}

template <int DH, bool F16>
__global__ __launch_bounds__(THREADS) void kv4_write_block_kernel(Pages c, const uint16_t* k, const uint16_t* v, int64_t k_tok, int64_t k_head,
                                                                  int64_t v_tok, int64_t v_head) {
  constexpr int LANES = DH / 8, G = DH / 32, ROWS = THREADS / LANES;   // tokens of a pass
  __shared__ uint32_t codes[BLOCK][LANES + 1];
  __shared__ uint8_t scales[BLOCK][G];
  const uint32_t id = group_id(), head = id % (uint32_t)c.heads;
  const Block b = block_of(c, id / (uint32_t)c.heads);
  const int64_t page = page_of(c, b.seq, b.pos);
  if (page < 0) return;
  const int64_t tile = page * c.heads + head;
  const int c8 = threadIdx.x % LANES, g = c8 >> 2, p = c8 & 3, t0 = (int)(b.pos & (PAGE - 1));
#pragma unroll
  for (int i = 0; i < BLOCK / ROWS; ++i) {
    const int t = i * ROWS + threadIdx.x / LANES;
    const bool live = t >= b.first && t < b.end;   // (lanes of a group together)
    float x[8] = {}, y[8] = {};
    if (live) {
      unpack8t<F16>(*(const v4i*)(k + (b.row + t) * k_tok + head * k_head + 8 * c8), x);
      unpack8t<F16>(*(const v4i*)(v + (b.row + t) * v_tok + head * v_head + 8 * c8), y);
    }
    uint32_t ks, vs;
    const uint32_t kw = encode8(x, ks), vw = encode8(y, vs);
    codes[t][c8] = vw;
    if (p == 0) scales[t][g] = (uint8_t)vs;
    if (!live) continue;
    *(uint32_t*)(c.k4 + (tile * PAGE + t0 + t) * (DH / 2) + p * (DH / 8) + g * 4) = kw;
    if (p == 0) c.ks[(tile * PAGE + t0 + t) * G + g] = (uint8_t)ks;
  }
  __syncthreads();
  // 16 bytes of V: channel n of two groups, the 8 tokens of part p; then the scales of a part and group, 8 bytes
  const bool all = b.first == 0 && b.end == BLOCK;
  uint8_t *to = c.v4 + tile * (PAGE * DH / 2) + t0 * (DH / 2), *sc = c.vs + tile * (PAGE * G) + t0 * G;
  for (int i = threadIdx.x; i < BLOCK * DH / 32; i += THREADS) {
    const int n = i & 15, vp = i >> 4 & 3, g2 = i >> 6;
    uint32_t w[4] = {};
#pragma unroll
    for (int e = 0; e < 16; ++e) {   // (half a group's channels, then the other's)
      const int t = 16 * (e >> 2 & 1) + 4 * vp + (e & 3), at = 4 * (2 * g2 + (e >> 3)) + (n >> 3);
      const uint32_t byte = (codes[t][at] >> 4 * (n & 7) & 15) | (codes[t][at + 2] >> 4 * (n & 7) & 15) << 4;
      w[e >> 2] |= byte << 8 * (e & 3);
    }
    if (all) {
      *(v4i*)(to + i * 16) = v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int t = 16 * (e >> 2 & 1) + 4 * vp + (e & 3);
        if (t >= b.first && t < b.end) to[i * 16 + e] = (uint8_t)(w[e >> 2] >> 8 * (e & 3));
      }
    }
  }
  for (int i = threadIdx.x; i < BLOCK * G; i += THREADS) {
    const int e = i & 7, vg = i / 8 % G, vp = i / (8 * G), t = 16 * (e >> 2) + 4 * vp + (e & 3);
    if (t >= b.first && t < b.end) sc[i] = scales[t][vg];
  }
}

template <int DH>
__global__ __launch_bounds__(THREADS) void kv4_read_block_kernel(Pages c, uint16_t* k, uint16_t* v, int64_t blocks) {
  constexpr int LANES = DH / 8, G = DH / 32, ROWS = THREADS / LANES;
  __shared__ __align__(16) uint8_t codes[BLOCK * DH / 2];
  __shared__ uint8_t scales[BLOCK * G];
  const uint32_t id = group_id(), head = id % (uint32_t)c.heads;
  const int64_t want = id / (uint32_t)c.heads, o_tok = c.heads * DH;
  if (want >= blocks) return;
  for (uint16_t* out : {k, v})
    zero_outside(c.starts, c.seqs, c.rows, out + head * DH, o_tok, DH, (uint32_t)want, (uint32_t)blocks, threadIdx.x, THREADS);
  const Block b = block_of(c, want);
  if (b.seq < 0) return;
  const int64_t page = page_of(c, b.seq, b.pos), tile = page * c.heads + head;
  const int c8 = threadIdx.x % LANES, g = c8 >> 2, p = c8 & 3, t0 = (int)(b.pos & (PAGE - 1));
  if (page >= 0) {
    const uint8_t *from = c.v4 + tile * (PAGE * DH / 2) + t0 * (DH / 2), *sc = c.vs + tile * (PAGE * G) + t0 * G;
    for (int i = threadIdx.x; i < BLOCK * DH / 32; i += THREADS) *(v4i*)(codes + i * 16) = *(const v4i*)(from + i * 16);
    for (int i = threadIdx.x; i < BLOCK * G; i += THREADS) scales[i] = sc[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < BLOCK / ROWS; ++i) {
    const int t = i * ROWS + threadIdx.x / LANES;
    if (t < b.first || t >= b.end) continue;
    v4i x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    if (page >= 0) {
      const uint32_t kw = *(const uint32_t*)(c.k4 + (tile * PAGE + t0 + t) * (DH / 2) + p * (DH / 8) + g * 4);
      uint32_t vw = 0;
#pragma unroll
      for (int n = 0; n < 8; ++n) vw |= (uint32_t)(codes[v_code_at<DH>(t, g, 8 * (p & 1) + n)] >> (p < 2 ? 0 : 4) & 15) << 4 * n;
      x = decode8(kw, scale_at(c.ks[(tile * PAGE + t0 + t) * G + g], 0));
      y = decode8(vw, scale_at(scales[v_scale_at<DH>(t, g)], 0));
    }
    *(v4i*)(k + (b.row + t) * o_tok + head * DH + 8 * c8) = x;
    *(v4i*)(v + (b.row + t) * o_tok + head * DH + 8 * c8) = y;
  }
}

// ---------------------------------------------------------------- attention

constexpr int KB = 32, WAVES = THREADS / 64;   // keys of a wave's step
constexpr float LOWEST = -0x1.fffffep127f;

struct AttnArgs {
  Pages c;
  const uint16_t* q;
  int64_t q_tok, q_head;
  int q_heads, group, row_tiles;    // row_tiles: waves that share the heads of a group where those of one token are too many
  int tokens, tile_rows;            // tokens of a wave's rows, and how many rows those are at most
  uint32_t places, shares;          // shares: waves that share a head's work evenly; 0: one for each place's rows
  int64_t segments;                 // of a head, at most
  float sl2;
  uint16_t* out;
  float *part, *stats;              // [heads][segments][tile_rows][DH], [..][2]: sums, and the maximum and sum of the weights
  int2* parts;                      // [places][row_tiles]: a tile's first segment, and its last
};

__device__ __forceinline__ v4f mfma16(const v4i a, const v4i b, const v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float sum_quarters(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The codes and scales of a step's 32 keys as a lane holds them. Lane (part p = lane / 16, n = lane % 16): K of keys n and
// 16 + n, channels 32 j + 8 p .. + 8; V of keys 16 (e / 4) + 4 p + e % 4 at channels 32 g + n and 32 g + 16 + n.
template <int DH>
struct Step {
  static constexpr int G = DH / 32;
  uint32_t k[2][G], ks[2], v[G][2], vs[G][2];
  __device__ __forceinline__ void load(const Pages& c, int64_t tile, int half, int lane) {
    const int n = lane & 15, p = lane >> 4;
    typedef uint32_t vec __attribute__((ext_vector_type(G)));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int64_t key = tile * PAGE + half * KB + 16 * x + n;
      const vec w = *(const vec*)(c.k4 + key * (DH / 2) + p * (DH / 8));
#pragma unroll
      for (int j = 0; j < G; ++j) k[x][j] = w[j];
      if constexpr (G == 4) ks[x] = *(const uint32_t*)(c.ks + key * G);
      else ks[x] = *(const uint16_t*)(c.ks + key * G);
    }
    const uint8_t *vc = c.v4 + tile * (PAGE * DH / 2) + half * (KB * DH / 2), *sc = c.vs + tile * (PAGE * G) + half * (KB * G) + p * (8 * G);
#pragma unroll
    for (int g2 = 0; g2 < G / 2; ++g2) {
      const v4i w = *(const v4i*)(vc + ((g2 * 4 + p) * 16 + n) * 16), s = *(const v4i*)(sc + g2 * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * g2 + (e >> 1)][e & 1] = w[e];
        vs[2 * g2 + (e >> 1)][e & 1] = s[e];
      }
    }
  }
};

// A head's work as a line of units, each a tile of rows against a page: sequence by sequence its tiles of tokens, of each the
// pages of its keys. Wave i of n takes the units from i U / n to (i + 1) U / n, wherever those end (n: no more than there are
// units): all of them finish together, however different the sequences are. What a wave does of one tile is a segment; a
// tile whose keys are cut has several, one behind the other, which a second kernel joins. Every head has a line of its own,
// cut alike, and the waves of all heads at one place of it are neighbours: they read the same pages at the same time, which
// memory likes (61 sequences of up to 6032 tokens, 8 heads, pages anywhere: 59 us, and 75 with one line of all heads, at four waves a tile).
constexpr int UNIT = PAGE;

struct Spot {
  int64_t seq;
  uint32_t units_before, tiles_before, tiles, units;   // of the line; of the sequence: its tiles, and units of each
};
struct Line {
  const AttnArgs& a;
  // (sums stop at MOST, which a call's work lies below: starts that fall can make more of it, and make none)
  static constexpr uint32_t MOST = 1u << 30;
  uint32_t total, n, all_w, all_t, w, t, l;   // a lane's sequence of 64: units and tiles up to it, its tiles' units
  uint32_t own_w, own_t;

  __device__ __forceinline__ void look(int64_t s0) {
    const int64_t s = s0 + (threadIdx.x & 63);
    l = own_t = 0;
    if (s < a.c.seqs) {
      const int count = a.c.starts ? span(a.c.starts, s, a.c.rows).n : 1;
      own_t = (uint32_t)min(((int64_t)count + a.tokens - 1) / a.tokens * a.row_tiles, (int64_t)MOST);
      l = (uint32_t)((min(max((int64_t)a.c.lens[s], (int64_t)0), a.c.width * PAGE) + UNIT - 1) / UNIT);
    }
    w = own_w = (uint32_t)min((uint64_t)own_t * l, (uint64_t)MOST);
    t = own_t;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_up(w, o), y = __shfl_up(t, o);
      if ((threadIdx.x & 63) >= o) w = min(w + x, MOST), t = min(t + y, MOST);
    }
    all_w = __shfl(w, 63), all_t = __shfl(t, 63);
  }
  __device__ __forceinline__ explicit Line(const AttnArgs& args) : a(args) {
    uint32_t tiles = 0;
    total = 0;
    for (int64_t s0 = 0; s0 < a.c.seqs; s0 += 64) {
      look(s0);
      total = min(total + all_w, MOST), tiles = min(tiles + all_t, MOST);
    }
    n = total < MOST && tiles <= (uint32_t)(a.segments - a.shares) ? min(a.shares, total) : 0;
  }
  // the sequence at which f(its units up to and with it, its number) becomes true
  template <typename F>
  __device__ __forceinline__ Spot find(F f) {
    uint32_t before = 0, tiles = 0;
    for (int64_t s0 = 0; s0 < a.c.seqs; s0 += 64) {
      if (a.c.seqs > 64) look(s0);
      const uint64_t hit = __ballot(f(before + w, s0 + (threadIdx.x & 63)));
      if (hit) {
        const int at = __builtin_ctzll(hit);
        const uint32_t ow = __shfl(own_w, at), ot = __shfl(own_t, at);
        return {s0 + at, (uint32_t)__builtin_amdgcn_readfirstlane(before + __shfl(w, at) - ow),
                (uint32_t)__builtin_amdgcn_readfirstlane(tiles + __shfl(t, at) - ot), (uint32_t)__builtin_amdgcn_readfirstlane(ot),
                (uint32_t)__builtin_amdgcn_readfirstlane((int)__shfl(l, at))};
      }
      before += all_w, tiles += all_t;
    }
    return {-1, 0, 0, 0, 0};
  }
  __device__ __forceinline__ uint32_t share(uint32_t i) const { return (uint32_t)((uint64_t)i * total / n); }
};

// A segment: up to 16 RT rows (tokens x the heads that share a head of the cache) over a run of keys, 32 a step, by one wave. S^T = K Q^T on v_mfma_f32_16x16x32_bf16: a lane holds one row and 8 of the 32 keys; the row's maximum needs two
// exchanges; P^T goes from those registers into O^T += V^T P^T. fp16 q and P enter as two bf16 values each, high and low.
constexpr int RT = 1;   // 16-row tiles of a wave (with two, which leave room for fewer waves: 20 rows of 16 sequences 43 us for 39, 64 rows 64 for 67)
template <int DH>
constexpr int ATTN_WAVES = DH == 128 ? 3 : 4;   // a SIMD

template <int DH, bool F16>
__global__ __launch_bounds__(THREADS, ATTN_WAVES<DH>) void kv4_attn_kernel(AttnArgs a) {
  constexpr int G = DH / 32, NT = DH / 16;
  const uint32_t id = __builtin_amdgcn_readfirstlane(group_id() * WAVES + (threadIdx.x >> 6)), heads = (uint32_t)a.c.heads;
  // where the wave is: a head, a sequence, a tile in it (tokens, part of the group), and the units of its keys
  int64_t seq;
  uint32_t head, tile = 0, unit = 0, units = 0, left = 1, tiles = 0, tiles_before = 0;   // left: units to go
  if (a.shares) {
    const uint32_t mine = id / heads;
    head = id - mine * heads;
    Line line(a);
    if (mine >= line.n) return;
    const uint32_t u = line.share(mine);
    left = line.share(mine + 1) - u;
    const Spot at = line.find([&](uint32_t upto, int64_t) { return upto > u; });
    seq = at.seq, tiles = at.tiles, units = at.units, tiles_before = at.tiles_before;
    tile = (u - at.units_before) / units;
    unit = u - at.units_before - tile * units;
  } else {
    const uint32_t rest = id / heads, at = rest / a.row_tiles;
    head = id - rest * heads;
    tile = rest - at * a.row_tiles;
    if (at >= a.places) return;
    if (a.c.starts && tile == 0)
      zero_outside(a.c.starts, a.c.seqs, a.c.rows, a.out + (int64_t)head * a.group * DH, (int64_t)a.q_heads * DH, a.group * DH, at, a.places,
                   threadIdx.x & 63, 64);
    seq = at;
    if (a.c.starts) {
      const Place pl = place(a.c.starts, a.c.seqs, a.c.rows, a.tokens, at);
      if (pl.seq < 0) return;
      seq = pl.seq;
      tile += pl.tile * a.row_tiles;
    }
  }
  while (true) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // (what is made of it is made here again for each segment: kept, it would take 30 registers)
  const int n = lane & 15, p = lane >> 4;
  seq = __builtin_amdgcn_readfirstlane((int)seq);
  // (read by vector loads, for the kernel writes memory too: brought back to what one value of a wave is)
  const Span of = a.c.starts ? span(a.c.starts, seq, a.c.rows) : Span{seq, 1};
  const int64_t first = __builtin_amdgcn_readfirstlane((int)of.first);
  const int count = __builtin_amdgcn_readfirstlane(of.n);
  const uint32_t row_tile = tile % a.row_tiles;
  const int token0 = (int)(tile / a.row_tiles) * a.tokens;
  // (the rows' places go by the length as it is, the keys end where the table does)
  const int64_t held = __builtin_amdgcn_readfirstlane(a.c.lens[seq]), len = min(max(held, (int64_t)0), a.c.width * PAGE);
  // row i of the tile: token token0 + i / heads_here, head i % heads_here of the group (from row_tile on where they are many)
  const int group0 = row_tile * 16 * RT, heads_here = min(a.group - group0, a.row_tiles > 1 ? 16 * RT : a.group);
  const int rows = min(a.tokens, count - token0) * heads_here;
  const int64_t seen = held - count + token0 + 1;   // keys that the first token sees, were all of them in the table
  const int upto = (int)max((int64_t)0, min(len, seen + min(a.tokens, count - token0) - 1));
  const uint32_t run = a.shares ? min(left, units - unit) : 0;
  const int k0 = (int)unit * UNIT, k1 = a.shares ? min(upto, k0 + (int)run * UNIT) : upto;
  const bool whole = !a.shares || run == units;
  if (a.shares && head == 0) {   // where the tile's segments begin and end, for the join
    const int64_t from = a.c.starts ? min(max((int64_t)a.c.starts[seq], (int64_t)0), a.c.rows) / a.tokens : 0;
    int* at = (int*)(a.parts + (from + seq) * a.row_tiles + tile);
    const int mine = (int)(id / heads + tiles_before + tile);
    if (lane == 0 && unit == 0) at[0] = mine;
    if (lane == 0 && unit + run == units) at[1] = mine;
  }

  v4i qh[RT][G], ql[F16 ? RT : 1][G];
  int own[RT];   // keys that the lane's row sees
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int i = rt * 16 + n, tok = i / heads_here, h = i - tok * heads_here;
    own[rt] = i < rows ? (int)min((int64_t)k1, seen + tok) : 0;
    const uint16_t* from = a.q + (first + token0 + tok) * a.q_tok + ((int64_t)head * a.group + group0 + h) * a.q_head + 8 * p;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const v4i x = i < rows ? *(const v4i*)(from + 32 * j) : v4i{0, 0, 0, 0};
      if constexpr (F16) {
        float f[8];
        unpack8t<true>(x, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t hi = pack2<LBW_DTYPE_BF16>(f[2 * e], f[2 * e + 1]);
          qh[rt][j][e] = (int)hi;
          // (an infinity has no rest)
          const float r0 = f[2 * e] - lo16<false>(hi), r1 = f[2 * e + 1] - hi16<false>(hi);
          ql[rt][j][e] = (int)pack2<LBW_DTYPE_BF16>(r0 == r0 ? r0 : 0.f, r1 == r1 ? r1 : 0.f);
        }
      } else {
        qh[rt][j] = x;
      }
    }
  }

  v4f o[RT][NT];
  float top[RT], total[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = -INFINITY, total[rt] = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[rt][i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // the pages of the run, 64 at a time, one a lane
  int page0 = k0 / PAGE, mine = -1;
  const auto pages = [&] {
    const int64_t t = page0 + lane;
    mine = t * PAGE < k1 ? (int)page_of(a.c, seq, t * PAGE) : -1;
  };
  pages();
  // a step's codes are loaded while the step before it is worked on
  Step<DH> next;
  const auto fetch = [&](int key) {
    if (key / PAGE - page0 >= 64) {
      page0 = key / PAGE;
      pages();
    }
    const int page = __builtin_amdgcn_readlane(mine, key / PAGE - page0);
    if (page >= 0) next.load(a.c, (int64_t)page * heads + head, key / KB & 1, lane);
    return page;
  };
  int next_page = -1, first_held = INT32_MAX;   // the first key in a page that there is
  if (k0 < k1) next_page = fetch(k0);
  for (int key = k0; key < k1; key += KB) {
    const int page = next_page;
    Step<DH> st = next;
    if (key + KB < k1) next_page = fetch(key + KB);
    if (page < 0) continue;
    first_held = min(first_held, key);
    // Some row may not see all of these keys: those behind the last hold what they like, and a NaN must not reach the rows
    // that do not see it through a weight of zero. Their scales become 1 (127), and the NaN is put where it belongs below.
    const bool edge = key + KB > seen;
    bool odd = false;
    if (edge) {
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at_key = key + 16 * (e >> 2) + 4 * p + (e & 3);
          const bool nan = (st.vs[g][e >> 2] >> 8 * (e & 3) & 255) == 255;
          if (at_key < seen || (at_key < k1 && !nan)) continue;
          odd = odd || at_key < k1;
          st.vs[g][e >> 2] = (st.vs[g][e >> 2] & ~(255u << 8 * (e & 3))) | 127u << 8 * (e & 3);
        }
    }
    v4i kf[2][G], ph[RT], pl[F16 ? RT : 1];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < G; ++j) kf[x][j] = decode8(st.k[x][j], scale_at(st.ks[x], j));
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      v4f s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < G; ++j) {
          s[x] = mfma16(kf[x][j], qh[rt][j], s[x]);
          if constexpr (F16) s[x] = mfma16(kf[x][j], ql[rt][j], s[x]);
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key + 16 * x + 4 * p + i >= own[rt]) s[x][i] = -INFINITY;
        }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = max_xor32(max_xor16(mx)) * a.sl2;
      const float next = fmaxf(top[rt], mx);
      if (__any(next > top[rt])) {
        const float by = top[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[rt] - next);
#pragma unroll
        for (int i = 0; i < NT; ++i) o[rt][i] *= by;
        total[rt] *= by;
        top[rt] = next;
      }
      const float off = top[rt] == -INFINITY ? 0.f : -top[rt];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = __builtin_amdgcn_exp2f(fmaf(s[x][i], a.sl2, off));
        total[rt] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t hi = pack2<LBW_DTYPE_BF16>(pr[2 * i], pr[2 * i + 1]);
          ph[rt][2 * x + i] = (int)hi;
          if constexpr (F16) pl[rt][2 * x + i] = (int)pack2<LBW_DTYPE_BF16>(pr[2 * i] - lo16<false>(hi), pr[2 * i + 1] - hi16<false>(hi));
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // (V's values made before their weights are there only take registers)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t two[8];   // channel 32 g + n low, 32 g + 16 + n high, of the lane's 8 keys
#define LBW_KEY(e) two[e] = __builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(st.v[g][e >> 2], scale_at(st.vs[g][e >> 2], e & 3), e & 3));
      LBW_KEY(0) LBW_KEY(1) LBW_KEY(2) LBW_KEY(3) LBW_KEY(4) LBW_KEY(5) LBW_KEY(6) LBW_KEY(7)
#undef LBW_KEY
      v4i vf[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vf[0][e] = (int)__builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x05040100u);
        vf[1][e] = (int)__builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x07060302u);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          o[rt][2 * g + x] = mfma16(vf[x], ph[rt], o[rt][2 * g + x]);
          if constexpr (F16) o[rt][2 * g + x] = mfma16(vf[x], pl[rt], o[rt][2 * g + x]);
        }
    }
    if (__any(odd)) {
      for (int t = (int)max((int64_t)0, seen - key); t < min(KB, k1 - key); ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int64_t at_scale = ((int64_t)page * a.c.heads + head) * (PAGE * G) + v_scale_at<DH>((key & (PAGE - 1)) + t, g);
          if (a.c.vs[at_scale] != 255) continue;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float x = o[rt][2 * g + (i >> 2)][i & 3];
              o[rt][2 * g + (i >> 2)][i & 3] = key + t < own[rt] ? __builtin_nanf("") : x;
            }
        }
    }
  }

  // O^T's lane (p, n) holds channels 16 i + 4 p .. + 4 of row n
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int i = rt * 16 + n;
    const float sum = sum_quarters(total[rt]);
    // A sum of zero over keys that there are: all scores are minus infinity, and the row has no softmax (NaN), unless another
    // segment has scores of it: to the join such a segment has a maximum, LOWEST, and a row that sees nothing has none.
    const bool low = sum == 0.f && first_held < own[rt];
    if (i < rows) {
      if (whole) {
        const int tok = i / heads_here, h = i - tok * heads_here;
        uint16_t* to = a.out + ((first + token0 + tok) * a.q_heads + (int64_t)head * a.group + group0 + h) * DH + 4 * p;
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : low ? __builtin_nanf("") : 0.f;
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          constexpr int DT = F16 ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16;
          *(uint2*)(to + 16 * x) = make_uint2(pack2<DT>(o[rt][x][0] * inv, o[rt][x][1] * inv), pack2<DT>(o[rt][x][2] * inv, o[rt][x][3] * inv));
        }
      } else {
        const int64_t at = ((int64_t)head * a.segments + id / heads + tiles_before + tile) * a.tile_rows + i;
#pragma unroll
        for (int x = 0; x < NT; ++x) *(v4f*)(a.part + at * DH + 16 * x + 4 * p) = o[rt][x];
        if (p == 0) *(float2*)(a.stats + at * 2) = make_float2(low ? LOWEST : top[rt], sum);
      }
    }
  }
  if (!a.shares || left == run) return;
  left -= run;
  unit = 0;
  if (++tile == tiles) {   // the next sequence that has any work
    tile = 0;
    do {
      tiles_before += tiles;
      ++seq;
      units = (uint32_t)((min(max((int64_t)__builtin_amdgcn_readfirstlane(a.c.lens[seq]), (int64_t)0), a.c.width * PAGE) + UNIT - 1) / UNIT);
      const int rows_of = a.c.starts ? __builtin_amdgcn_readfirstlane(span(a.c.starts, seq, a.c.rows).n) : 1;
      tiles = (uint32_t)((rows_of + a.tokens - 1) / a.tokens) * a.row_tiles;
    } while (units * tiles == 0);
  }
  }
}

// The segments of a row's tile joined, where it has several, and zeros where it has none: a workgroup a row and head, DH / 4
// lanes a segment, so that 8 (16) segments are read at once, four times over; each group of lanes keeps a running maximum and
// sum, and the groups' are joined in LDS.
template <int DH, bool F16>
__global__ __launch_bounds__(THREADS) void kv4_join_kernel(AttnArgs a) {
  constexpr int LANES = DH / 4, GROUPS = THREADS / LANES, AHEAD = 4, DT = F16 ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16;
  __shared__ __align__(16) v4f sums[GROUPS][LANES];
  __shared__ float2 stats[GROUPS];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t i = group_id();
  if (i >= a.c.rows * a.q_heads) return;
  const int64_t row = i / a.q_heads;
  const int hq = (int)(i - row * a.q_heads), head = hq / a.group, g = hq - head * a.group;
  int64_t seq = row, place = row;
  int token = 0;
  if (a.c.starts) {
    seq = last_of(a.c.seqs + 1, row, [&](int64_t s) { return (int64_t)a.c.starts[s]; });
    if (seq >= a.c.seqs) seq = -1;
    if (seq >= 0) {
      const Span of = span(a.c.starts, seq, a.c.rows);
      token = (int)(row - of.first);
      place = of.first / a.tokens + seq + token / a.tokens;
      if (token < 0 || token >= of.n) seq = -1;   // (starts that fall: a sequence that does not hold the row)
    }
  }
  int parts = 0;
  int64_t at = 0;   // the first segment's row
  if (seq >= 0 && a.c.lens[seq] > 0 && place < (int64_t)a.places) {
    const int row_tile = g / (16 * RT), heads_here = min(a.group - row_tile * 16 * RT, a.row_tiles > 1 ? 16 * RT : a.group);
    const int2 of = a.parts[place * a.row_tiles + row_tile];
    // (starts that fall leave places that no wave has written)
    parts = of.x >= 0 && of.y >= of.x && of.y < a.segments ? of.y - of.x + 1 : 0;
    if (parts == 1) return;   // (the one segment wrote the row)
    at = (head * a.segments + of.x) * a.tile_rows + token % a.tokens * heads_here + g - row_tile * 16 * RT;
  }
  float most = -INFINITY, total = 0.f;
  v4f x = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = group; s0 < parts; s0 += GROUPS * AHEAD) {
    float2 st[AHEAD];
    v4f p[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int s = s0 + k * GROUPS;
      const int64_t mine = at + (int64_t)s * a.tile_rows;
      st[k] = s < parts ? *(const float2*)(a.stats + mine * 2) : make_float2(-INFINITY, 0.f);
      p[k] = s < parts ? *(const v4f*)(a.part + mine * DH + lane * 4) : v4f{0.f, 0.f, 0.f, 0.f};
    }
    float next = most;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) next = fmaxf(next, st[k].x);
    const float before = most == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(most - next);
    total *= before;
    x *= before;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float by = st[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[k].x - next);
      total = fmaf(by, st[k].y, total);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(by, p[k][e], x[e]);
    }
    most = next;
  }
  sums[group][lane] = x;
  if (lane == 0) stats[group] = make_float2(most, total);
  __syncthreads();
  if (group) return;
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) top = fmaxf(top, stats[k].x);
  total = 0.f;
  x = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const float by = stats[k].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(stats[k].x - top);
    total = fmaf(by, stats[k].y, total);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaf(by, sums[k][lane][e], x[e]);
  }
  const float inv = total > 0.f || total != total ? 1.f / total : top > -INFINITY ? __builtin_nanf("") : 0.f;
  *(uint2*)(a.out + i * DH + lane * 4) = make_uint2(pack2<DT>(x[0] * inv, x[1] * inv), pack2<DT>(x[2] * inv, x[3] * inv));
}

// How a call's work is cut: tokens of a wave's rows, waves for a group's heads; the waves that share a head's work evenly (of
// all heads as many as run at once), or 0: each tile of rows has one of its own. To share takes a second kernel and a look at
// every sequence, about 2 us and 1 for 20 rows; not to share takes as long as the longest sequence's wave, 1.65 us a unit
// (which the table's width bounds), unless there are several waves for every place, which even out by themselves. Measured,
// us, shared and not (32 heads over 8, lengths of up to 100, 500 and 4000): 64 sequences 16, 12; 21, 23; 69, 127; 256: 31, 16;
// 54, 39; 173, 206; 1024: 94, 42; 157, 110; 526, 536; 128 and 256 of 5 tokens each, up to 3000: 160, 169; 284, 234.
struct Plan {
  int tokens, tile_rows, row_tiles, shares;
  int64_t places, segments;
  int64_t parts_at(int64_t heads, int64_t dim) const { return heads * segments * tile_rows * (dim + 2) * 4; }   // bytes
  int64_t bytes(int64_t heads, int64_t dim) const { return shares ? parts_at(heads, dim) + places * row_tiles * 8 : 0; }
};
Plan plan(int64_t seqs, int64_t rows, int64_t group, int64_t heads, int64_t dim, bool single, int64_t width) {
  Plan p;
  p.tokens = (int)std::max<int64_t>(1, 16 * RT / group);
  p.tile_rows = (int)std::min<int64_t>(16 * RT, p.tokens * group);
  p.row_tiles = (int)((group + 16 * RT - 1) / (16 * RT));
  p.places = single ? seqs : places_of(rows, seqs, p.tokens);
  const int waves = dim == 128 ? ATTN_WAVES<128> : ATTN_WAVES<64>;
  const int64_t tiles = p.places * p.row_tiles, most = (width * PAGE + UNIT - 1) / UNIT;
  p.shares = 16 * most > rows + 40 && tiles * heads < 4 * 1024 * waves && tiles * most < 1 << 30 ? (int)(1024 * waves / heads) : 0;
  p.segments = p.shares ? p.shares + tiles : 0;
  return p;
}

template <int DH, bool F16>
void launch_attn(const AttnArgs& a, hipStream_t stream) {
  const int64_t grid = a.shares ? a.shares * a.c.heads : (int64_t)a.places * a.c.heads * a.row_tiles;
  kv4_attn_kernel<DH, F16><<<grid_of((grid + WAVES - 1) / WAVES), THREADS, 0, stream>>>(a);
  if (a.shares) kv4_join_kernel<DH, F16><<<grid_of(a.c.rows * a.q_heads), THREADS, 0, stream>>>(a);
}

int check_pages(int64_t seqs, int64_t rows, int64_t heads, int64_t dim, const int32_t* starts, const int32_t* lens,
                const int32_t* table, int64_t t_s_seq, int64_t width, int64_t pages, const void* k4, const void* ks, const void* v4,
                const void* vs) {
  if (!lens || !table || !k4 || !ks || !v4 || !vs) return LBW_E_NULL;
  if (seqs < 1 || seqs > 65535 || rows < 1 || rows >= 1ll << 31 || (!starts && rows != seqs) || heads < 1 || heads > 4096 ||
      (dim != 64 && dim != 128) || width < 1 || width >= 1ll << 25 || pages < 1 || pages >= 1ll << 31 || t_s_seq < 0)
    return LBW_E_SHAPE;
  for (const void* p : {k4, ks, v4, vs})
    if ((uintptr_t)p % 16) return LBW_E_ALIGN;
  for (const void* p : {(const void*)starts, (const void*)lens, (const void*)table})
    if ((uintptr_t)p % 4) return LBW_E_ALIGN;
  return LBW_OK;
}
// Workgroups of a write or read.
int64_t groups_of(const int32_t* starts, int64_t rows, int64_t seqs, int64_t heads, int64_t dim) {
  return starts ? blocks_of(rows, seqs) * heads : (seqs * 2 * heads * (dim / 8) + THREADS - 1) / THREADS;
}
bool aligned(const void* p, int64_t tok, int64_t head) { return (uintptr_t)p % 16 == 0 && tok % 8 == 0 && head % 8 == 0 && tok >= 0 && head >= 0; }

}  // namespace
}  // namespace lbw

using namespace lbw;

extern "C" int lbw_kv4_write(const void* k, const void* v, int dtype, int64_t seqs, int64_t rows, int64_t heads, int64_t dim,
                             int64_t k_s_tok, int64_t k_s_head, int64_t v_s_tok, int64_t v_s_head, const int32_t* starts,
                             const int32_t* lens, const int32_t* table, int64_t t_s_seq, int64_t width, int64_t pages, uint8_t* k4,
                             uint8_t* ks, uint8_t* v4, uint8_t* vs, void* stream) {
  if (!k || !v) return LBW_E_NULL;
  if (const int st = check_pages(seqs, rows, heads, dim, starts, lens, table, t_s_seq, width, pages, k4, ks, v4, vs)) return st;
  if (dtype != LBW_DTYPE_BF16 && dtype != LBW_DTYPE_FP16) return LBW_E_SHAPE;
  if (!aligned(k, k_s_tok, k_s_head) || !aligned(v, v_s_tok, v_s_head)) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const Pages c = {k4, ks, v4, vs, heads, pages, width, t_s_seq, seqs, rows, starts, lens, table};
  const bool blocks = starts;
  const int64_t groups = groups_of(starts, rows, seqs, heads, dim);
  if (groups > 1 << 30) return LBW_E_SHAPE;
  const dim3 grid = grid_of(groups);
  const uint16_t *kp = (const uint16_t*)k, *vp = (const uint16_t*)v;
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (blocks && dim == 128) {
    if (f16) kv4_write_block_kernel<128, true><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
    else kv4_write_block_kernel<128, false><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
  } else if (blocks) {
    if (f16) kv4_write_block_kernel<64, true><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
    else kv4_write_block_kernel<64, false><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
  } else if (dim == 128) {
    if (f16) kv4_write_kernel<128, true><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
    else kv4_write_kernel<128, false><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
  } else {
    if (f16) kv4_write_kernel<64, true><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
    else kv4_write_kernel<64, false><<<grid, THREADS, 0, s>>>(c, kp, vp, k_s_tok, k_s_head, v_s_tok, v_s_head);
  }
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

extern "C" int lbw_kv4_read(int64_t seqs, int64_t rows, int64_t heads, int64_t dim, const int32_t* starts, const int32_t* lens,
                            const int32_t* table, int64_t t_s_seq, int64_t width, int64_t pages, const uint8_t* k4, const uint8_t* ks,
                            const uint8_t* v4, const uint8_t* vs, void* k, void* v, void* stream) {
  if (!k || !v) return LBW_E_NULL;
  if (const int st = check_pages(seqs, rows, heads, dim, starts, lens, table, t_s_seq, width, pages, k4, ks, v4, vs)) return st;
  if (((uintptr_t)k | (uintptr_t)v) % 16) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const Pages c = {(uint8_t*)k4, (uint8_t*)ks, (uint8_t*)v4, (uint8_t*)vs, heads, pages, width, t_s_seq, seqs, rows, starts, lens, table};
  const int64_t n = blocks_of(rows, seqs), groups = groups_of(starts, rows, seqs, heads, dim);
  if (groups > 1 << 30) return LBW_E_SHAPE;
  const bool blocks = starts;
  const dim3 grid = grid_of(groups);
  if (blocks && dim == 128) kv4_read_block_kernel<128><<<grid, THREADS, 0, (hipStream_t)stream>>>(c, (uint16_t*)k, (uint16_t*)v, n);
  else if (blocks) kv4_read_block_kernel<64><<<grid, THREADS, 0, (hipStream_t)stream>>>(c, (uint16_t*)k, (uint16_t*)v, n);
  else if (dim == 128) kv4_read_kernel<128><<<grid, THREADS, 0, (hipStream_t)stream>>>(c, (uint16_t*)k, (uint16_t*)v);
  else kv4_read_kernel<64><<<grid, THREADS, 0, (hipStream_t)stream>>>(c, (uint16_t*)k, (uint16_t*)v);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

extern "C" int64_t lbw_kv4_attn_workspace_bytes(int64_t seqs, int64_t rows, int64_t q_heads, int64_t heads, int64_t dim, int64_t width,
                                                int single) {
  if (seqs < 1 || rows < 1 || heads < 1 || q_heads < heads) return 0;
  const Plan p = plan(seqs, rows, q_heads / heads, heads, dim, single, width);
  return p.bytes(heads, dim);
}

extern "C" int lbw_kv4_attn(const void* q, int dtype, int64_t seqs, int64_t rows, int64_t q_heads, int64_t heads, int64_t dim,
                            int64_t q_s_tok, int64_t q_s_head, const int32_t* starts, const int32_t* lens, const int32_t* table,
                            int64_t t_s_seq, int64_t width, int64_t pages, const uint8_t* k4, const uint8_t* ks, const uint8_t* v4,
                            const uint8_t* vs, float sm_scale, void* out, void* workspace, void* stream) {
  if (!q || !out) return LBW_E_NULL;
  if (const int st = check_pages(seqs, rows, heads, dim, starts, lens, table, t_s_seq, width, pages, k4, ks, v4, vs)) return st;
  if ((dtype != LBW_DTYPE_BF16 && dtype != LBW_DTYPE_FP16) || q_heads < heads || q_heads > 4096 || q_heads % heads ||
      !(sm_scale > 0.f) || !(sm_scale < INFINITY))
    return LBW_E_SHAPE;
  const Plan p = plan(seqs, rows, q_heads / heads, heads, dim, !starts, width);
  if (p.places * heads * p.row_tiles > 1 << 30 || rows * q_heads > 1 << 30) return LBW_E_SHAPE;
  if (p.shares && !workspace) return LBW_E_NULL;
  if (!aligned(q, q_s_tok, q_s_head) || ((uintptr_t)out | (uintptr_t)workspace) % 16) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  float* part = (float*)workspace;
  const AttnArgs a = {{(uint8_t*)k4, (uint8_t*)ks, (uint8_t*)v4, (uint8_t*)vs, heads, pages, width, t_s_seq, seqs, rows, starts, lens, table},
                      (const uint16_t*)q, q_s_tok, q_s_head, (int)q_heads, (int)(q_heads / heads), p.row_tiles, p.tokens, p.tile_rows,
                      (uint32_t)p.places, (uint32_t)p.shares, p.segments, sm_scale * LOG2E, (uint16_t*)out, part,
                      part ? part + heads * p.segments * p.tile_rows * dim : nullptr,
                      part ? (int2*)((uint8_t*)part + p.parts_at(heads, dim)) : nullptr};
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (dim == 128) f16 ? launch_attn<128, true>(a, (hipStream_t)stream) : launch_attn<128, false>(a, (hipStream_t)stream);
  else f16 ? launch_attn<64, true>(a, (hipStream_t)stream) : launch_attn<64, false>(a, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
