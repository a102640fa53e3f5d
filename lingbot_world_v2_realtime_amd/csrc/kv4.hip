// A cache of K and V in 4 bits, in pages of 64 tokens (include/lbw_causal.h): tokens written, read back, and attended.
//
// Codes are e2m1 with a power of two for each 32 channels of a token: a value is exact in bf16, and v_cvt_scalef32_pk_bf16_fp4
// makes two of them, scale and all, in one instruction, so the products are bf16 matrix products with nothing to correct.
// The layouts are those of the products' operands: a lane's 16 bytes of K are its key's channels in the four steps of
// 32; its 16 bytes of V are 8 keys at 4 channels, in the order in which S^T leaves their weights in registers.
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

// Where row r of a call's tokens belongs: its sequence and its place in it; seq < 0 for a row of none.
struct Token {
  int64_t seq, pos;
};
__device__ __forceinline__ Token token_of(const Pages& c, int64_t r) {
  int64_t s = r, left = 1;   // (left: the sequence's rows from r on)
  if (c.starts) {
    s = last_of(c.seqs + 1, r, [&](int64_t i) { return (int64_t)c.starts[i]; });
    if (s < 0 || s >= c.seqs) return {-1, 0};
    left = min((int64_t)c.starts[s + 1], c.rows) - r;
  }
  return {s, (int64_t)c.lens[s] - left};
}
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

// A wave a token; 16 (8) lanes a head of K or V.
template <int DH, bool F16>
__global__ __launch_bounds__(THREADS) void kv4_write_kernel(Pages c, const uint16_t* k, const uint16_t* v, int64_t k_tok, int64_t k_head,
                                                            int64_t v_tok, int64_t v_head) {
  constexpr int LANES = DH / 8;
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)group_id() * (THREADS / 64) + (threadIdx.x >> 6);
  if (r >= c.rows) return;
  const Token at = token_of(c, r);
  const int64_t page = page_of(c, at.seq, at.pos);
  if (page < 0) return;
  const int t = (int)(at.pos % PAGE), c8 = lane % LANES, g = c8 >> 2, p = c8 & 3;
  for (int64_t i0 = 0; i0 < 2 * c.heads; i0 += 64 / LANES) {
    const int64_t i = i0 + lane / LANES;
    const bool live = i < 2 * c.heads, is_k = i < c.heads;   // (groups of four lanes are live together)
    const int64_t h = is_k ? i : i - c.heads, tile = page * c.heads + h;
    float x[8] = {};
    if (live) unpack8t<F16>(*(const v4i*)((is_k ? k + r * k_tok + h * k_head : v + r * v_tok + h * v_head) + 8 * c8), x);
    uint32_t scale;
    const uint32_t w = encode8(x, scale), other = dpp_u32<DPP_XOR2>(w);
    if (!live) continue;
    if (is_k) {
      *(uint32_t*)(c.k4 + (tile * PAGE + t) * (DH / 2) + p * (DH / 8) + g * 4) = w;
      if (p == 0) c.ks[(tile * PAGE + t) * (DH / 32) + g] = (uint8_t)scale;
    } else {
      // channels 8 (p & 1) + .. of the low (p < 2) or the high 16: the first four bytes by the one, the others by the other
      uint8_t* to = c.v4 + tile * (PAGE * DH / 2);
      const uint32_t lo = p < 2 ? w : other, hi = p < 2 ? other : w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = (p < 2 ? 0 : 4) + e;
        to[v_code_at<DH>(t, g, 8 * (p & 1) + n)] = (uint8_t)((lo >> 4 * n & 15) | (hi >> 4 * n & 15) << 4);
      }
      if (p == 0) c.vs[tile * (PAGE * DH / 32) + v_scale_at<DH>(t, g)] = (uint8_t)scale;
    }
  }
}

// 8 codes, two a byte -> bf16. The instruction takes the exponent of its scale operand alone; 255 gives NaN.
__device__ __forceinline__ v4i decode8(uint32_t w, float scale) {
  return v4i{(int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
             (int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
             (int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
             (int)__builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

template <int DH>
__global__ __launch_bounds__(THREADS) void kv4_read_kernel(Pages c, uint16_t* k, uint16_t* v) {
  constexpr int LANES = DH / 8;
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)group_id() * (THREADS / 64) + (threadIdx.x >> 6);
  if (r >= c.rows) return;
  const Token at = token_of(c, r);
  const int64_t page = page_of(c, at.seq, at.pos);
  const int t = (int)(at.pos % PAGE), c8 = lane % LANES, g = c8 >> 2, p = c8 & 3;
  for (int64_t i = lane / LANES; i < 2 * c.heads; i += 64 / LANES) {
    const bool is_k = i < c.heads;
    const int64_t h = is_k ? i : i - c.heads, tile = page * c.heads + h;
    v4i x = {0, 0, 0, 0};
    if (page >= 0 && is_k) {
      x = decode8(*(const uint32_t*)(c.k4 + (tile * PAGE + t) * (DH / 2) + p * (DH / 8) + g * 4), scale_of(c.ks[(tile * PAGE + t) * (DH / 32) + g]));
    } else if (page >= 0) {
      const uint8_t* from = c.v4 + tile * (PAGE * DH / 2);
      uint32_t w = 0;
#pragma unroll
      for (int n = 0; n < 8; ++n) w |= (uint32_t)(from[v_code_at<DH>(t, g, 8 * (p & 1) + n)] >> (p < 2 ? 0 : 4) & 15) << 4 * n;
      x = decode8(w, scale_of(c.vs[tile * (PAGE * DH / 32) + v_scale_at<DH>(t, g)]));
    }
    *(v4i*)((is_k ? k : v) + (r * c.heads + h) * DH + 8 * c8) = x;
  }
}

// ---------------------------------------------------------------- attention

constexpr int KB = 32, WAVES = THREADS / 64;   // keys of a wave's step

struct AttnArgs {
  Pages c;
  const uint16_t* q;
  int64_t q_tok, q_head;
  int q_heads, group, row_tiles;    // row_tiles: workgroups that share the heads of a group where those of one token are too many
  int tokens;                       // tokens of a workgroup's rows
  uint32_t places;
  int chunk, splits;                // keys of a workgroup; workgroups of a row's keys (1: no partial sums)
  float sl2;
  uint16_t* out;
  float *part, *stats;              // [rows][q_heads][splits][DH], [..][2]: sums, and the maximum and sum of the weights
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

// A workgroup: up to 16 RT rows (tokens x the heads that share a head of the cache) over a chunk of keys, 32 keys a wave and
// step. S^T = K Q^T on v_mfma_f32_16x16x32_bf16: a lane holds one row and 8 of the 32 keys; the row's maximum needs two
// exchanges; P^T goes from those registers into O^T += V^T P^T. fp16 q and P enter as two bf16 values each, high and low.
template <int DH, bool F16, int RT>
__global__ __launch_bounds__(THREADS) void kv4_attn_kernel(AttnArgs a) {
  constexpr int G = DH / 32, NT = DH / 16;
  __shared__ __align__(16) float part[WAVES][16][DH + 4];
  __shared__ float stats[WAVES][16][2];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, p = lane >> 4;
  const uint32_t id = group_id();
  uint32_t split = id % a.splits, rest = id / a.splits;
  const uint32_t row_tile = rest % a.row_tiles;
  rest /= a.row_tiles;
  const uint32_t head = rest % a.c.heads, at = rest / a.c.heads;
  if (at >= a.places) return;
  if (a.splits == 1 && a.c.starts && row_tile == 0)
    zero_outside(a.c.starts, a.c.seqs, a.c.rows, a.out + (int64_t)head * a.group * DH, (int64_t)a.q_heads * DH, a.group * DH, at, a.places);
  // the sequence, its rows in the call, and the first of this workgroup's tokens
  int64_t seq = at, first = at;
  int count = 1, token0 = 0;
  if (a.c.starts) {
    const Place pl = place(a.c.starts, a.c.seqs, a.c.rows, a.tokens, at);
    if (pl.seq < 0) return;
    const Span s = span(a.c.starts, pl.seq, a.c.rows);
    seq = pl.seq, first = s.first, count = s.n, token0 = pl.tile * a.tokens;
  }
  const int64_t len = min(max((int64_t)a.c.lens[seq], (int64_t)0), a.c.width * PAGE);
  // row i of the workgroup: token token0 + i / group, head i % group of the group (heads from row_tile on where they are many)
  const int group0 = row_tile * 16 * RT, heads_here = min(a.group - group0, a.row_tiles > 1 ? 16 * RT : a.group);
  const int rows = min(a.tokens, count - token0) * heads_here;
  const int64_t seen = len - count + token0 + 1;   // keys that the first token sees
  const int upto = (int)max((int64_t)0, min(len, seen + min(a.tokens, count - token0) - 1));
  const int k0 = split * a.chunk, k1 = min(upto, k0 + a.chunk);
  if (a.splits > 1 && k0 >= len) return;   // (nobody reads its part)

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
  // the pages of the chunk (64 at most), one a lane
  const int page0 = k0 / PAGE;
  int64_t held = -1;
  if (page0 + lane < a.c.width && (int64_t)(page0 + lane) * PAGE < k1) held = page_of(a.c, seq, (int64_t)(page0 + lane) * PAGE);
  const int mine = (int)held;

  for (int key = k0 + w * KB; key < k1; key += WAVES * KB) {
    const int page = __builtin_amdgcn_readlane(mine, key / PAGE - page0);
    if (page < 0) continue;
    Step<DH> st;
    st.load(a.c, (int64_t)page * a.c.heads + head, key / KB & 1, lane);
    v4i kf[2][G], vf[G][2];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < G; ++j) kf[x][j] = decode8(st.k[x][j], scale_of(st.ks[x] >> 8 * j & 255));
    // Some row may not see all of these keys: those behind the last hold what they like, and a NaN must not reach the rows
    // that do not see it through a weight of zero.
    const bool edge = key + KB > seen;
    bool odd = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      uint32_t two[8];   // channel 32 g + n low, 32 g + 16 + n high, of the lane's 8 keys
#define LBW_KEY(e)                                                                                                         \
  {                                                                                                                        \
    uint32_t b = st.vs[g][e >> 2] >> 8 * (e & 3) & 255;                                                                    \
    if (edge && key + 16 * (e >> 2) + 4 * p + (e & 3) >= seen && (b == 255 || key + 16 * (e >> 2) + 4 * p + (e & 3) >= k1)) {   \
      odd = odd || key + 16 * (e >> 2) + 4 * p + (e & 3) < k1;                                                             \
      b = 127;                                                                                                             \
    }                                                                                                                      \
    two[e] = __builtin_bit_cast(uint32_t, (bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(st.v[g][e >> 2], scale_of(b), e & 3)); \
  }
      LBW_KEY(0) LBW_KEY(1) LBW_KEY(2) LBW_KEY(3) LBW_KEY(4) LBW_KEY(5) LBW_KEY(6) LBW_KEY(7)
#undef LBW_KEY
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vf[g][0][e] = (int)__builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x05040100u);
        vf[g][1][e] = (int)__builtin_amdgcn_perm(two[2 * e + 1], two[2 * e], 0x07060302u);
      }
    }
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
      v4i ph, pl;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = __builtin_amdgcn_exp2f(fmaf(s[x][i], a.sl2, off));
        total[rt] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t hi = pack2<LBW_DTYPE_BF16>(pr[2 * i], pr[2 * i + 1]);
          ph[2 * x + i] = (int)hi;
          if constexpr (F16) pl[2 * x + i] = (int)pack2<LBW_DTYPE_BF16>(pr[2 * i] - lo16<false>(hi), pr[2 * i + 1] - hi16<false>(hi));
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          o[rt][2 * g + x] = mfma16(vf[g][x], ph, o[rt][2 * g + x]);
          if constexpr (F16) o[rt][2 * g + x] = mfma16(vf[g][x], pl, o[rt][2 * g + x]);
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

  // the waves' sums, a tile of 16 rows at a time: O^T's lane (p, n) holds channels 16 i + 4 p .. + 4 of row n
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (rt * 16 >= rows) break;
    if (rt) __syncthreads();
#pragma unroll
    for (int i = 0; i < NT; ++i) *(v4f*)&part[w][n][16 * i + 4 * p] = o[rt][i];
    const float sum = sum_quarters(total[rt]);
    if (p == 0) stats[w][n][0] = top[rt], stats[w][n][1] = sum;
    __syncthreads();
    constexpr int PER = 16 * DH / THREADS, LANES = DH / PER;   // channels of a thread
    const int row = threadIdx.x / LANES, c0 = (threadIdx.x % LANES) * PER, i = rt * 16 + row;
    if (i < rows) {
      float most = -INFINITY, sums = 0.f, x[PER] = {};
#pragma unroll
      for (int v = 0; v < WAVES; ++v) most = fmaxf(most, stats[v][row][0]);
#pragma unroll
      for (int v = 0; v < WAVES; ++v) {
        const float by = stats[v][row][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(stats[v][row][0] - most);
        sums = fmaf(by, stats[v][row][1], sums);
#pragma unroll
        for (int e = 0; e < PER; ++e) x[e] = fmaf(by, part[v][row][c0 + e], x[e]);
      }
      const int tok = i / heads_here, h = i - tok * heads_here;
      const int64_t r = (first + token0 + tok) * a.q_heads + (int64_t)head * a.group + group0 + h;
      if (a.splits == 1) {
        const float inv = sums > 0.f || sums != sums ? 1.f / sums : 0.f;
#pragma unroll
        for (int e = 0; e < PER; e += 2)
          *(uint32_t*)(a.out + r * DH + c0 + e) = pack2<F16 ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16>(x[e] * inv, x[e + 1] * inv);
      } else {
#pragma unroll
        for (int e = 0; e < PER; e += 4) *(v4f*)(a.part + (r * a.splits + split) * DH + c0 + e) = v4f{x[e], x[e + 1], x[e + 2], x[e + 3]};
        if (c0 == 0) a.stats[(r * a.splits + split) * 2] = most, a.stats[(r * a.splits + split) * 2 + 1] = sums;
      }
    }
  }
}

// The chunks of a row's keys joined: a wave a row and head, DH / 64 channels a lane.
template <int DH, bool F16>
__global__ __launch_bounds__(THREADS) void kv4_join_kernel(AttnArgs a) {
  constexpr int PER = DH / 64;
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)group_id() * WAVES + (threadIdx.x >> 6);
  if (i >= a.c.rows * a.q_heads) return;
  int64_t seq = i / a.q_heads;
  if (a.c.starts) {
    seq = last_of(a.c.seqs + 1, seq, [&](int64_t s) { return (int64_t)a.c.starts[s]; });
    if (seq >= a.c.seqs) seq = -1;
  }
  const int64_t len = seq < 0 ? 0 : min(max((int64_t)a.c.lens[seq], (int64_t)0), a.c.width * PAGE);
  const int parts = (int)((len + a.chunk - 1) / a.chunk);
  float most = -INFINITY, sums = 0.f, x[PER] = {};
  for (int s = 0; s < parts; ++s) most = fmaxf(most, a.stats[(i * a.splits + s) * 2]);
  for (int s = 0; s < parts; ++s) {
    const float m = a.stats[(i * a.splits + s) * 2], by = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - most);
    sums = fmaf(by, a.stats[(i * a.splits + s) * 2 + 1], sums);
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = fmaf(by, a.part[(i * a.splits + s) * DH + lane * PER + e], x[e]);
  }
  const float inv = sums > 0.f || sums != sums ? 1.f / sums : 0.f;
  if constexpr (PER == 2) *(uint32_t*)(a.out + i * DH + 2 * lane) = pack2<F16 ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16>(x[0] * inv, x[1] * inv);
  else store1<F16 ? LBW_DTYPE_FP16 : LBW_DTYPE_BF16>(a.out, i * DH + lane, x[0] * inv);
}

// How a call's work is cut: 16-row tiles of a workgroup, tokens of its rows, workgroups for a group's heads, keys of a chunk.
struct Plan {
  int rt, tokens, row_tiles, chunk, splits;
  int64_t places;
};
Plan plan(int64_t seqs, int64_t rows, int64_t group, int64_t heads, bool single, int64_t width) {
  Plan p;
  const int64_t each = single ? group : group * ((rows + seqs - 1) / seqs);   // rows of a sequence, about
  p.rt = each <= 16 ? 1 : each <= 32 ? 2 : 4;
  p.tokens = (int)std::max<int64_t>(1, 16 * p.rt / group);
  p.row_tiles = (int)((group + 16 * p.rt - 1) / (16 * p.rt));
  p.places = single ? seqs : places_of(rows, seqs, p.tokens);
  const int64_t keys = width * PAGE, base = std::max<int64_t>(1, std::min(p.places, rows) * heads * p.row_tiles);
  int64_t chunk = (keys * base / 2048 + 127) / 128 * 128;
  chunk = std::min<int64_t>(std::max<int64_t>(chunk, 128), 4096 - PAGE);
  p.chunk = (int)chunk;
  p.splits = (int)std::max<int64_t>(1, (keys + chunk - 1) / chunk);
  return p;
}

template <int DH, bool F16>
void launch_attn(const AttnArgs& a, int rt, hipStream_t stream) {
  const dim3 grid = grid_of((int64_t)a.places * a.c.heads * a.row_tiles * a.splits);
  if (rt == 1) kv4_attn_kernel<DH, F16, 1><<<grid, THREADS, 0, stream>>>(a);
  else if (rt == 2) kv4_attn_kernel<DH, F16, 2><<<grid, THREADS, 0, stream>>>(a);
  else kv4_attn_kernel<DH, F16, 4><<<grid, THREADS, 0, stream>>>(a);
  if (a.splits > 1) kv4_join_kernel<DH, F16><<<grid_of((a.c.rows * a.q_heads + WAVES - 1) / WAVES), THREADS, 0, stream>>>(a);
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
  const dim3 grid = grid_of((rows + 3) / 4);
  const uint16_t *kp = (const uint16_t*)k, *vp = (const uint16_t*)v;
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (dim == 128) {
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
  const dim3 grid = grid_of((rows + 3) / 4);
  if (dim == 128) kv4_read_kernel<128><<<grid, THREADS, 0, (hipStream_t)stream>>>(c, (uint16_t*)k, (uint16_t*)v);
  else kv4_read_kernel<64><<<grid, THREADS, 0, (hipStream_t)stream>>>(c, (uint16_t*)k, (uint16_t*)v);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

extern "C" int64_t lbw_kv4_attn_workspace_bytes(int64_t seqs, int64_t rows, int64_t q_heads, int64_t heads, int64_t dim, int64_t width,
                                                int single) {
  if (seqs < 1 || rows < 1 || heads < 1 || q_heads < heads) return 0;
  const Plan p = plan(seqs, rows, q_heads / heads, heads, single, width);
  return p.splits > 1 ? rows * q_heads * p.splits * (dim + 2) * 4 : 0;
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
  const Plan p = plan(seqs, rows, q_heads / heads, heads, !starts, width);
  if (p.places * heads * p.row_tiles * p.splits > 1 << 30 || rows * q_heads > 1ll << 31) return LBW_E_SHAPE;
  if (p.splits > 1 && !workspace) return LBW_E_NULL;
  if (!aligned(q, q_s_tok, q_s_head) || ((uintptr_t)out | (uintptr_t)workspace) % 16) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  float* part = (float*)workspace;
  const AttnArgs a = {{(uint8_t*)k4, (uint8_t*)ks, (uint8_t*)v4, (uint8_t*)vs, heads, pages, width, t_s_seq, seqs, rows, starts, lens, table},
                      (const uint16_t*)q, q_s_tok, q_s_head, (int)q_heads, (int)(q_heads / heads), p.row_tiles, p.tokens,
                      (uint32_t)p.places, p.chunk, p.splits, sm_scale * LOG2E, (uint16_t*)out, part,
                      part ? part + rows * q_heads * p.splits * dim : nullptr};
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (dim == 128) f16 ? launch_attn<128, true>(a, p.rt, (hipStream_t)stream) : launch_attn<128, false>(a, p.rt, (hipStream_t)stream);
  else f16 ? launch_attn<64, true>(a, p.rt, (hipStream_t)stream) : launch_attn<64, false>(a, p.rt, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
