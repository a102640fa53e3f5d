// Gradients of attention over packed sequences (include/lbw_causal.h), from S formed again: with P = exp2(S - lse) and
// D = rowsum(dO o),
//   dV = P^T dO,   dS = P (dO V^T - D),   dQ = scale dS K,   dK = scale dS^T Q.
//
// Three kernels: D; dK and dV, a workgroup for a tile of keys, which walks the queries of every head that shares them; dQ, a
// workgroup for a tile of queries, which walks the keys. S and dO V^T are formed in both (7 products for 5), so that no
// sum needs atomics: each has one order, whatever runs beside it.
//
// 5 sequences of up to 1508, 12 heads of 128 over 4: D 7.6 us, dK and dV 79, dQ 45, the forward 39. dK and dV take one wave a SIMD
// (their sums are 128 registers a lane, K and V of the keys 64), whose products, exponentials and scalar work follow one
// another: the longest workgroup's 36 steps of 128 queries are what the call waits for, 2.2 us each.
#include "lbw_packed.h"

namespace lbw {
namespace packed {

int check(int dtype, int64_t seqs, int64_t q_rows, int64_t k_rows, int64_t q_heads, int64_t k_heads, int64_t dim, float sm_scale);
bool aligned(const void* p, int64_t tok, int64_t head, int64_t dim);

namespace {

constexpr int WAVES = 4, THREADS = 64 * WAVES;

struct BwdArgs {
  Shape s;
  const uint16_t *dout, *out, *rest, *q, *k, *v;
  int64_t do_tok, do_head, q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const float* lse;
  float* delta;
  uint16_t *dq, *dk, *dv;
  uint32_t tiles;
};

// D of every row and head: a row by 16 (8) lanes. The output is taken with the rest of its rounding: without it D is off by
// 2^-9 of the row, the same way for each of its keys, which keys with a common part add up (dQ of sequences of up to 133: 1.2 to
// 2.4 times as far from 64 bits as that of the plain products in the type, against 0.9 to 1.2).
template <int DH, bool F16>
__global__ __launch_bounds__(THREADS) void packed_delta_kernel(BwdArgs a) {
  constexpr int LANES = DH / 8;
  const int64_t i = ((int64_t)group_id() * THREADS + threadIdx.x) / LANES;
  if (i >= a.s.q_rows * a.s.q_heads) return;
  const int64_t row = i / a.s.q_heads, head = i - row * a.s.q_heads;
  const int c = (threadIdx.x % LANES) * 8;
  float x[8], y[8], z[8], sum = 0.f;
  unpack8t<F16>(*(const v4i*)(a.dout + row * a.do_tok + head * a.do_head + c), x);
  unpack8t<F16>(*(const v4i*)(a.out + i * DH + c), y);
  unpack8t<F16>(*(const v4i*)(a.rest + i * DH + c), z);
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(x[e], y[e] + z[e], sum);
  sum += dpp<DPP_XOR1>(sum);
  sum += dpp<DPP_XOR2>(sum);
  sum += dpp<DPP_HALF_MIRROR>(sum);
  if constexpr (LANES == 16) sum += dpp<DPP_MIRROR>(sum);
  if (c == 0) a.delta[head * a.s.q_rows + row] = sum;
}

// dS in fp16 may leave that type's range in either direction. Each lane (a query, or a key) holds its values times a power
// of two of its own, so that the largest so far lies in [2^8, 2^14) (lower where that power would have to pass 2^126), and its
// sums with the same factor: `by` is what they have to be multiplied by when it changes (seldom; 1 else).
struct Range {
  float scale = 1.f;
  bool set = false;
  __device__ __forceinline__ bool fit(const v16f& ds, float& by) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(ds[i]));
    m = max_xor32(m);
    by = 1.f;
    if (m > 0.f && m < INFINITY && (!set || m * scale >= 16384.f)) {
      // 2^8 to 2^9 for now: a few binades up before the next change
      const float next = ldexpf(1.f, max(-126, min(126, 8 - (int)(__float_as_uint(m) >> 23) + 127)));
      if (set) by = next / scale;
      scale = next;
      set = true;
    }
    return __any(by != 1.f);
  }
};

// log2 of a weight, as it is held (LIFT): s sl2 - lse.
template <bool F16>
__device__ __forceinline__ float weight_exponent(float s, float sl2, float lse) {
  return F16 ? fmaf(s, sl2, LIFT<F16> - lse) : fmaf(s, sl2, -lse);
}

template <int MT>
__device__ __forceinline__ void times(v16f (&o)[MT], float by) {
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[mt][i] *= by;
}

template <bool F16>
__device__ __forceinline__ void pack16(const v16f& x, float scale, v4i (&f)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) f[u][e] = (int)pack<F16>(x[8 * u + 2 * e] * scale, x[8 * u + 2 * e + 1] * scale);
}

// What that rounding took off, rounded.
template <bool F16>
__device__ __forceinline__ void pack16_rest(const v16f& x, float scale, const v4i (&f)[2], v4i (&rest)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      rest[u][e] = (int)pack<F16>(fmaf(x[8 * u + 2 * e], scale, -lo16<F16>((uint32_t)f[u][e])), fmaf(x[8 * u + 2 * e + 1], scale, -hi16<F16>((uint32_t)f[u][e])));
}
// dS adds up to zero over a query's keys and its roundings do not, which the common part of K's rows makes a part of dQ: in one
// part dQ is 1.54 to 1.72 times as far from 64 bits as that of the plain products (dK 1.41 to 1.63), in two, each rounded, 0.9 to
// 1.2. dQ has two always (167 to 172 us for a training step of 4096 tokens, 12 heads over 4); dK where the sequence is so
// short that the roundings do not average out.
constexpr int SHORT = 128;

// ---------------------------------------------------------------- dK, dV

// A workgroup takes 32 KW keys, 32 a wave, and its QW = 4 / KW waves of the same keys take every QW-th 32 queries, their sums
// added at the end: with 128 keys a stage's queries serve four waves, with 32 there are four times as many workgroups, each a
// quarter as long. There no two waves share queries: each brings its own, two stages ahead of the barriers that the others
// need, and has read the next queries from LDS before the products of these are done.
template <int DH, bool F16, int KW>
__global__ __launch_bounds__(THREADS, DH == 128 ? 1 : 2) void packed_dkv_kernel(BwdArgs a) {
  constexpr bool ALONE = KW == 1;
  constexpr int QW = WAVES / KW, QR = ALONE ? 32 : 64, SUB = ALONE ? 1 : QR / 32 / QW;   // queries of a stage; 32s of a wave in it
  constexpr int NS = DH / 16, MT = DH / 32, KT = 32 * KW, TILE = QR * row_bytes<DH>, STAGE = 2 * TILE + 2 * 64 * 4;
  // (the loads of a stage take longer than its products where memory is far)
  constexpr int STAGES = ALONE ? 2 : 4, RINGS = ALONE ? WAVES : 1, LOADERS = ALONE ? 1 : WAVES;
  constexpr int SUMS = (WAVES - KW) * 2 * MT * 16 * 64 * 4;   // LDS bytes of the sums of all waves but the first of each 32 keys
  constexpr int LDS = std::max(std::max(RINGS * STAGES * STAGE, WAVES * STAGING<DH>), SUMS);
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ int odd[WAVES];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kw = w % KW, qw = QW > 1 ? w / KW : 0;
  uint32_t head, tile;
  head_tile(group_id(), a.s.k_heads, 1, a.s.common, head, tile);
  if (tile >= a.tiles) return;
  const int64_t o_tok = (int64_t)a.s.k_heads * DH;
  const Where at = where(a.s.k_starts, a.s.starts, a.s.seqs, a.s.k_rows, a.s.q_rows, KT, tile);
  zero_outside(at.begin, at.end, a.s.k_rows, a.dk + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  zero_outside(at.begin, at.end, a.s.k_rows, a.dv + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  if (at.seq < 0) return;
  const Span qs = at.other, ks = at.own;
  const int n = qs.n, m = ks.n, shift = m - n;
  const int k0 = (at.tiles - 1 - at.tile) * KT, key0 = k0 + 32 * kw, key = key0 + (lane & 31);   // (the first keys have the most queries)
  // the first query that sees a key, and the stage it lies in
  const auto first = [&](int j) { return a.s.causal ? max(0, j - shift) : 0; };
  const int q_stage = first(k0) / QR, stages = max(0, (n + QR - 1) / QR - q_stage), each = ALONE ? WAVES : 1;
  const int own = first(key), w_first = first(key0), w_all = first(key0 + 31);
  const bool fine = min(n, m) <= SHORT;

  v4i kf[NS], vf[NS];
  load_rows<DH>(a.k + (ks.first + key0) * a.k_tok + head * a.k_head, a.k_tok, m - key0, lane, kf);
  load_rows<DH>(a.v + (ks.first + key0) * a.v_tok + head * a.v_head, a.v_tok, m - key0, lane, vf);
  const int loader = ALONE ? 0 : w;
  Loader<DH, QR, LOADERS> ql, dl;
  ql.init(loader, lane, a.q_tok);
  dl.init(loader, lane, a.do_tok);
  arrived(kf);
  arrived(vf);
  // of all heads' stages one behind the other: each, or (ALONE) every fourth from the wave's number on
  const int steps = ALONE ? max(0, (stages * a.s.group - w + WAVES - 1) / WAVES) : stages * a.s.group;
  // What is loaded next: a head's queries from r on. Pointers that move on by a stage: made from the numbers each time, the
  // scalar unit would take as long as the products.
  const uint16_t *q_next, *d_next;
  const float* stat_next;
  int g_next, r_next;
  const auto queries_from = [&](int r) {   // of head g_next, or of one behind it
    while (r >= stages * QR) r -= stages * QR, ++g_next;
    const int64_t h = (int64_t)head * a.s.group + g_next;
    r_next = q_stage * QR + r;
    q_next = a.q + (qs.first + r_next) * a.q_tok + h * a.q_head;
    d_next = a.dout + (qs.first + r_next) * a.do_tok + h * a.do_head;
    stat_next = (w == 0 || ALONE ? a.lse : a.delta) + h * a.s.q_rows + qs.first + r_next;
  };
  const auto restart = [&] {
    g_next = 0;
    if (steps > 0) queries_from(ALONE ? w * QR : 0);
  };
  restart();
  const int64_t to_delta = a.delta - a.lse;
  const int end = (q_stage + stages) * QR;
  uint8_t* ring = lds + (ALONE ? w * STAGES * STAGE : 0);
  const auto issue = [&](int stage) __attribute__((always_inline)) {
    uint8_t* to = ring + stage * STAGE;
    ql.issue(rows_buffer<DH>(q_next, a.q_tok, n - r_next, QR), loader, to);
    dl.issue(rows_buffer<DH>(d_next, a.do_tok, n - r_next, QR), loader, to + TILE);
    // (64 values a load: of the sums, then of D; one for each of the first two waves, where they share)
    if (ALONE || w < 2) dma4(stat_next, n - r_next, lane * 4, to + 2 * TILE + (ALONE ? 0 : w * 256));
    if (ALONE) dma4(stat_next + to_delta, n - r_next, lane * 4, to + 2 * TILE + 256);
    r_next += each * QR;
    q_next += each * QR * a.q_tok;
    d_next += each * QR * a.do_tok;
    stat_next += each * QR;
    if (r_next >= end) {
      const int over = r_next - end;
      ++g_next;
      queries_from(over);
    }
  };
  RowReads<DH> rr;
  TurnedReads<DH> tr;
  rr.init(lane);
  tr.init(lane);
  v16f dk[MT], dv[MT];
  Range range;

  // The sums stay in the accumulation registers: the compiler would move them to the others and back, 256 moves a step.
  const auto stay = [&] {
    if constexpr (DH == 128) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) asm volatile("" : "+a"(dk[mt]), "+a"(dv[mt]));
    }
  };
  v4i qa[NS], da[NS];
  // (reads in one go ahead of the products that use them: the compiler would wait for each by itself)
  const auto read = [&](const uint8_t* qt, int x) __attribute__((always_inline)) {
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      qa[st] = rr.get(qt, x, st);
      da[st] = rr.get(qt + TILE, x, st);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // The 32 queries r .. + 32, x-th of the stage at qt, once read; meanwhile() runs when everything else of them is read.
  const auto work = [&](const uint8_t* qt, int x, int r, auto again, const auto& meanwhile) __attribute__((always_inline)) {
    const uint8_t* dt = qt + TILE;
    v16f s = zeros16(), dp = zeros16();
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      s = mfma<F16>(qa[st], kf[st], s);
      dp = mfma<F16>(da[st], vf[st], dp);
    }
    __builtin_amdgcn_sched_barrier(0);
    v4i td[2][MT], tq[2][MT];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) td[u][mt] = tr.get(dt, 2 * x + u, mt);
    const float* stats = (const float*)(qt + 2 * TILE) + 32 * x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 l = *(const float4*)(stats + 8 * i + 4 * hf), d = *(const float4*)(stats + 64 + 8 * i + 4 * hf);
      const float le[4] = {l.x, l.y, l.z, l.w}, de[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(weight_exponent<F16>(s[4 * i + e], a.s.sl2, le[e]));
        s[4 * i + e] = p;
        dp[4 * i + e] = p * (dp[4 * i + e] - de[e]);
      }
    }
    // queries that do not see a key; rows behind the last query are zeros, but a key that is not finite makes NaN of them
    const bool partly = r < w_all || r + 32 > n;
    if (partly) {
      branch_here();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (const int row = r + 8 * (i >> 2) + 4 * hf + (i & 3); row < own || row >= n) s[i] = dp[i] = 0.f;
    }
    v4i pf[2], df[2];
    pack16<F16>(s, 1.f, pf);
    float by;
    if constexpr (F16) {
      if (range.fit(dp, by)) times(dk, by);
    }
    pack16<F16>(dp, range.scale, df);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) tq[u][mt] = tr.get(qt, 2 * x + u, mt);
    if (decltype(again)::value && partly) {   // (a query that is not finite has weights that are not)
      branch_here();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          td[u][mt] = clean<F16>(td[u][mt]);
          tq[u][mt] = clean<F16>(tq[u][mt]);
        }
      add_odd<DH, F16>(dv, dt, x, hf, [&](int j) { return r + j >= own; });
    }
    __builtin_amdgcn_sched_barrier(0);
    meanwhile();
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) dv[mt] = mfma<F16>(td[u][mt], pf[u], dv[mt]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) dk[mt] = mfma<F16>(tq[u][mt], df[u], dk[mt]);
    if (fine) {
      branch_here();
      v4i rest[2];
      pack16_rest<F16>(dp, range.scale, df, rest);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) dk[mt] = mfma<F16>(tq[u][mt], rest[u], dk[mt]);
    }
  };
  const auto pass = [&](auto again) __attribute__((always_inline)) {
    range = Range();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) dk[mt] = dv[mt] = zeros16();
    if constexpr (ALONE) {
      constexpr int LOADS = 2 * Loader<DH, QR, LOADERS>::N + 2;
      int r = w * QR;   // from the first stage's start on
      if (steps > 0) {
        while (r >= stages * QR) r -= stages * QR;
        issue(0);
        if (steps > 1) issue(1);
        wait_dma_but<LOADS>(steps > 1);
        asm volatile("" ::: "memory");
        if constexpr (!decltype(again)::value) read(ring, 0);
      }
      for (int step = 0; step < steps; ++step) {
        const uint8_t* here = ring + (step & 1) * STAGE;
        const auto next = [&]() __attribute__((always_inline)) {
          if (step + 1 < steps) {
            // (lgkmcnt(0): the wave has these queries in registers, and the stage is free)
            __builtin_amdgcn_s_waitcnt(0xC07F);
            asm volatile("" ::: "memory");
            if (step + 2 < steps) issue(step & 1);
            wait_dma_but<LOADS>(step + 2 < steps);
            asm volatile("" ::: "memory");
          }
        };
        stay();
        if constexpr (decltype(again)::value) {   // (few registers rather than speed)
          read(here, 0);
          work(here, 0, q_stage * QR + r, again, [] {});
          next();
        } else {
          work(here, 0, q_stage * QR + r, again, [&]() __attribute__((always_inline)) {
            next();
            if (step + 1 < steps) read(ring + (1 - (step & 1)) * STAGE, 0);
          });
        }
        r += WAVES * QR;
        while (r >= stages * QR) r -= stages * QR;
        stay();
      }
    } else {
      for (int i = 0; i < min(STAGES - 1, steps); ++i) issue(i);
      for (int step = 0, here = q_stage * QR; step < steps; ++step, here = here + QR < n ? here + QR : q_stage * QR) {
        const int stage = step % STAGES;
        const uint8_t* qt = ring + stage * STAGE;
        stay();
        const int ahead = min(STAGES - 2, steps - 1 - step);
        if (w < 2) wait_dma_but<2 * Loader<DH, QR, LOADERS>::N + 1>(ahead);
        else wait_dma_but<2 * Loader<DH, QR, LOADERS>::N>(ahead);
        __syncthreads();   // the stage is in LDS, and every wave is done with the one before it
        if (step + STAGES - 1 < steps) issue((step + STAGES - 1) % STAGES);
#pragma unroll 1
        for (int i32 = 0; i32 < SUB; ++i32) {
          const int x = i32 * QW + qw, r = here + 32 * x;
          if (r >= n || r + 31 < w_first) continue;
          read(qt, x);
          work(qt, x, r, again, [] {});
        }
        stay();
      }
    }
  };
  pass(ic<0>{});
  const bool bad = any_odd(dk) | any_odd(dv);
  if (lane == 0) odd[w] = bad;
  __syncthreads();   // every wave is done with the stages
  if (__builtin_expect(a.s.causal && __builtin_amdgcn_readfirstlane(odd[0] | odd[1] | odd[2] | odd[3]), 0)) {
    restart();
    pass(ic<1>{});
    __syncthreads();
  }
  const float lift = __builtin_amdgcn_exp2f(-LIFT<F16>);
  float k_by = a.s.scale * lift / range.scale;
  if constexpr (QW > 1) {   // the sums of the other waves of these keys, in their order
    float* sums = (float*)lds + lane;
    if (qw) {
      float* mine = sums + (w - KW) * (2 * MT * 16 * 64);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          mine[(mt * 16 + i) * 64] = dk[mt][i] * k_by;
          mine[((MT + mt) * 16 + i) * 64] = dv[mt][i];
        }
    }
    __syncthreads();
    if (qw) return;
    times(dk, k_by);
    k_by = 1.f;
    for (int q = 1; q < QW; ++q) {
      const float* other = sums + (q * KW + kw - KW) * (2 * MT * 16 * 64);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          dk[mt][i] += other[(mt * 16 + i) * 64];
          dv[mt][i] += other[((MT + mt) * 16 + i) * 64];
        }
    }
  }
  if (key0 >= m) return;
  // (staged where no other wave may still be reading: of the sums, those that it has read itself)
  static_assert(STAGING<DH> <= 2 * MT * 16 * 64 * 4, "a wave's staging lies inside the sums it reads");
  uint8_t* mine = lds + (QW > 1 ? kw * (2 * MT * 16 * 64 * 4) : w * STAGING<DH>);
  store_turned<DH, F16>(dk, k_by, mine, lane, a.dk + (ks.first + key0) * o_tok + head * DH, o_tok, m - key0);
  __builtin_amdgcn_wave_barrier();
  store_turned<DH, F16>(dv, lift, mine, lane, a.dv + (ks.first + key0) * o_tok + head * DH, o_tok, m - key0);
}

// ---------------------------------------------------------------- dQ

constexpr int KT = 64;

// QW and the waves that share queries as in the forward.
template <int DH, bool F16, int QW>
__global__ __launch_bounds__(THREADS, DH == 128 ? 2 : 4) void packed_dq_kernel(BwdArgs a) {
  constexpr int KW = WAVES / QW, QT = 32 * QW;
  static_assert(KW == 1 || KW == 2, "a tile has 64 keys");
  constexpr int NS = DH / 16, MT = DH / 32, TILE = KT * row_bytes<DH>, STAGE = 2 * TILE;
  constexpr int SUMS = KW > 1 ? QW * MT * 16 * 256 : 0;
  constexpr int LDS = std::max(2 * STAGE, std::max(WAVES * STAGING<DH>, SUMS));
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ int odd[WAVES];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qw = w % QW, kw = KW > 1 ? w / QW : 0;
  uint32_t head, tile;
  head_tile(group_id(), a.s.k_heads, a.s.group, a.s.common, head, tile);
  if (tile >= a.tiles) return;
  const int64_t o_tok = (int64_t)a.s.q_heads * DH;
  const Where at = where(a.s.starts, a.s.k_starts, a.s.seqs, a.s.q_rows, a.s.k_rows, QT, tile);
  zero_outside(at.begin, at.end, a.s.q_rows, a.dq + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  if (at.seq < 0) return;
  const Span qs = at.own, ks = at.other;
  const int n = qs.n, m = ks.n, shift = m - n, q0 = at.tile * QT;
  const int row0 = q0 + 32 * qw, row = row0 + (lane & 31);
  const auto seen = [&](int r) { return a.s.causal ? max(0, min(m, min(r, n - 1) + shift + 1)) : m; };
  const int upto = seen(q0 + QT - 1), w_upto = row0 < n ? seen(row0 + 31) : 0, w_first = seen(row0);
  const int tiles = (upto + KT - 1) / KT;

  const uint16_t *kb, *vb;
  int left;
  const auto from_start = [&] {
    kb = a.k + ks.first * a.k_tok + (head / a.s.group) * a.k_head;
    vb = a.v + ks.first * a.v_tok + (head / a.s.group) * a.v_head;
    left = m;
  };
  Loader<DH, KT, WAVES> kl, vl;
  kl.init(w, lane, a.k_tok);
  vl.init(w, lane, a.v_tok);
  const auto issue = [&](int stage) {   // the next tile
    kl.issue(rows_buffer<DH>(kb, a.k_tok, left, KT), w, lds + stage * STAGE);
    vl.issue(rows_buffer<DH>(vb, a.v_tok, left, KT), w, lds + stage * STAGE + TILE);
    kb += KT * a.k_tok;
    vb += KT * a.v_tok;
    left -= KT;
  };
  from_start();
  if (tiles > 0) issue(0);
  v4i qf[NS], df[NS];
  load_rows<DH>(a.q + (qs.first + row0) * a.q_tok + head * a.q_head, a.q_tok, n - row0, lane, qf);
  load_rows<DH>(a.dout + (qs.first + row0) * a.do_tok + head * a.do_head, a.do_tok, n - row0, lane, df);
  const int64_t stat = (int64_t)head * a.s.q_rows + qs.first + row;
  float lse = row < n ? a.lse[stat] : INFINITY, delta = row < n ? a.delta[stat] : 0.f;
  arrived(qf);
  arrived(df);
  asm volatile("" : "+v"(lse), "+v"(delta));
  RowReads<DH> rr;
  TurnedReads<DH> tr;
  rr.init(lane);
  tr.init(lane);
  v16f dq[MT];
  Range range;
  const auto pass = [&](auto again, int lane) __attribute__((always_inline)) {
    range = Range();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) dq[mt] = zeros16();
    for (int t = 0; t < tiles; ++t) {
      const int stage = t & 1;
      const uint8_t *kt = lds + stage * STAGE, *vt = kt + TILE;
      wait_dma();
      __syncthreads();
      if (t + 1 < tiles) issue(1 - stage);
#pragma unroll 1
      for (int x = kw; x < KT / 32; x += KW) {
        const int j0 = t * KT + 32 * x;
        if (j0 >= w_upto) continue;
        if constexpr (decltype(again)::value) {   // (read again rather than kept: the other pass has no registers to spare)
          load_rows<DH>(a.q + (qs.first + row0) * a.q_tok + head * a.q_head, a.q_tok, n - row0, lane, qf);
          load_rows<DH>(a.dout + (qs.first + row0) * a.do_tok + head * a.do_head, a.do_tok, n - row0, lane, df);
        }
        const int hf = lane >> 5, own = seen(row0 + (lane & 31));
        v16f s = zeros16(), dp = zeros16();
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          s = mfma<F16>(rr.get(kt, x, st), qf[st], s);
          dp = mfma<F16>(rr.get(vt, x, st), df[st], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] = __builtin_amdgcn_exp2f(weight_exponent<F16>(s[i], a.s.sl2, lse)) * (dp[i] - delta);
        const bool partly = j0 + 32 > w_first;   // keys that a query does not see
        if (partly) {
          branch_here();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (j0 + 8 * (i >> 2) + 4 * hf + (i & 3) >= own) dp[i] = 0.f;
        }
        v4i pf[2], rest[2], tk[2][MT];
        float by;
        if constexpr (F16) {
          if (range.fit(dp, by)) times(dq, by);
        }
        pack16<F16>(dp, range.scale, pf);
        pack16_rest<F16>(dp, range.scale, pf, rest);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) tk[u][mt] = tr.get(kt, 2 * x + u, mt);
        if (decltype(again)::value && partly) {
          branch_here();
          // a key that is not finite has weights that are not, where it is seen, or (its scores being minus infinity) zero
          add_odd<DH, F16, true>(dq, kt, x, hf, [&](int j) { return j0 + j < own; });
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) tk[u][mt] = clean<F16>(tk[u][mt]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) dq[mt] = mfma<F16>(tk[u][mt], pf[u], dq[mt]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) dq[mt] = mfma<F16>(tk[u][mt], rest[u], dq[mt]);
      }
    }
  };
  pass(ic<0>{}, lane);
  // (the lane's number again, unknown to the compiler: what it makes of it is not held in registers all through the loop)
  int late = threadIdx.x;
  asm volatile("" : "+v"(late));
  late &= 63;
  const bool bad = any_odd(dq);
  if (late == 0) odd[w] = bad;
  __syncthreads();   // every wave is done with the stages
  if (__builtin_expect(a.s.causal && __builtin_amdgcn_readfirstlane(odd[0] | odd[1] | odd[2] | odd[3]), 0)) {
    rr.init(late);
    tr.init(late);
    kl.init(w, late, a.k_tok);
    vl.init(w, late, a.v_tok);
    from_start();
    issue(0);   // (there is a tile: without one the sums are zeros)
    pass(ic<1>{}, late);
    __syncthreads();
  }
  float by = a.s.scale * __builtin_amdgcn_exp2f(-LIFT<F16>) / range.scale;
  if constexpr (KW > 1) {   // the same of the wave of the other keys
    float* other = (float*)lds + qw * (MT * 16) * 64 + late;
    if (kw) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) other[(mt * 16 + i) * 64] = dq[mt][i] * by;
    }
    __syncthreads();
    if (kw) return;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) dq[mt][i] = fmaf(dq[mt][i], by, other[(mt * 16 + i) * 64]);
    by = 1.f;
  }
  if (row0 >= n) return;
  static_assert(KW == 1 || STAGING<DH> <= MT * 16 * 256, "a wave's staging lies inside what it reads");
  store_turned<DH, F16>(dq, by, lds + (KW > 1 ? qw * MT * 16 * 256 : w * STAGING<DH>), late, a.dq + (qs.first + row0) * o_tok + head * DH,
                        o_tok, n - row0);
}

template <int DH, bool F16>
void launch(BwdArgs a, hipStream_t stream) {
  const int64_t rows = a.s.q_rows * a.s.q_heads;
  packed_delta_kernel<DH, F16><<<grid_of((rows * (DH / 8) + THREADS - 1) / THREADS), THREADS, 0, stream>>>(a);
  if (a.dk) {
    // As many keys a workgroup as leave two for every CU, or, where each is short, more than one (measured, us, for 128, 64 and
    // 32 keys: 32 heads over 8, 4 sequences of 1024: 175, 136, 162; one of 2048: 299, 185, 137; 12 over 12, one of 6000: 340, 353,
    // 395; 16 over 16, one of 1024: 52, 40, 46).
    const auto groups = [&](int keys) { return xcd_groups(places_of(a.s.k_rows, a.s.seqs, keys), a.s.k_heads, 1); };
    const bool brief = a.s.q_rows / a.s.seqs * a.s.group <= 1024;
    const int keys = groups(128) >= 512 ? 128 : groups(64) >= (brief ? 256 : 512) ? 64 : 32;
    a.tiles = (uint32_t)places_of(a.s.k_rows, a.s.seqs, keys);
    const dim3 grid = grid_of(groups(keys));
    if (keys == 128) packed_dkv_kernel<DH, F16, 4><<<grid, THREADS, 0, stream>>>(a);
    else if (keys == 64) packed_dkv_kernel<DH, F16, 2><<<grid, THREADS, 0, stream>>>(a);
    else packed_dkv_kernel<DH, F16, 1><<<grid, THREADS, 0, stream>>>(a);
  }
  if (a.dq) {
    const auto groups = [&](int queries) { return xcd_groups(places_of(a.s.q_rows, a.s.seqs, queries), a.s.k_heads, a.s.group); };
    // (us for 128 and 64 queries: 32 heads, one sequence of 2048, 544 workgroups of 128: 105, 99; of 4096: 283, 283; 16 of 256: 68, 78)
    const bool wide = groups(128) >= 1024;
    a.tiles = (uint32_t)places_of(a.s.q_rows, a.s.seqs, wide ? 128 : 64);
    if (wide) packed_dq_kernel<DH, F16, 4><<<grid_of(groups(128)), THREADS, 0, stream>>>(a);
    else packed_dq_kernel<DH, F16, 2><<<grid_of(groups(64)), THREADS, 0, stream>>>(a);
  }
}

}  // namespace
}  // namespace packed
}  // namespace lbw

using namespace lbw;

extern "C" int64_t lbw_packed_attn_bwd_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t q_heads, int64_t k_heads) {
  (void)k_rows, (void)k_heads;
  return q_rows * q_heads * 4;
}

extern "C" int lbw_packed_attn_bwd(const void* d_out, const void* out, const void* rest, const float* lse, const void* q, const void* k,
                                   const void* v, int dtype, int64_t seqs, int64_t q_rows, int64_t k_rows, int64_t q_heads,
                                   int64_t k_heads, int64_t dim, int64_t do_s_tok, int64_t do_s_head, int64_t q_s_tok,
                                   int64_t q_s_head, int64_t k_s_tok, int64_t k_s_head, int64_t v_s_tok, int64_t v_s_head,
                                   const int32_t* starts, const int32_t* k_starts, int causal, float sm_scale, void* dq,
                                   void* dk, void* dv, void* workspace, void* stream) {
  if (!d_out || !out || !rest || !lse || !q || !k || !v || !starts || !k_starts || !workspace || !dk != !dv) return LBW_E_NULL;
  if (const int st = packed::check(dtype, seqs, q_rows, k_rows, q_heads, k_heads, dim, sm_scale)) return st;
  if (!packed::aligned(d_out, do_s_tok, do_s_head, dim) || !packed::aligned(q, q_s_tok, q_s_head, dim) || !packed::aligned(k, k_s_tok, k_s_head, dim) ||
      !packed::aligned(v, v_s_tok, v_s_head, dim))
    return LBW_E_ALIGN;
  for (const void* p : {out, rest, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)workspace})
    if ((uintptr_t)p % 16) return LBW_E_ALIGN;
  if ((uintptr_t)starts % 4 || (uintptr_t)k_starts % 4 || (uintptr_t)lse % 4) return LBW_E_ALIGN;
  if (k_rows < 1 || (places_of(q_rows, seqs, 64) + 8) * q_heads > 1 << 30 || (places_of(k_rows, seqs, 32) + 8) * k_heads > 1 << 30 ||
      q_rows * q_heads * dim / 8 / packed::THREADS > 1 << 30)
    return LBW_E_SHAPE;
  if (const int st = check_device()) return st;
  packed::BwdArgs a = {{seqs, q_rows, k_rows, (int)q_heads, (int)k_heads, (int)(q_heads / k_heads), (int)packed::xcd_common(k_heads), starts, k_starts, causal,
                        sm_scale, sm_scale * packed::LOG2E},
                       (const uint16_t*)d_out, (const uint16_t*)out, (const uint16_t*)rest, (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v,
                       do_s_tok, do_s_head, q_s_tok, q_s_head, k_s_tok, k_s_head, v_s_tok, v_s_head, lse, (float*)workspace,
                       (uint16_t*)dq, (uint16_t*)dk, (uint16_t*)dv, 0};
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (dim == 128) f16 ? packed::launch<128, true>(a, (hipStream_t)stream) : packed::launch<128, false>(a, (hipStream_t)stream);
  else f16 ? packed::launch<64, true>(a, (hipStream_t)stream) : packed::launch<64, false>(a, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
