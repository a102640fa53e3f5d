// Gradients of attention over packed sequences (include/lbw_causal.h), from S formed again: with P = exp2(S - lse) and
// D = rowsum(dO o),
//   dV = P^T dO,   dS = P (dO V^T - D),   dQ = scale dS K,   dK = scale dS^T Q.
//
// Three kernels: D; dK and dV, a workgroup for a tile of keys, which walks the queries of every head that shares them; dQ, a
// workgroup for a tile of queries, which walks the keys. S and dO V^T are formed in both (7 products for 5), so that no
// sum needs atomics: each has one order, whatever runs beside it.
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
// 2^-9 of the row, the same way for each of its keys, which keys with a common part add up (dQ of such keys: 1.7 times as
// far from 64 bits as its own rounding, against 1.4).
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
// of two of its own, so that the largest so far lies in [2^4, 2^14), and its sums with the same factor: `by` is what they have to be
// multiplied by when it changes (seldom; 1 else).
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

// ---------------------------------------------------------------- dK, dV

constexpr int QR = 64;   // queries of a stage

template <int DH, bool F16>
__global__ __launch_bounds__(THREADS, DH == 128 ? 1 : 2) void packed_dkv_kernel(BwdArgs a) {
  constexpr int NS = DH / 16, MT = DH / 32, KT = 32 * WAVES, TILE = QR * row_bytes<DH>, STAGE = 2 * TILE + 2 * QR * 4;
  constexpr int LDS = 2 * STAGE > WAVES * STAGING<DH> ? 2 * STAGE : WAVES * STAGING<DH>;
  __shared__ __align__(16) uint8_t lds[LDS];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t head, tile;
  head_tile(group_id(), a.s.k_heads, head, tile);
  if (tile >= a.tiles) return;
  const int64_t o_tok = (int64_t)a.s.k_heads * DH;
  zero_outside(a.s.k_starts, a.s.seqs, a.s.k_rows, a.dk + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  zero_outside(a.s.k_starts, a.s.seqs, a.s.k_rows, a.dv + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  const Place at = place(a.s.k_starts, a.s.seqs, a.s.k_rows, KT, tile);
  if (at.seq < 0) return;
  const Span qs = span(a.s.starts, at.seq, a.s.q_rows), ks = span(a.s.k_starts, at.seq, a.s.k_rows);
  const int n = qs.n, m = ks.n, shift = m - n;
  const int k0 = at.tile * KT, key0 = k0 + 32 * w, key = key0 + (lane & 31);   // (the first keys have the most queries)
  // the first query that sees a key, and the stage it lies in
  const auto first = [&](int j) { return a.s.causal ? max(0, j - shift) : 0; };
  const int q_stage = first(k0) / QR, stages = max(0, (n + QR - 1) / QR - q_stage);
  const int own = first(key), w_first = first(key0), w_all = first(key0 + 31);

  v4i kf[NS], vf[NS];
  load_rows<DH>(a.k + (ks.first + key0) * a.k_tok + head * a.k_head, a.k_tok, m - key0, lane, kf);
  load_rows<DH>(a.v + (ks.first + key0) * a.v_tok + head * a.v_head, a.v_tok, m - key0, lane, vf);
  Loader<DH, QR, WAVES> ql, dl;
  ql.init(w, lane, a.q_tok);
  dl.init(w, lane, a.do_tok);
  const int steps = stages * a.s.group;
  const auto issue = [&](int g, int r, int stage) {
    const int64_t h = (int64_t)head * a.s.group + g;
    uint8_t* to = lds + stage * STAGE;
    ql.issue(rows_buffer<DH>(a.q + (qs.first + r) * a.q_tok + h * a.q_head, a.q_tok, n - r, QR), w, to);
    dl.issue(rows_buffer<DH>(a.dout + (qs.first + r) * a.do_tok + h * a.do_head, a.do_tok, n - r, QR), w, to + TILE);
    if (w < 2) dma4((w ? a.delta : a.lse) + h * a.s.q_rows + qs.first + r, n - r, lane * 4, to + 2 * TILE + w * QR * 4);
  };
  RowReads<DH> rr;
  TurnedReads<DH> tr;
  rr.init(lane);
  tr.init(lane);
  v16f dk[MT], dv[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) dk[mt] = dv[mt] = zeros16();
  Range range;

  if (steps > 0) issue(0, q_stage * QR, 0);
  for (int step = 0, g = 0, r0 = q_stage * QR; step < steps; ++step) {
    const int stage = step & 1, here = r0;
    const uint8_t *qt = lds + stage * STAGE, *dt = qt + TILE;
    wait_dma();
    __syncthreads();
    r0 += QR;
    if (r0 >= n) {   // the next head's queries
      r0 = q_stage * QR;
      ++g;
    }
    if (step + 1 < steps) issue(g, r0, 1 - stage);
#pragma unroll 1
    for (int x = 0; x < QR / 32; ++x) {
      const int r = here + 32 * x;
      if (r >= n || r + 31 < w_first) continue;
      v16f s = zeros16(), dp = zeros16();
#pragma unroll
      for (int st = 0; st < NS; ++st) s = mfma<F16>(rr.get(qt, x, st), kf[st], s);
#pragma unroll
      for (int st = 0; st < NS; ++st) dp = mfma<F16>(rr.get(dt, x, st), vf[st], dp);
      const float* stats = (const float*)(qt + 2 * TILE) + 32 * x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 l = *(const float4*)(stats + 8 * i + 4 * hf), d = *(const float4*)(stats + QR + 8 * i + 4 * hf);
        const float le[4] = {l.x, l.y, l.z, l.w}, de[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float p = __builtin_amdgcn_exp2f(fmaf(s[4 * i + e], a.s.sl2, LIFT<F16> - le[e]));
          if (r < w_all) p = r + 8 * i + 4 * hf + e >= own ? p : 0.f;
          s[4 * i + e] = p;
          dp[4 * i + e] = p == 0.f ? 0.f : p * (dp[4 * i + e] - de[e]);
        }
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
        for (int mt = 0; mt < MT; ++mt) {
          dv[mt] = mfma<F16>(tr.get(dt, 2 * x + u, mt), pf[u], dv[mt]);
          dk[mt] = mfma<F16>(tr.get(qt, 2 * x + u, mt), df[u], dk[mt]);
        }
    }
  }
  __syncthreads();
  if (key0 >= m) return;
  const float lift = __builtin_amdgcn_exp2f(-LIFT<F16>);
  uint8_t* mine = lds + w * STAGING<DH>;
  store_turned<DH, F16>(dk, a.s.scale * lift / range.scale, mine, lane, a.dk + (ks.first + key0) * o_tok + head * DH, o_tok, m - key0);
  __builtin_amdgcn_wave_barrier();
  store_turned<DH, F16>(dv, lift, mine, lane, a.dv + (ks.first + key0) * o_tok + head * DH, o_tok, m - key0);
}

// ---------------------------------------------------------------- dQ

constexpr int KT = 64, QT = 32 * WAVES;

template <int DH, bool F16>
__global__ __launch_bounds__(THREADS, 2) void packed_dq_kernel(BwdArgs a) {
  constexpr int NS = DH / 16, MT = DH / 32, TILE = KT * row_bytes<DH>, STAGE = 2 * TILE;
  constexpr int LDS = 2 * STAGE > WAVES * STAGING<DH> ? 2 * STAGE : WAVES * STAGING<DH>;
  __shared__ __align__(16) uint8_t lds[LDS];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t head, tile;
  head_tile(group_id(), a.s.q_heads, head, tile);
  if (tile >= a.tiles) return;
  const int64_t o_tok = (int64_t)a.s.q_heads * DH;
  zero_outside(a.s.starts, a.s.seqs, a.s.q_rows, a.dq + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  const Place at = place(a.s.starts, a.s.seqs, a.s.q_rows, QT, tile);
  if (at.seq < 0) return;
  const Span qs = span(a.s.starts, at.seq, a.s.q_rows), ks = span(a.s.k_starts, at.seq, a.s.k_rows);
  const int n = qs.n, m = ks.n, shift = m - n;
  const int q0 = (at.tiles - 1 - at.tile) * QT;
  const int row0 = q0 + 32 * w, row = row0 + (lane & 31);
  const auto seen = [&](int r) { return a.s.causal ? max(0, min(m, min(r, n - 1) + shift + 1)) : m; };
  const int upto = seen(q0 + QT - 1), w_upto = row0 < n ? seen(row0 + 31) : 0, w_first = seen(row0), own = seen(row);
  const int tiles = (upto + KT - 1) / KT;

  const uint16_t* kb = a.k + ks.first * a.k_tok + (head / a.s.group) * a.k_head;
  const uint16_t* vb = a.v + ks.first * a.v_tok + (head / a.s.group) * a.v_head;
  Loader<DH, KT, WAVES> kl, vl;
  kl.init(w, lane, a.k_tok);
  vl.init(w, lane, a.v_tok);
  const auto issue = [&](int t, int stage) {
    const int64_t r = (int64_t)t * KT;
    kl.issue(rows_buffer<DH>(kb + r * a.k_tok, a.k_tok, m - t * KT, KT), w, lds + stage * STAGE);
    vl.issue(rows_buffer<DH>(vb + r * a.v_tok, a.v_tok, m - t * KT, KT), w, lds + stage * STAGE + TILE);
  };
  if (tiles > 0) issue(0, 0);
  v4i qf[NS], df[NS];
  load_rows<DH>(a.q + (qs.first + row0) * a.q_tok + head * a.q_head, a.q_tok, n - row0, lane, qf);
  load_rows<DH>(a.dout + (qs.first + row0) * a.do_tok + head * a.do_head, a.do_tok, n - row0, lane, df);
  const int64_t stat = (int64_t)head * a.s.q_rows + qs.first + row;
  const float lse = row < n ? a.lse[stat] : INFINITY, delta = row < n ? a.delta[stat] : 0.f;
  RowReads<DH> rr;
  TurnedReads<DH> tr;
  rr.init(lane);
  tr.init(lane);
  v16f dq[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) dq[mt] = zeros16();
  Range range;

  for (int t = 0; t < tiles; ++t) {
    const int stage = t & 1;
    const uint8_t *kt = lds + stage * STAGE, *vt = kt + TILE;
    wait_dma();
    __syncthreads();
    if (t + 1 < tiles) issue(t + 1, 1 - stage);
#pragma unroll 1
    for (int x = 0; x < KT / 32; ++x) {
      const int j0 = t * KT + 32 * x;
      if (j0 >= w_upto) continue;
      v16f s = zeros16(), dp = zeros16();
#pragma unroll
      for (int st = 0; st < NS; ++st) s = mfma<F16>(rr.get(kt, x, st), qf[st], s);
#pragma unroll
      for (int st = 0; st < NS; ++st) dp = mfma<F16>(rr.get(vt, x, st), df[st], dp);
      const bool whole = j0 + 32 <= w_first;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float p = __builtin_amdgcn_exp2f(fmaf(s[i], a.s.sl2, LIFT<F16> - lse));
        if (!whole) p = j0 + 8 * (i >> 2) + 4 * hf + (i & 3) < own ? p : 0.f;
        dp[i] = p == 0.f ? 0.f : p * (dp[i] - delta);
      }
      v4i pf[2];
      float by;
      if constexpr (F16) {
        if (range.fit(dp, by)) times(dq, by);
      }
      pack16<F16>(dp, range.scale, pf);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) dq[mt] = mfma<F16>(tr.get(kt, 2 * x + u, mt), pf[u], dq[mt]);
    }
  }
  __syncthreads();
  if (row0 >= n) return;
  const float lift = __builtin_amdgcn_exp2f(-LIFT<F16>);
  store_turned<DH, F16>(dq, a.s.scale * lift / range.scale, lds + w * STAGING<DH>, lane, a.dq + (qs.first + row0) * o_tok + head * DH,
                        o_tok, n - row0);
}

template <int DH, bool F16>
void launch(BwdArgs a, hipStream_t stream) {
  const int64_t rows = a.s.q_rows * a.s.q_heads;
  packed_delta_kernel<DH, F16><<<grid_of((rows * (DH / 8) + THREADS - 1) / THREADS), THREADS, 0, stream>>>(a);
  if (a.dk) {
    a.tiles = (uint32_t)places_of(a.s.k_rows, a.s.seqs, 32 * WAVES);
    packed_dkv_kernel<DH, F16><<<grid_of((int64_t)a.tiles * a.s.k_heads), THREADS, 0, stream>>>(a);
  }
  if (a.dq) {
    a.tiles = (uint32_t)places_of(a.s.q_rows, a.s.seqs, QT);
    packed_dq_kernel<DH, F16><<<grid_of((int64_t)a.tiles * a.s.q_heads), THREADS, 0, stream>>>(a);
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
  if (k_rows < 1 || places_of(q_rows, seqs, packed::QT) * q_heads > 1 << 30 || places_of(k_rows, seqs, 32 * packed::WAVES) * k_heads > 1 << 30 ||
      q_rows * q_heads * dim / 8 / packed::THREADS > 1 << 30)
    return LBW_E_SHAPE;
  if (const int st = check_device()) return st;
  packed::BwdArgs a = {{seqs, q_rows, k_rows, (int)q_heads, (int)k_heads, (int)(q_heads / k_heads), starts, k_starts, causal,
                        sm_scale, sm_scale * packed::LOG2E},
                       (const uint16_t*)d_out, (const uint16_t*)out, (const uint16_t*)rest, (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v,
                       do_s_tok, do_s_head, q_s_tok, q_s_head, k_s_tok, k_s_head, v_s_tok, v_s_head, lse, (float*)workspace,
                       (uint16_t*)dq, (uint16_t*)dk, (uint16_t*)dv, 0};
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (dim == 128) f16 ? packed::launch<128, true>(a, (hipStream_t)stream) : packed::launch<128, false>(a, (hipStream_t)stream);
  else f16 ? packed::launch<64, true>(a, (hipStream_t)stream) : packed::launch<64, false>(a, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
