// Attention over packed sequences, forward (include/lbw_causal.h): S = q k^T, softmax, times v, a tile of keys after
// another with the running maximum and sum.
//
// A workgroup takes 128 queries of a head and sequence, 32 a wave, and walks the keys 64 at a time (two stages in LDS).
// S^T = K Q^T on v_mfma_f32_32x32x16: a lane holds one query and 32 of the 64 keys, so the row's maximum and sum are
// register work and one exchange between the wave's halves; P^T goes in the type of v from those registers into
// O^T += V^T P^T, whose V^T comes from the rows of v by transposing LDS reads.
#include "lbw_packed.h"

namespace lbw {
namespace packed {
namespace {

constexpr int WAVES = 4, KT = 64, THREADS = 64 * WAVES;

struct FwdArgs {
  Shape s;
  const uint16_t *q, *k, *v;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  uint16_t *out, *rest;
  float* lse;
  uint32_t tiles;
};

// QW waves side by side take 32 queries each; the 4 / QW that share queries take every (4 / QW)-th 32 keys, and join at the
// end what each has: where 128 queries a workgroup would leave the card half empty, 64 make twice as many, half as long.
template <int DH, bool F16, int QW>
__global__ __launch_bounds__(THREADS, 2) void packed_fwd_kernel(FwdArgs a) {
  constexpr int KW = WAVES / QW, QT = 32 * QW, XS = KT / 32 / KW;   // XS: 32 keys of a wave in a tile
  static_assert(KW == 1 || KW == 2, "a tile has 64 keys");
  constexpr int NS = DH / 16, MT = DH / 32, TILE = KT * row_bytes<DH>, STAGE = 2 * TILE;
  constexpr int SUMS = KW > 1 ? QW * (MT * 16 + 2) * 256 : 0;   // LDS bytes of what the second waves have
  constexpr int LDS = std::max(2 * STAGE, std::max(WAVES * STAGING<DH>, SUMS));
  __shared__ __align__(16) uint8_t lds[LDS];
  const int lane = threadIdx.x & 63, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qw = w % QW, kw = w / QW;
  uint32_t head, tile;
  head_tile(group_id(), a.s.k_heads, a.s.group, a.s.common, head, tile);
  if (tile >= a.tiles) return;
  const int64_t o_tok = (int64_t)a.s.q_heads * DH;
  const Where at = where(a.s.starts, a.s.k_starts, a.s.seqs, a.s.q_rows, a.s.k_rows, QT, tile);
  zero_outside(at.begin, at.end, a.s.q_rows, a.out + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  if (at.seq < 0) return;
  const Span qs = at.own, ks = at.other;
  const int n = qs.n, m = ks.n, shift = m - n, q0 = at.tile * QT;
  const int row0 = q0 + 32 * qw, row = row0 + (lane & 31);
  // keys that the tile's last query sees, and the wave's last and first
  const auto seen = [&](int r) { return a.s.causal ? max(0, min(m, min(r, n - 1) + shift + 1)) : m; };
  const int upto = seen(q0 + QT - 1), w_upto = row0 < n ? seen(row0 + 31) : 0, w_first = seen(row0), own = seen(row);
  const int tiles = (upto + KT - 1) / KT;

  const uint16_t* kb = a.k + ks.first * a.k_tok + (head / a.s.group) * a.k_head;
  const uint16_t* vb = a.v + ks.first * a.v_tok + (head / a.s.group) * a.v_head;
  Loader<DH, KT, WAVES> kl, vl;
  kl.init(w, lane, a.k_tok);
  vl.init(w, lane, a.v_tok);
  int left = m;
  const auto issue = [&](int stage) {   // the next tile
    kl.issue(rows_buffer<DH>(kb, a.k_tok, left, KT), w, lds + stage * STAGE);
    vl.issue(rows_buffer<DH>(vb, a.v_tok, left, KT), w, lds + stage * STAGE + TILE);
    kb += KT * a.k_tok;
    vb += KT * a.v_tok;
    left -= KT;
  };
  if (tiles > 0) issue(0);
  v4i qf[NS];
  load_rows<DH>(a.q + (qs.first + row0) * a.q_tok + head * a.q_head, a.q_tok, n - row0, lane, qf);
  arrived(qf);
  RowReads<DH> kr;
  TurnedReads<DH> vr;
  kr.init(lane);
  vr.init(lane);

  v16f o[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) o[mt] = zeros16();
  float top = -INFINITY, total = 0.f;

  const auto step = [&](int t, auto stage) {
    const uint8_t* kt = lds + decltype(stage)::value * STAGE;
    const uint8_t* vt = kt + TILE;
    wait_dma();
    __syncthreads();   // the tile is in LDS, and every wave is done with the other stage
    if (t + 1 < tiles) issue(1 - decltype(stage)::value);
    const int j0 = t * KT + 32 * XS * kw;   // the wave's keys of the tile
    if (j0 >= w_upto) return;
    // (reads in one go ahead of the products that use them: the compiler would wait for each by itself)
    v16f s[XS];
    v4i kf[XS][NS];
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int x = 0; x < XS; ++x) kf[x][st] = kr.get(kt, XS * kw + x, st);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < XS; ++x) s[x] = zeros16();
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int x = 0; x < XS; ++x) s[x] = mfma<F16>(kf[x][st], qf[st], s[x]);
    if (j0 + 32 * XS > w_first) {   // keys that a query does not see
      branch_here();
#pragma unroll
      for (int x = 0; x < XS; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (j0 + 32 * x + 8 * (i >> 2) + 4 * hf + (i & 3) >= own) s[x][i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < XS; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[x][i]);
    mx = max_xor32(mx) * a.s.sl2;
    const float next = fmaxf(top, mx);
    if (__any(next > top)) {
      // a row that has seen nothing yet has sums of zero, whatever they are multiplied by
      const float by = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - next);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[mt][i] *= by;
      total *= by;
      top = next;
    }
    const float off = (top == -INFINITY ? 0.f : -top) + LIFT<F16>;
    v4i pf[2 * XS];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2 * XS; ++u) {
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + j], a.s.sl2, off));
      sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      pf[u] = v4i{(int)pack<F16>(p[0], p[1]), (int)pack<F16>(p[2], p[3]), (int)pack<F16>(p[4], p[5]), (int)pack<F16>(p[6], p[7])};
    }
    total += sum;
#pragma unroll
    for (int u = 0; u < 2 * XS; ++u)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt] = mfma<F16>(vr.get(vt, 2 * XS * kw + u, mt), pf[u], o[mt]);
  };
  for (int t = 0; t < tiles; t += 2) {
    step(t, ic<0>{});
    if (t + 1 < tiles) step(t + 1, ic<1>{});
  }
  total = sum_xor32(total);
  __syncthreads();   // every wave is done with the stages
  if constexpr (KW > 1) {
    float* other = (float*)lds + qw * (MT * 16 + 2) * 64 + lane;
    if (kw) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) other[(mt * 16 + i) * 64] = o[mt][i];
      other[MT * 16 * 64] = top;
      other[(MT * 16 + 1) * 64] = total;
    }
    __syncthreads();
    if (kw) return;
    const float t1 = other[MT * 16 * 64], both = fmaxf(top, t1);
    const float by0 = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - both), by1 = t1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t1 - both);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[mt][i] = fmaf(by1, other[(mt * 16 + i) * 64], by0 * o[mt][i]);
    total = fmaf(by1, other[(MT * 16 + 1) * 64], by0 * total);
    top = both;
  }
  if (row0 >= n) return;
  // (staged where no other wave may still be reading)
  static_assert(KW == 1 || STAGING<DH> <= (MT * 16 + 2) * 256, "a wave's staging lies inside what it reads");
  uint8_t* mine = lds + (KW > 1 ? qw * (MT * 16 + 2) * 256 : w * STAGING<DH>);
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  store_turned<DH, F16>(o, inv, mine, lane, a.out + (qs.first + row0) * o_tok + head * DH, o_tok, n - row0);
  if (a.rest) {
    __builtin_amdgcn_wave_barrier();
    store_turned<DH, F16, true>(o, inv, mine, lane, a.rest + (qs.first + row0) * o_tok + head * DH, o_tok, n - row0);
  }
  if (a.lse && row < n && lane < 32)
    a.lse[(int64_t)head * a.s.q_rows + qs.first + row] = own > 0 ? top + __builtin_amdgcn_logf(total) - LIFT<F16> : INFINITY;
}

template <int DH, bool F16>
void launch(FwdArgs a, hipStream_t stream) {
  const auto groups = [&](int queries) { return xcd_groups(places_of(a.s.q_rows, a.s.seqs, queries), a.s.k_heads, a.s.group); };
  const bool wide = groups(128) >= 512;   // (two a CU)
  a.tiles = (uint32_t)places_of(a.s.q_rows, a.s.seqs, wide ? 128 : 64);
  if (wide) packed_fwd_kernel<DH, F16, 4><<<grid_of(groups(128)), THREADS, 0, stream>>>(a);
  else packed_fwd_kernel<DH, F16, 2><<<grid_of(groups(64)), THREADS, 0, stream>>>(a);
}

}  // namespace
}  // namespace packed
}  // namespace lbw

using namespace lbw;

namespace lbw {
namespace packed {

int check(int dtype, int64_t seqs, int64_t q_rows, int64_t k_rows, int64_t q_heads, int64_t k_heads, int64_t dim, float sm_scale) {
  if ((dtype != LBW_DTYPE_BF16 && dtype != LBW_DTYPE_FP16) || seqs < 1 || seqs > 65535 || q_rows < 1 || q_rows >= 1ll << 31 ||
      k_rows < 0 || k_rows >= 1ll << 31 || q_heads < 1 || q_heads > 4096 || k_heads < 1 || q_heads % k_heads ||
      (dim != 64 && dim != 128) || !(sm_scale > 0.f) || !(sm_scale < INFINITY))
    return LBW_E_SHAPE;
  return LBW_OK;
}
// (the kernels tell rows past a sequence's end by their offsets: those of different tokens lie apart)
bool aligned(const void* p, int64_t tok, int64_t head, int64_t dim) {
  return (uintptr_t)p % 16 == 0 && tok % 8 == 0 && head % 8 == 0 && tok >= dim && tok < 1 << 24 && head >= 0;
}

}  // namespace packed
}  // namespace lbw

extern "C" int lbw_packed_attn_fwd(const void* q, const void* k, const void* v, int dtype, int64_t seqs, int64_t q_rows,
                                   int64_t k_rows, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t q_s_tok,
                                   int64_t q_s_head, int64_t k_s_tok, int64_t k_s_head, int64_t v_s_tok, int64_t v_s_head,
                                   const int32_t* starts, const int32_t* k_starts, int causal, float sm_scale, void* out,
                                   void* rest, float* lse, void* stream) {
  if (!q || (k_rows && (!k || !v)) || !starts || !k_starts || !out) return LBW_E_NULL;
  if (const int st = packed::check(dtype, seqs, q_rows, k_rows, q_heads, k_heads, dim, sm_scale)) return st;
  if (!packed::aligned(q, q_s_tok, q_s_head, dim) || !packed::aligned(k, k_s_tok, k_s_head, dim) || !packed::aligned(v, v_s_tok, v_s_head, dim) ||
      ((uintptr_t)out | (uintptr_t)rest) % 16 || (uintptr_t)starts % 4 || (uintptr_t)k_starts % 4 || (uintptr_t)lse % 4)
    return LBW_E_ALIGN;
  if ((places_of(q_rows, seqs, 64) + 8) * q_heads > 1 << 30) return LBW_E_SHAPE;
  if (const int st = check_device()) return st;
  packed::FwdArgs a = {{seqs, q_rows, k_rows, (int)q_heads, (int)k_heads, (int)(q_heads / k_heads), (int)packed::xcd_common(k_heads), starts, k_starts, causal,
                        sm_scale, sm_scale * packed::LOG2E},
                       (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, q_s_tok, q_s_head, k_s_tok, k_s_head,
                       v_s_tok, v_s_head, (uint16_t*)out, (uint16_t*)rest, lse, 0};
  const bool f16 = dtype == LBW_DTYPE_FP16;
  if (dim == 128) f16 ? packed::launch<128, true>(a, (hipStream_t)stream) : packed::launch<128, false>(a, (hipStream_t)stream);
  else f16 ? packed::launch<64, true>(a, (hipStream_t)stream) : packed::launch<64, false>(a, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
