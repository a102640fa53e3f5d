// Attention over packed sequences, forward (include/lbw_causal.h): S = q k^T, softmax, times v, a tile of keys after
// another with the running maximum and sum.
//
// A workgroup takes 128 queries of a head and sequence, 32 a wave, or 64 by two waves each, and walks the keys 64 at a time (two
// stages in LDS).
// S^T = K Q^T on v_mfma_f32_32x32x16: a lane holds one query and 32 of the 64 keys, so the row's maximum and sum are
// register work and one exchange between the wave's halves; P^T goes in the type of v from those registers into
// O^T += V^T P^T, whose V^T comes from the rows of v by transposing LDS reads.
//
// Bound by the matrix units and the softmax's vector work beside them, of which either is busy about half of the time (two
// waves a SIMD cover each other in part). 12 heads of 128, one sequence of 12064: 447 to 475 us, 0.94 to 1.0 PFLOP/s of the
// products that are seen, 0.75 to 0.8 of what a library product of 8192^3 reaches here. 8 sequences of up to 1508, 32 heads over
// 8: 96 us, 0.66 PFLOP/s (the diagonal tiles are half masked, the longest sequence's last tile is 24 steps). 61 captions of up
// to 77, 16 heads of 64, fp16: 9.4 us, launch and one trip to memory and back.
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
__global__ __launch_bounds__(THREADS, DH == 128 ? 2 : 4) void packed_fwd_kernel(FwdArgs a) {
  constexpr int KW = WAVES / QW, QT = 32 * QW, XS = KT / 32 / KW;   // XS: 32 keys of a wave in a tile
  static_assert(KW == 1 || KW == 2, "a tile has 64 keys");
  constexpr int NS = DH / 16, MT = DH / 32, TILE = KT * row_bytes<DH>, STAGE = 2 * TILE;
  constexpr int SUMS = KW > 1 ? QW * (MT * 16 + 2) * 256 : 0;   // LDS bytes of what the second waves have
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
  zero_outside(at.begin, at.end, a.s.q_rows, a.out + head * DH, o_tok, DH, tile, a.tiles, threadIdx.x, THREADS);
  if (at.seq < 0) return;
  const Span qs = at.own, ks = at.other;
  const int n = qs.n, m = ks.n, shift = m - n, q0 = at.tile * QT;
  const int row0 = q0 + 32 * qw, row = row0 + (lane & 31);
  // keys that the tile's last query sees, and the wave's last and first
  const auto seen = [&](int r) { return a.s.causal ? max(0, min(m, min(r, n - 1) + shift + 1)) : m; };
  const int upto = seen(q0 + QT - 1), w_upto = row0 < n ? seen(row0 + 31) : 0, w_first = seen(row0), own = seen(row);
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
  v4i qf[NS];
  load_rows<DH>(a.q + (qs.first + row0) * a.q_tok + head * a.q_head, a.q_tok, n - row0, lane, qf);
  arrived(qf);
  RowReads<DH> kr;
  TurnedReads<DH> vr;
  kr.init(lane);
  vr.init(lane);

  v16f o[MT];
  float top, total;

  const auto arrive = [&](int t, int stage) __attribute__((always_inline)) {
    wait_dma();
    __syncthreads();   // the tile is in LDS, and every wave is done with the other stage
    if (t + 1 < tiles) issue(1 - stage);
  };
  // XN times 32 keys of a tile, from the x0-th on
  const auto work = [&](int t, int stage, int x0, auto xn, auto again, const RowReads<DH>& kr, const TurnedReads<DH>& vr, int hf, int own, const v4i (&qf)[NS]) __attribute__((always_inline)) {
    constexpr int XN = decltype(xn)::value;
    const uint8_t* kt = lds + stage * STAGE;
    const uint8_t* vt = kt + TILE;
    const int j0 = t * KT + 32 * x0;
    if (j0 >= w_upto) return;
    // (reads in one go ahead of the products that use them: the compiler would wait for each by itself)
    v16f s[XN];
    v4i kf[XN][NS];
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int x = 0; x < XN; ++x) kf[x][st] = kr.get(kt, x0 + x, st);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < XN; ++x) s[x] = zeros16();
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int x = 0; x < XN; ++x) s[x] = mfma<F16>(kf[x][st], qf[st], s[x]);
    const bool partly = j0 + 32 * XN > w_first;   // keys that a query does not see
    if (partly) {
      branch_here();
#pragma unroll
      for (int x = 0; x < XN; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (j0 + 32 * x + 8 * (i >> 2) + 4 * hf + (i & 3) >= own) s[x][i] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < XN; ++x)
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
    v4i pf[2 * XN];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2 * XN; ++u) {
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[u >> 1][8 * (u & 1) + j], a.s.sl2, off));
      sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      pf[u] = v4i{(int)pack<F16>(p[0], p[1]), (int)pack<F16>(p[2], p[3]), (int)pack<F16>(p[4], p[5]), (int)pack<F16>(p[6], p[7])};
    }
    total += sum;
    if (decltype(again)::value && partly) {
#pragma unroll
      for (int u = 0; u < 2 * XN; ++u)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          o[mt] = mfma<F16>(clean<F16>(vr.get(vt, 2 * x0 + u, mt)), pf[u], o[mt]);
          __builtin_amdgcn_sched_barrier(0);
        }
      add_odd<DH, F16>(o, vt, x0, hf, [&](int j) { return j0 + j < own; });   // (XN is 1)
      return;
    }
#pragma unroll
    for (int u = 0; u < 2 * XN; ++u)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[mt] = mfma<F16>(vr.get(vt, 2 * x0 + u, mt), pf[u], o[mt]);
  };
  const auto clear = [&] {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] = zeros16();
    top = -INFINITY, total = 0.f;
  };
  clear();
  for (int t = 0; t < tiles; t += 2) {
    arrive(t, 0);
    work(t, 0, XS * kw, ic<XS>{}, ic<0>{}, kr, vr, hf, own, qf);
    if (t + 1 < tiles) {
      arrive(t + 1, 1);
      work(t + 1, 1, XS * kw, ic<XS>{}, ic<0>{}, kr, vr, hf, own, qf);
    }
  }
  // (the lane's number again, unknown to the compiler: what it makes of it is not held in registers all through the loop)
  int late = threadIdx.x;
  asm volatile("" : "+v"(late));
  late &= 63;
  const bool bad = any_odd(o);
  if (late == 0) odd[w] = bad;
  __syncthreads();   // every wave is done with the stages
  if (__builtin_expect(a.s.causal && __builtin_amdgcn_readfirstlane(odd[0] | odd[1] | odd[2] | odd[3]), 0)) {
    RowReads<DH> kr;
    TurnedReads<DH> vr;
    kr.init(late);
    vr.init(late);
    kl.init(w, late, a.k_tok);
    vl.init(w, late, a.v_tok);
    from_start();
    issue(0);   // (there is a tile: without one the sums are zeros)
    clear();
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      arrive(t, t & 1);
#pragma unroll 1
      for (int x = XS * kw; x < XS * (kw + 1); ++x) {
        int l = late;
        asm volatile("" : "+v"(l));
        v4i qx[NS];   // (read again rather than kept)
        load_rows<DH>(a.q + (qs.first + row0) * a.q_tok + head * a.q_head, a.q_tok, n - row0, l, qx);
        work(t, t & 1, x, ic<1>{}, ic<1>{}, kr, vr, l >> 5, seen(row0 + (l & 31)), qx);
      }
    }
    __syncthreads();
  }
  total = sum_xor32(total);
  if constexpr (KW > 1) {
    float* other = (float*)lds + qw * (MT * 16 + 2) * 64 + late;
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
  // A row that sees nothing is zero; one whose scores are all minus infinity has no softmax, and is NaN (0 / 0).
  const float inv = total > 0.f || total != total ? 1.f / total : seen(row0 + (late & 31)) > 0 ? __builtin_nanf("") : 0.f;
  store_turned<DH, F16>(o, inv, mine, late, a.out + (qs.first + row0) * o_tok + head * DH, o_tok, n - row0);
  if (a.rest) {
    __builtin_amdgcn_wave_barrier();
    store_turned<DH, F16, true>(o, inv, mine, late, a.rest + (qs.first + row0) * o_tok + head * DH, o_tok, n - row0);
  }
  if (const int row = row0 + late; a.lse && row < n && late < 32)
    a.lse[(int64_t)head * a.s.q_rows + qs.first + row] = seen(row) > 0 ? top + __builtin_amdgcn_logf(total) - LIFT<F16> : INFINITY;
}

template <int DH, bool F16>
void launch(FwdArgs a, hipStream_t stream) {
  const auto groups = [&](int queries) { return xcd_groups(places_of(a.s.q_rows, a.s.seqs, queries), a.s.k_heads, a.s.group); };
  // Two a CU (us for 128 and 64 queries: 32 heads over 8, one sequence of 1024, 288 workgroups of 128: 31, 29; of 2048, 544: 61, 65;
  // 4 of 1024: 59, 74).
  const bool wide = groups(128) >= 512;
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
