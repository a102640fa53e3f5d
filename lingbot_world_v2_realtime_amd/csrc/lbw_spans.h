// Sequences packed one behind the other: which rows one has, and which one a row or a tile of rows belongs to, from their
// starts in device memory.
#pragma once

#include "lbw_causal.h"
#include "lbw_rows.h"

namespace lbw {

// Rows [first, first + n) of a tensor: a sequence's part, kept inside the tensor whatever the starts say.
struct Span {
  int64_t first;
  int n;
};
__device__ __forceinline__ Span span(const int32_t* starts, int64_t s, int64_t rows) {
  const int64_t a = min(max((int64_t)starts[s], (int64_t)0), rows), b = min(max((int64_t)starts[s + 1], a), rows);
  return {a, (int)(b - a)};
}

// The last i of 0 .. n - 1 at which f(i) <= want, f not falling; -1 if there is none. The whole wave takes part, 64
// places a step: one step for 64 sequences, two for 4096.
template <typename F>
__device__ __forceinline__ int64_t last_of(int64_t n, int64_t want, F f) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0;
  bool found = false;
  while (true) {
    const int64_t step = (n + 63) / 64, at = lo + lane * step;
    const int below = __popcll(__ballot(lane * step < n && f(at) <= want));
    found = found || below > 0;
    if (below == 0) return found ? lo : -1;
    lo += (below - 1) * step;
    if (step == 1) return lo;
    n = min(step, n - (below - 1) * step);
  }
}

// Tiles of T rows of every sequence, numbered with gaps: those of sequence s from starts[s] / T + s on, which leaves room for
// every tile (a sequence from a to b has b / T - a / T + 1 at most) and needs no sum over the sequences before it. There are
// places_of(rows) numbers; a number without a tile has seq < 0 (one before its sequence's first, too: where starts fall, the
// search may end at a sequence that begins behind it).
struct Place {
  int seq, tile, tiles;   // (tiles: of the sequence)
};
inline int64_t places_of(int64_t rows, int64_t seqs, int T) { return rows / T + seqs; }
__device__ __forceinline__ Place place(const int32_t* starts, int64_t seqs, int64_t rows, int T, uint32_t want) {
  const auto base = [&](int64_t s) { return min(max((int64_t)starts[s], (int64_t)0), rows) / T + s; };
  const int64_t s = last_of(seqs, want, base);
  if (s < 0) return {-1, 0, 0};
  const int tiles = (span(starts, s, rows).n + T - 1) / T;
  const int64_t tile = want - base(s);
  if (tile < 0 || tile >= tiles) return {-1, 0, 0};
  return {__builtin_amdgcn_readfirstlane((int)s), __builtin_amdgcn_readfirstlane((int)tile), __builtin_amdgcn_readfirstlane(tiles)};
}

// A workgroup's place for a kernel whose tiles cost more the higher their number in the sequence is: the costly ones of all
// sequences first, where they are few enough to be looked at by the lanes of a wave (all of their starts in one load), else
// sequence by sequence. With it the rows of its sequence in both tensors (those cut into tiles, and the other one), and where
// the sequences of the first begin and end.
struct Where {
  int seq, tile, tiles;   // seq < 0: nothing to do
  Span own, other;
  int64_t begin, end;
};
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t x) {
  x += dpp_u32<DPP_XOR1>(x);
  x += dpp_u32<DPP_XOR2>(x);
  x += dpp_u32<DPP_HALF_MIRROR>(x);
  x += dpp_u32<DPP_MIRROR>(x);
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = r[0] + r[1];
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __builtin_amdgcn_readfirstlane(r[0] + r[1]);
}
__device__ __forceinline__ Where where(const int32_t* starts, const int32_t* others, int64_t seqs, int64_t rows, int64_t other_rows, int T,
                                       uint32_t want) {
  if (seqs > 63) {
    const auto inside = [&](int64_t x) { return min(max(x, (int64_t)0), rows); };
    const int64_t begin = inside(starts[0]), end = max(inside(starts[seqs]), begin);
    const Place p = place(starts, seqs, rows, T, want);
    if (p.seq < 0) return {-1, 0, 0, {0, 0}, {0, 0}, begin, end};
    return {p.seq, p.tiles - 1 - p.tile, p.tiles, span(starts, p.seq, rows), span(others, p.seq, other_rows), begin, end};
  }
  const int lane = threadIdx.x & 63, n_seqs = (int)seqs;
  const int a = lane <= n_seqs ? min(max(starts[lane], 0), (int)rows) : 0, b = lane <= n_seqs ? min(max(others[lane], 0), (int)other_rows) : 0;
  const int a1 = __shfl_down(a, 1), b1 = __shfl_down(b, 1);   // (of all lanes: one that is switched off gives nothing)
  const int rows_of = lane < n_seqs ? max(a1 - a, 0) : 0, others_of = lane < n_seqs ? max(b1 - b, 0) : 0;
  const int64_t begin = __builtin_amdgcn_readlane(a, 0), end = max((int64_t)__builtin_amdgcn_readlane(a, n_seqs), begin);
  const uint32_t tiles = (uint32_t)(rows_of + T - 1) / (uint32_t)T;
  const auto upward = [&](uint32_t t) { return wave_sum_u32(tiles > t ? tiles - t : 0); };   // tiles of number t and more
  if (want >= upward(0)) return {-1, 0, 0, {0, 0}, {0, 0}, begin, end};
  // the largest t with more than `want` tiles from it upward
  uint32_t lo = 0, hi = (uint32_t)rows / (uint32_t)T + 1;   // (none from hi on)
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (upward(mid) > want) lo = mid;
    else hi = mid;
  }
  // of the sequences with a tile lo, the one that is left
  const uint32_t rank = want - upward(lo + 1);
  const uint64_t mask = __ballot(tiles > lo);
  const uint64_t hit = __ballot((mask >> lane & 1) && (uint32_t)__popcll(mask & ((1ull << lane) - 1)) == rank);
  const int s = __builtin_ctzll(hit);
  return {s, (int)lo, __builtin_amdgcn_readlane((int)tiles, s), {__builtin_amdgcn_readlane(a, s), __builtin_amdgcn_readlane(rows_of, s)},
          {__builtin_amdgcn_readlane(b, s), __builtin_amdgcn_readlane(others_of, s)}, begin, end};
}

// Rows of the tensor that belong to no sequence (before a, and from b on): zeros, a part of them for each of
// `parts` workgroups (or waves; `threads` of it). `width` 16-bit values (a multiple of 8) from base on in rows `stride` elements apart.
__device__ __forceinline__ void zero_outside(int64_t a, int64_t b, int64_t rows, uint16_t* base, int64_t stride, int width, uint32_t part,
                                             uint32_t parts, int thread, int threads) {
  const int64_t outside = a + rows - b;
  if (outside == 0) return;
  const int pieces = width / 8;
  for (int64_t i = part; i < outside; i += parts)
    for (int c = thread; c < pieces; c += threads)
      *(v4i*)(base + (i < a ? i : b + (i - a)) * stride + c * 8) = v4i{0, 0, 0, 0};
}

__device__ __forceinline__ void zero_outside(const int32_t* starts, int64_t seqs, int64_t rows, uint16_t* base, int64_t stride, int width,
                                             uint32_t part, uint32_t parts, int thread, int threads) {
  const int64_t a = min(max((int64_t)starts[0], (int64_t)0), rows);
  zero_outside(a, min(max((int64_t)starts[seqs], a), rows), rows, base, stride, width, part, parts, thread, threads);
}

}  // namespace lbw
