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
// places_of(rows) numbers; a number without a tile has seq < 0.
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
  if (tile >= tiles) return {-1, 0, 0};
  return {__builtin_amdgcn_readfirstlane((int)s), __builtin_amdgcn_readfirstlane((int)tile), __builtin_amdgcn_readfirstlane(tiles)};
}

// Rows of the tensor that belong to no sequence (before the first and behind the last): zeros, a part of them for each of
// `parts` workgroups (or waves; `threads` of it). `width` 16-bit values (a multiple of 8) from base on in rows `stride` elements apart.
__device__ __forceinline__ void zero_outside(const int32_t* starts, int64_t seqs, int64_t rows, uint16_t* base, int64_t stride,
                                             int width, uint32_t part, uint32_t parts, int thread, int threads) {
  const int64_t a = min(max((int64_t)starts[0], (int64_t)0), rows), b = min(max((int64_t)starts[seqs], a), rows);
  const int64_t outside = a + rows - b;
  if (outside == 0) return;
  const int pieces = width / 8;
  for (int64_t i = part; i < outside; i += parts)
    for (int c = thread; c < pieces; c += threads)
      *(v4i*)(base + (i < a ? i : b + (i - a)) * stride + c * 8) = v4i{0, 0, 0, 0};
}

}  // namespace lbw
