// The gated norm between two sub-layers of a block (include/lbw_block.h), forward and backward.
//
// Both directions are bound by memory: a row's inputs are read once into registers, where its statistics, its outputs
// and its gradients are formed, and nothing but the results goes back. A row belongs to a team of 64 lanes (a wave;
// no barrier) or of more waves of one workgroup (sums through LDS); thread i of a team of T holds the 8-value chunks
// i, i + T, ... of the row.
//
// 6032 x 1536 in bf16, LayerNorm, gate, shift and scale in 4 rows of fp32: forward 13.9 us (5.3 TB/s; a copy of 1 GiB
// reaches 5.1), backward 30.5 (3.6 TB/s, its fp32 sums left aside) and 6.1 for the sums over workgroups; one row 3.2.
//
// Norm statistics take two passes over the registers (mean, then the mean square of the differences): no
// cancellation.
//
// Backward, with u = norm(s), lin = u w + c, h = lin (1 + scale) + shift, s = a x + b gate pw v, v = post(y):
//   du = dh (1 + scale) w;  g = ds + r (du - [mean du] - u mean(du u))     (the bracket for LayerNorm)
//   dx = a g;  dv = b gate pw g;  dy = rv (dv - [mean dv] - v mean(dv v)), or dv without a post norm
// s and its statistics are formed again from x and y: the forward keeps nothing, and the rounded s_out would put its
// rounding into the vectors' gradients. Those need, for each modulation row and channel, only the three sums
//   A = sum dh u,  B = sum dh,  C = sum g v:
//   dshift = B, dscale = w A + c B, dgate = b pw C;  dweight = sum_rows (1 + scale) A, dbias = sum_rows (1 + scale) B,
//   dpost_weight = b sum_rows gate C
// A workgroup adds them over its rows (all of one modulation row) in registers and leaves one fp32 row each; a second
// kernel adds the workgroups of a modulation row, a third the modulation rows where a vector is shared by several. No
// atomics: the order of every sum is fixed by the sizes.
#include "lbw_rows.h"

namespace lbw {
namespace {

constexpr int MAX_TEAM = 512;
constexpr int SUM_ROWS = 3;         // A, B, C of a workgroup's rows
constexpr int SUM_COLS = 32;        // channels of a workgroup of the two summing kernels
constexpr int SLICES = 32;          // and the slices of the rows that it sums, at most

struct Vec {
  const void* p;
  int64_t s_batch, s_group;
};

struct NormArgs {
  const void *x, *y;
  int64_t rows, len, width, x_s_batch, x_s_tok, y_s_batch, y_s_tok, group_len;
  Vec gate, shift, scale;
  const void *weight, *bias, *post_weight;
  int norm, post_norm;
  float eps, a, b;
};

struct GradArgs {
  const void *ds, *dh;
  void *dx, *dy;
  float* sums;                      // [batch * groups][chunks][SUM_ROWS][width], or null: no vector's gradient is asked for
  int64_t groups, mrows, chunks, chunk_rows;   // mrows: modulation rows, those of every entry of the batch
};

struct VecGrads {
  void *gate, *shift, *scale, *weight, *bias, *post_weight;
  bool gate_rows, shift_rows, scale_rows;   // a gradient for every modulation row, or one for all
};

template <int DT>
__device__ __forceinline__ const char* at(const void* p, int64_t i) { return (const char*)p + i * elem_size(DT); }
template <int DT>
__device__ __forceinline__ char* at(void* p, int64_t i) { return (char*)p + i * elem_size(DT); }

__device__ __forceinline__ const char* vec_row(const Vec& v, int64_t b, int64_t g, int size) {
  return v.p ? (const char*)v.p + (b * v.s_batch + g * v.s_group) * size : nullptr;
}

// The part of a row that a thread of a team holds: NCH chunks of 8 values.
template <int NCH, bool VEC>
struct Span {
  int tid, team;
  int64_t width;
  __device__ __forceinline__ int64_t first(int c) const { return 8 * (int64_t)(tid + c * team); }
  // whether value e of chunk c lies in the row (with VEC the width is a multiple of 8)
  __device__ __forceinline__ bool in(int c, int e) const { return first(c) + (VEC ? 0 : e) < width; }
  template <int DT>
  __device__ __forceinline__ void load(Raw8<DT, VEC>* w, const void* p) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (first(c) < width) w[c].load(p, first(c), width);
      else w[c].zero();
    }
  }
  template <int DT>
  __device__ __forceinline__ void store(void* p, const float (*f)[8]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
      if (first(c) < width) store8<DT, VEC>(p, first(c), width, f[c]);
  }
  // op(f, value of the vector p at the same channel) over the span; p may be null
  template <int DT, typename F>
  __device__ __forceinline__ void with(float (*f)[8], const void* p, F op) const {
    if (!p) return;
    Raw8<DT, VEC> w[NCH];
    load(w, p);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float v[8];
      w[c].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) op(f[c][e], v[e]);
    }
  }
};

// A vector that the forward multiplies or adds. With one chunk a thread (few rows: the call is as long as its longest
// chain of loads) it is loaded at the row's start, with all the others; with more where it is used, for the
// registers.
template <int DT, int NCH, bool VEC>
struct Factor {
  const void* p;
  Raw8<DT, VEC> w[NCH];
  __device__ __forceinline__ Factor(const Span<NCH, VEC>& span, const void* at) : p(at) {
    if constexpr (NCH == 1) {
      if (p) span.load(w, p);
    }
  }
  // op(f, the vector's value at the same channel) over the span, unless there is no such vector
  template <typename F>
  __device__ __forceinline__ void apply(const Span<NCH, VEC>& span, float (*f)[8], F op) {
    if (!p) return;
    if constexpr (NCH > 1) span.load(w, p);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      float v[8];
      w[c].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) op(f[c][e], v[e]);
    }
  }
};

// Sums over a team, the same bits in all its threads. One wave: no LDS. Else every wave leaves its sums in `red`,
// which nobody may write again before another barrier has been passed.
template <int N>
__device__ __forceinline__ void team_sum(float* v, int team, float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if (team == 64) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[(threadIdx.x >> 6) * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int j = 0; j < team >> 6; ++j) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += red[j * N + i];
  }
}

constexpr int RED = 2 * (MAX_TEAM / 64);   // floats of a reduction's slot

// f <- (f - mean) / sqrt(. + eps), zero past the width; returns the factor.
template <int NCH, bool VEC>
__device__ __forceinline__ float normalise(float (*f)[8], int kind, const Span<NCH, VEC>& at, float eps, float* red) {
  // (divided, not multiplied by a rounded 1 / width: the mean of equal values is that value, and u = 0, wherever
  // their sum is exact)
  const float width = (float)at.width;
  if (kind == LBW_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += f[c][e];
    team_sum<1>(&s, at.team, red);
    const float mean = __fdiv_rn(s, width);
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[c][e] = at.in(c, e) ? f[c][e] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) q = fmaf(f[c][e], f[c][e], q);
  team_sum<1>(&q, at.team, red + RED);
  const float r = __frsqrt_rn(__fdiv_rn(q, width) + eps);
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) f[c][e] *= r;
  return r;
}

template <int DT, int VDT, int NCH, bool VEC>
__global__ __launch_bounds__(MAX_TEAM) void gated_norm_kernel(NormArgs a, int team, void* s_out, void* h_out) {
  __shared__ float red[4 * RED];
  const bool one = team == 64;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Span<NCH, VEC> span = {one ? (int)(threadIdx.x & 63) : (int)threadIdx.x, team, a.width};
  const int64_t row = one ? (int64_t)group_id() * (blockDim.x >> 6) + wave : group_id();
  if (row >= a.rows) return;   // whole workgroups, or whole waves where a wave is a team: nobody waits for them
  const int64_t b = row / a.len, t = row - b * a.len, g = t / a.group_len;
  Raw8<DT, VEC> xw[NCH], yw[NCH];
  float s[NCH][8];
  span.load(xw, at<DT>(a.x, b * a.x_s_batch + t * a.x_s_tok));
  if (a.y) span.load(yw, at<DT>(a.y, b * a.y_s_batch + t * a.y_s_tok));
  using V = Factor<VDT, NCH, VEC>;
  V post_weight(span, a.post_weight), gate(span, vec_row(a.gate, b, g, elem_size(VDT)));
  V weight(span, a.weight), bias(span, a.bias), scale(span, vec_row(a.scale, b, g, elem_size(VDT)));
  V shift(span, vec_row(a.shift, b, g, elem_size(VDT)));
  const auto mul = [](float& f, float w) { f *= w; };
  const auto add = [](float& f, float w) { f += w; };
  if (a.y) {
    float v[NCH][8];
#pragma unroll
    for (int c = 0; c < NCH; ++c) yw[c].get(v[c]);
    if (a.post_norm != LBW_NORM_NONE) normalise(v, a.post_norm, span, a.eps, red);
    post_weight.apply(span, v, mul);
    gate.apply(span, v, mul);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      xw[c].get(s[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] = fmaf(a.b, v[c][e], a.a * s[c][e]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      xw[c].get(s[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c][e] *= a.a;
    }
  }
  if (s_out) span.template store<DT>(at<DT>(s_out, row * a.width), s);
  if (a.norm == LBW_NORM_NONE) return;
  normalise(s, a.norm, span, a.eps, red + 2 * RED);
  weight.apply(span, s, mul);
  bias.apply(span, s, add);
  scale.apply(span, s, [](float& f, float w) { f *= 1.f + w; });
  shift.apply(span, s, add);
  span.template store<DT>(at<DT>(h_out, row * a.width), s);
}

// A workgroup takes the rows chunk * chunk_rows .. of modulation row workgroup / chunks: one after another with a
// team of several waves, one a wave where a wave is a team.
template <int DT, int VDT, int NCH, bool VEC>
__global__ __launch_bounds__(MAX_TEAM) void gated_norm_bwd_kernel(NormArgs a, GradArgs o, int team) {
  constexpr int ONE_WIDTH = 64 * 8 * NCH;   // the widest row of a one-wave team
  __shared__ float red[2][6 * RED];
  __shared__ float lds[SUM_ROWS * ONE_WIDTH];
  const bool one = team == 64;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const Span<NCH, VEC> span = {one ? (int)(threadIdx.x & 63) : (int)threadIdx.x, team, a.width};
  const int64_t id = group_id(), bg = id / o.chunks, chunk = id - bg * o.chunks;
  if (bg >= o.mrows) return;
  const int64_t b = bg / o.groups, g = bg - b * o.groups;
  int64_t t0 = g * a.group_len, t1 = min(t0 + a.group_len, a.len);
  t0 += chunk * o.chunk_rows;
  t1 = min(t1, t0 + o.chunk_rows);
  const int step = one ? (int)(blockDim.x >> 6) : 1;
  const float inv = 1.f / (float)a.width;

  float sa[NCH][8] = {}, sb[NCH][8] = {}, sc[NCH][8] = {};
  float gp[NCH][8], mw[NCH][8];   // b gate pw and (1 + scale) w, the same for all these rows
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      gp[c][e] = a.b;
      mw[c][e] = 1.f;
    }
  const auto mul = [](float& f, float w) { f *= w; };
  span.template with<VDT>(gp, a.post_weight, mul);
  span.template with<VDT>(gp, vec_row(a.gate, b, g, elem_size(VDT)), mul);
  span.template with<VDT>(mw, a.weight, mul);
  span.template with<VDT>(mw, vec_row(a.scale, b, g, elem_size(VDT)), [](float& f, float w) { f *= 1.f + w; });

  int turn = 0;   // the reductions' slots change from row to row: a wave may be a barrier ahead of another
  for (int64_t t = t0 + (one ? wave : 0); t < t1; t += step, turn ^= 1) {
    const int64_t row = b * a.len + t;
    Raw8<DT, VEC> xw[NCH], yw[NCH], dsw[NCH], dhw[NCH];
    span.load(xw, at<DT>(a.x, b * a.x_s_batch + t * a.x_s_tok));
    if (a.y) span.load(yw, at<DT>(a.y, b * a.y_s_batch + t * a.y_s_tok));
    if (o.dh) span.load(dhw, at<DT>(o.dh, row * a.width));
    if (o.ds) span.load(dsw, at<DT>(o.ds, row * a.width));
    float v[NCH][8], s[NCH][8], d[NCH][8];
    float rv = 1.f;
    if (a.y) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) yw[c].get(v[c]);
      if (a.post_norm != LBW_NORM_NONE) rv = normalise(v, a.post_norm, span, a.eps, red[turn]);
    }
    if (o.dh) {
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        xw[c].get(s[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[c][e] = a.y ? fmaf(gp[c][e], v[c][e], a.a * s[c][e]) : a.a * s[c][e];
      }
      const float r = normalise(s, a.norm, span, a.eps, red[turn] + 2 * RED);   // s is now u
      float m[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        dhw[c].get(d[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sa[c][e] = fmaf(d[c][e], s[c][e], sa[c][e]);
          sb[c][e] += d[c][e];
          d[c][e] *= mw[c][e];
          m[0] += d[c][e];
          m[1] = fmaf(d[c][e], s[c][e], m[1]);
        }
      }
      team_sum<2>(m, team, red[turn] + 4 * RED);
      const float m1 = a.norm == LBW_NORM_LAYER ? m[0] * inv : 0.f, m2 = m[1] * inv;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        float e8[8] = {};
        if (o.ds) dsw[c].get(e8);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[c][e] = fmaf(r, d[c][e] - m1 - s[c][e] * m2, e8[e]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < NCH; ++c) dsw[c].get(d[c]);
    }
    // d is now g, the stream's whole gradient
    if (o.dx) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[c][e] = a.a * d[c][e];
      span.template store<DT>(at<DT>(o.dx, row * a.width), s);
    }
    if (!a.y) continue;   // (for every row: no wave is left at a barrier)
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sc[c][e] = fmaf(d[c][e], v[c][e], sc[c][e]);
        d[c][e] *= gp[c][e];
      }
    if (!o.dy) continue;
    if (a.post_norm != LBW_NORM_NONE) {
      float m[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          m[0] += span.in(c, e) ? d[c][e] : 0.f;
          m[1] = fmaf(d[c][e], v[c][e], m[1]);
        }
      team_sum<2>(m, team, red[turn] + 5 * RED);
      const float m1 = a.post_norm == LBW_NORM_LAYER ? m[0] * inv : 0.f, m2 = m[1] * inv;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[c][e] = rv * (d[c][e] - m1 - v[c][e] * m2);
    }
    span.template store<DT>(at<DT>(o.dy, row * a.width), d);
  }
  if (!o.sums) return;
  float* out = o.sums + id * SUM_ROWS * a.width;
  if (one && blockDim.x > 64) {   // the waves' sums into one, in their order
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
      if (w == wave) {
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float* p = lds + e * (64 * NCH) + c * 64 + span.tid;   // neighbouring lanes, neighbouring banks
            const float p0 = w ? p[0] : 0.f, p1 = w ? p[ONE_WIDTH] : 0.f, p2 = w ? p[2 * ONE_WIDTH] : 0.f;
            p[0] = p0 + sa[c][e];
            p[ONE_WIDTH] = p1 + sb[c][e];
            p[2 * ONE_WIDTH] = p2 + sc[c][e];
          }
      }
      __syncthreads();
    }
    for (int64_t i = threadIdx.x; i < SUM_ROWS * a.width; i += blockDim.x) {
      const int k = (int)(i / a.width), ch = (int)(i - k * a.width);
      out[i] = lds[k * ONE_WIDTH + (ch & 7) * (64 * NCH) + (ch >> 3)];
    }
  } else {
    span.template store<LBW_DTYPE_FP32>(out, sa);
    span.template store<LBW_DTYPE_FP32>(out + a.width, sb);
    span.template store<LBW_DTYPE_FP32>(out + 2 * a.width, sc);
  }
}

// The gradients of what all modulation rows share, from sums over them: sum (1 + scale) A, sum (1 + scale) B, sum
// gate C, sum A, sum B, sum C.
template <int VDT>
__device__ __forceinline__ void finish(const NormArgs& a, const VecGrads& d, int64_t ch, const float* t) {
  if (d.weight) store1<VDT>(d.weight, ch, t[0]);
  if (d.bias) store1<VDT>(d.bias, ch, t[1]);
  if (d.post_weight) store1<VDT>(d.post_weight, ch, a.b * t[2]);
  if (d.gate && !d.gate_rows)
    store1<VDT>(d.gate, ch, a.b * (a.post_weight ? load1<VDT>(a.post_weight, ch) : 1.f) * t[5]);
  if (d.scale && !d.scale_rows)
    store1<VDT>(d.scale, ch, (a.weight ? load1<VDT>(a.weight, ch) : 1.f) * t[3] +
                                 (a.bias ? load1<VDT>(a.bias, ch) * t[4] : 0.f));
  if (d.shift && !d.shift_rows) store1<VDT>(d.shift, ch, t[4]);
}

template <int VDT>
__device__ __forceinline__ void weigh(const NormArgs& a, int64_t b, int64_t g, int64_t ch, const float* s, float* t) {
  const float sc = a.scale.p ? 1.f + load1<VDT>(a.scale.p, b * a.scale.s_batch + g * a.scale.s_group + ch) : 1.f;
  const float gt = a.gate.p ? load1<VDT>(a.gate.p, b * a.gate.s_batch + g * a.gate.s_group + ch) : 1.f;
  t[0] += sc * s[0];
  t[1] += sc * s[1];
  t[2] += gt * s[2];
#pragma unroll
  for (int k = 0; k < SUM_ROWS; ++k) t[SUM_ROWS + k] += s[k];
}

// The slices' sums of K values into those of slice 0, in halves (one slice adding all took 32 K reads in turn: 6.3 us
// for a kernel of two rows, 3.9 now). slices: a power of two, blockDim.x / SUM_COLS.
template <int K>
__device__ __forceinline__ void add_slices(float (*part)[K][SUM_COLS], int w, int lane, int slices, float* s) {
#pragma unroll
  for (int k = 0; k < K; ++k) part[w][k][lane] = s[k];
  for (int half = slices >> 1; half; half >>= 1) {
    __syncthreads();
    if (w < half) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        s[k] += part[w + half][k][lane];
        part[w][k][lane] = s[k];
      }
    }
  }
}

int slices_for(int64_t rows) {   // (two at least: whole waves)
  int n = 2;
  while (n < SLICES && n < rows) n *= 2;
  return n;
}

// The workgroups' sums of one modulation row (workgroup / tiles), SUM_COLS channels a workgroup, its half-waves
// taking them in turn, four in flight (6032 x 1536 in 4 rows, 252 workgroups' sums each: 6.1 us; with eight in flight
// 6.9, with 64 channels 6.4, with 16 channels 10.6): the row's own gradients, and its sums left where
// its first workgroup's were for the kernel below (which a single modulation row does not need: `last`).
template <int VDT>
__global__ __launch_bounds__(SUM_COLS * SLICES) void norm_group_sums_kernel(NormArgs a, GradArgs o, VecGrads d, int tiles,
                                                                            int last) {
  __shared__ float part[SLICES][SUM_ROWS][SUM_COLS];
  const int lane = threadIdx.x % SUM_COLS, w = threadIdx.x / SUM_COLS, slices = blockDim.x / SUM_COLS;
  const int64_t id = group_id(), bg = id / tiles, ch = SUM_COLS * (id - bg * tiles) + lane;
  const int64_t b = bg / o.groups, g = bg - b * o.groups;
  if (bg >= o.mrows) return;
  float* base = o.sums + bg * o.chunks * SUM_ROWS * a.width;
  float s[SUM_ROWS] = {};
  if (ch < a.width) {
    constexpr int U = 4;
    int64_t i = w;
    for (; i + (U - 1) * slices < o.chunks; i += U * slices) {
      float f[U][SUM_ROWS];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < SUM_ROWS; ++k) f[u][k] = base[((i + u * slices) * SUM_ROWS + k) * a.width + ch];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < SUM_ROWS; ++k) s[k] += f[u][k];
    }
    for (; i < o.chunks; i += slices)
#pragma unroll
      for (int k = 0; k < SUM_ROWS; ++k) s[k] += base[(i * SUM_ROWS + k) * a.width + ch];
  }
  add_slices<SUM_ROWS>(part, w, lane, slices, s);   // (past its first barrier every read of this row's sums is over)
  if (w || ch >= a.width) return;
  const int64_t at = bg * a.width + ch;
  if (d.shift && d.shift_rows) store1<VDT>(d.shift, at, s[1]);
  if (d.scale && d.scale_rows)
    store1<VDT>(d.scale, at, (a.weight ? load1<VDT>(a.weight, ch) : 1.f) * s[0] +
                                 (a.bias ? load1<VDT>(a.bias, ch) * s[1] : 0.f));
  if (d.gate && d.gate_rows)
    store1<VDT>(d.gate, at, a.b * (a.post_weight ? load1<VDT>(a.post_weight, ch) : 1.f) * s[2]);
  if (last) {
    float t[2 * SUM_ROWS] = {};
    weigh<VDT>(a, b, g, ch, s, t);
    finish<VDT>(a, d, ch, t);
  } else {
#pragma unroll
    for (int k = 0; k < SUM_ROWS; ++k) base[k * a.width + ch] = s[k];
  }
}

// The modulation rows' sums, weighted and added: the gradients of what they share.
template <int VDT>
__global__ __launch_bounds__(SUM_COLS * SLICES) void norm_shared_sums_kernel(NormArgs a, GradArgs o, VecGrads d) {
  __shared__ float part[SLICES][2 * SUM_ROWS][SUM_COLS];
  const int lane = threadIdx.x % SUM_COLS, w = threadIdx.x / SUM_COLS, slices = blockDim.x / SUM_COLS;
  const int64_t ch = SUM_COLS * (int64_t)blockIdx.x + lane;
  float t[2 * SUM_ROWS] = {};
  if (ch < a.width) {
    for (int64_t bg = w; bg < o.mrows; bg += slices) {
      const int64_t b = bg / o.groups;
      const float* p = o.sums + bg * o.chunks * SUM_ROWS * a.width + ch;
      const float s[SUM_ROWS] = {p[0], p[a.width], p[2 * a.width]};
      weigh<VDT>(a, b, bg - b * o.groups, ch, s, t);
    }
  }
  add_slices<2 * SUM_ROWS>(part, w, lane, slices, t);
  if (w || ch >= a.width) return;
  finish<VDT>(a, d, ch, t);
}

// Chunks a thread holds and threads a row's team has: the fewest idle lanes, and of those the smallest team (one wave
// needs no barrier; a tenth is added for those that do).
void pick(int64_t width, int most, int& nch, int& team) {
  int64_t best = INT64_MAX;
  for (int c = most; c >= 1; --c) {
    const int64_t t = (width + 8 * 64 * c - 1) / (8 * 64 * c) * 64;
    if (t > MAX_TEAM) continue;
    const int64_t cost = 10 * t * c + (t > 64 ? t * c : 0);
    if (cost < best) {
      best = cost;
      nch = c;
      team = (int)t;
    }
  }
}

// The backward holds three sums, two vectors and four rows of each: a third chunk spills (130 registers), and only
// the widest rows need it.
void pick_bwd(int64_t width, int& nch, int& team) { pick(width, width <= 2 * 8 * MAX_TEAM ? 2 : 3, nch, team); }

bool good(const void* p, int size) { return ((uintptr_t)p & (size - 1)) == 0; }

// LBW_OK, and in `vec` whether every row can be read 8 values at a time.
int check(const NormArgs& a, int dtype, int vec_dtype, int64_t batch, bool& vec, int64_t& rows) {
  if (!a.x) return LBW_E_NULL;
  if (dtype < 0 || dtype > LBW_DTYPE_FP32 || (vec_dtype != dtype && vec_dtype != LBW_DTYPE_FP32)) return LBW_E_SHAPE;
  if (batch < 1 || a.len < 1 || a.width < 1 || a.width > LBW_NORM_MAX_WIDTH || batch > (1 << 30) || a.len > (1 << 30) ||
      batch * a.len > (1 << 30) || a.group_len < 1)
    return LBW_E_SHAPE;
  if (a.norm < 0 || a.norm > LBW_NORM_RMS || a.post_norm < 0 || a.post_norm > LBW_NORM_RMS) return LBW_E_SHAPE;
  if (!a.y && (a.gate.p || a.post_weight || a.post_norm)) return LBW_E_NULL;
  if (a.norm == LBW_NORM_NONE && (a.weight || a.bias || a.scale.p || a.shift.p)) return LBW_E_SHAPE;
  const int es = elem_size(dtype), vs = elem_size(vec_dtype);
  rows = batch * a.len;
  const void* vs_p[] = {a.gate.p, a.shift.p, a.scale.p, a.weight, a.bias, a.post_weight};
  vec = a.width % 8 == 0;
  for (const void* p : {a.x, a.y}) {
    if (!good(p, es)) return LBW_E_ALIGN;
    vec = vec && good(p, 16);
  }
  for (const void* p : vs_p) {
    if (!good(p, vs)) return LBW_E_ALIGN;
    vec = vec && good(p, 16);
  }
  for (int64_t s : {a.x_s_batch, a.x_s_tok, a.y ? a.y_s_batch : 0, a.y ? a.y_s_tok : 0}) vec = vec && s * es % 16 == 0;
  for (const Vec* v : {&a.gate, &a.shift, &a.scale})
    if (v->p) vec = vec && v->s_batch * vs % 16 == 0 && v->s_group * vs % 16 == 0;
  return LBW_OK;
}

template <int DT, int VDT, bool VEC>
void forward(const NormArgs& a, void* s_out, void* h_out, hipStream_t stream) {
  // Few rows are a matter of latency: one chunk a thread and more threads a row (1536 channels, LayerNorm and post
  // norm: 1 row 4.7 -> 3.7 us, 64 rows 5.6 -> 4.1, 1024 rows 6.0 -> 5.6; but 2048 rows 8.1 -> 8.2, and with 4096
  // channels 14.2 -> 15.9).
  constexpr int FEW = 1024;
  int nch = 0, team = 0;
  pick(a.width, a.rows <= FEW && a.width <= 8 * MAX_TEAM ? 1 : 3, nch, team);
  const int threads = team == 64 ? 256 : team;
  const dim3 grid = grid_of(team == 64 ? (a.rows + 3) / 4 : a.rows);
  if (nch == 1) gated_norm_kernel<DT, VDT, 1, VEC><<<grid, threads, 0, stream>>>(a, team, s_out, h_out);
  else if (nch == 2) gated_norm_kernel<DT, VDT, 2, VEC><<<grid, threads, 0, stream>>>(a, team, s_out, h_out);
  else gated_norm_kernel<DT, VDT, 3, VEC><<<grid, threads, 0, stream>>>(a, team, s_out, h_out);
}

// Rows of a workgroup of the backward. More workgroups keep more rows in flight, but each leaves three fp32 rows
// behind that are written and read again (against six of `dtype` for every row of the tensors). With one chunk a
// thread 12 waves a CU are the best over widths (bf16, all gradients with their sums over rows: 6032 x 1536 8 waves
// 43.9 us, 12 36.5, 16 36.0, but 3016 x 2304 33.3 with 12, 40.2 with 16), where a wave is a team 16 (24000 x 512: 8
// waves 43.0, 16 37.8, 24 45.4), with two chunks 8, the registers' bound (4524 x 2048: 38.8, with 12 and 16 47.7: a
// second round).
void split(int64_t rows, int64_t len, int64_t group_len, int nch, int team, int64_t& chunk_rows, int64_t& chunks) {
  const int64_t gl = group_len < len ? group_len : len;
  const int waves = team == 64 ? 8 : team >> 6, room = nch == 1 ? (team == 64 ? 16 : 12) : 8;   // of a workgroup, and of a CU
  const int64_t blocks = 256 * (room > waves ? room / waves : 1);
  const int64_t step = team == 64 ? 8 : 1;
  int64_t r = (rows + blocks - 1) / blocks;
  r = (r + step - 1) / step * step;
  if (r < 4) r = 4;
  chunk_rows = r < gl ? r : gl;
  chunks = (gl + chunk_rows - 1) / chunk_rows;
}

template <int DT, int VDT, bool VEC>
void backward(const NormArgs& a, const GradArgs& o, int nch, int team, hipStream_t stream) {
  const int threads = team == 64 ? (int)(64 * (o.chunk_rows < 8 ? o.chunk_rows : 8)) : team;
  const dim3 grid = grid_of(o.mrows * o.chunks);
  if (nch == 1) gated_norm_bwd_kernel<DT, VDT, 1, VEC><<<grid, threads, 0, stream>>>(a, o, team);
  else if (nch == 2) gated_norm_bwd_kernel<DT, VDT, 2, VEC><<<grid, threads, 0, stream>>>(a, o, team);
  else gated_norm_bwd_kernel<DT, VDT, 3, VEC><<<grid, threads, 0, stream>>>(a, o, team);
}

// f(row format, vector format, 8 at a time) as compile-time values
template <typename F>
void by_type(int dtype, int vec_dtype, bool vec, F f) {
  const auto g = [&](auto d, auto v) {
    if (vec) f(d, v, std::integral_constant<bool, true>{});
    else f(d, v, std::integral_constant<bool, false>{});
  };
  using Bf = std::integral_constant<int, LBW_DTYPE_BF16>;
  using Hf = std::integral_constant<int, LBW_DTYPE_FP16>;
  using Fl = std::integral_constant<int, LBW_DTYPE_FP32>;
  if (dtype == LBW_DTYPE_FP32) g(Fl{}, Fl{});
  else if (dtype == LBW_DTYPE_FP16) vec_dtype == dtype ? g(Hf{}, Hf{}) : g(Hf{}, Fl{});
  else vec_dtype == dtype ? g(Bf{}, Bf{}) : g(Bf{}, Fl{});
}

}  // namespace
}  // namespace lbw

using namespace lbw;

extern "C" int lbw_gated_norm(const void* x, const void* y, int dtype, int vec_dtype, int64_t batch, int64_t len,
                              int64_t width, int64_t x_s_batch, int64_t x_s_tok, int64_t y_s_batch, int64_t y_s_tok,
                              const void* gate, int64_t gate_s_batch, int64_t gate_s_group, const void* shift,
                              int64_t shift_s_batch, int64_t shift_s_group, const void* scale, int64_t scale_s_batch,
                              int64_t scale_s_group, int64_t group_len, const void* weight, const void* bias,
                              const void* post_weight, int norm, int post_norm, float eps, float residual_scale,
                              float branch_scale, void* s_out, void* h_out, void* stream) {
  NormArgs a = {x, y, 0, len, width, x_s_batch, x_s_tok, y_s_batch, y_s_tok, group_len,
                {gate, gate_s_batch, gate_s_group}, {shift, shift_s_batch, shift_s_group},
                {scale, scale_s_batch, scale_s_group}, weight, bias, post_weight, norm, post_norm, eps, residual_scale,
                branch_scale};
  bool vec;
  if (const int st = check(a, dtype, vec_dtype, batch, vec, a.rows)) return st;
  if ((norm == LBW_NORM_NONE ? !s_out : !h_out) || (norm == LBW_NORM_NONE && h_out)) return LBW_E_NULL;
  for (void* p : {s_out, h_out}) {
    if (!good(p, elem_size(dtype))) return LBW_E_ALIGN;
    vec = vec && good(p, 16);
  }
  if (const int st = check_device()) return st;
  by_type(dtype, vec_dtype, vec, [&](auto d, auto v, auto w) {
    forward<d.value, v.value, w.value>(a, s_out, h_out, (hipStream_t)stream);
  });
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

extern "C" int64_t lbw_gated_norm_bwd_workspace_bytes(int64_t batch, int64_t len, int64_t width, int64_t groups,
                                                      int64_t group_len) {
  if (batch < 1 || len < 1 || width < 1 || width > LBW_NORM_MAX_WIDTH || groups < 1 || group_len < 1) return 0;
  int nch = 0, team = 0;
  pick_bwd(width, nch, team);
  int64_t chunk_rows, chunks;
  split(batch * len, len, group_len, nch, team, chunk_rows, chunks);
  return batch * groups * chunks * SUM_ROWS * width * (int64_t)sizeof(float);
}

extern "C" int lbw_gated_norm_bwd(const void* ds, const void* dh, const void* x, const void* y, int dtype,
                                  int vec_dtype, int64_t batch, int64_t len, int64_t width, int64_t x_s_batch,
                                  int64_t x_s_tok, int64_t y_s_batch, int64_t y_s_tok, const void* gate,
                                  int64_t gate_s_batch, int64_t gate_s_group, const void* scale,
                                  int64_t scale_s_batch, int64_t scale_s_group, int rowwise,
                                  int64_t groups, int64_t group_len, const void* weight, const void* bias,
                                  const void* post_weight, int norm, int post_norm, float eps,
                                  float residual_scale, float branch_scale, void* dx, void* dy, void* dgate,
                                  void* dshift, void* dscale, void* dweight, void* dbias, void* dpost_weight,
                                  void* workspace, void* stream) {
  NormArgs a = {x, y, 0, len, width, x_s_batch, x_s_tok, y_s_batch, y_s_tok, group_len,
                {gate, gate_s_batch, gate_s_group}, {nullptr, 0, 0},
                {scale, scale_s_batch, scale_s_group}, weight, bias, post_weight, norm, post_norm, eps, residual_scale,
                branch_scale};
  bool vec;
  if (const int st = check(a, dtype, vec_dtype, batch, vec, a.rows)) return st;
  if (!ds && !dh) return LBW_E_NULL;
  if (dh && norm == LBW_NORM_NONE) return LBW_E_SHAPE;
  if (!dh && (dshift || dscale || dweight || dbias)) return LBW_E_NULL;
  if ((dgate && !gate) || (dscale && !scale) || (dweight && !weight) || (dbias && !bias) ||
      (dpost_weight && !post_weight) || (dy && !y))
    return LBW_E_NULL;
  // every token's modulation row has to be among those the vectors' gradients hold
  if (groups < 1 || groups > (1 << 30) || group_len > (1 << 30) || (len - 1) / group_len >= groups ||
      batch * groups > (1 << 30))
    return LBW_E_SHAPE;
  const VecGrads d = {dgate, dshift, dscale, dweight, dbias, dpost_weight, (rowwise & 1) != 0, (rowwise & 2) != 0,
                      (rowwise & 4) != 0};
  const bool sums = dgate || dshift || dscale || dweight || dbias || dpost_weight;
  if (sums && !workspace) return LBW_E_NULL;
  for (const void* p : {ds, dh, (const void*)dx, (const void*)dy}) {
    if (!good(p, elem_size(dtype))) return LBW_E_ALIGN;
    vec = vec && good(p, 16);
  }
  for (void* p : {dgate, dshift, dscale, dweight, dbias, dpost_weight})
    if (!good(p, elem_size(vec_dtype))) return LBW_E_ALIGN;
  if (sums && !good(workspace, 16)) return LBW_E_ALIGN;
  int nch = 0, team = 0;
  pick_bwd(width, nch, team);
  GradArgs o = {ds, dh, dx, dy, sums ? (float*)workspace : nullptr, groups, batch * groups, 0, 0};
  split(a.rows, len, group_len, nch, team, o.chunk_rows, o.chunks);
  if (o.mrows * o.chunks > (1 << 30) || o.mrows * ((width + SUM_COLS - 1) / SUM_COLS) > (1 << 30))
    return LBW_E_SHAPE;
  if (const int st = check_device()) return st;
  by_type(dtype, vec_dtype, vec, [&](auto dt, auto vt, auto w) {
    backward<dt.value, vt.value, w.value>(a, o, nch, team, (hipStream_t)stream);
    if (!sums) return;
    const unsigned tiles = (unsigned)((width + SUM_COLS - 1) / SUM_COLS);
    norm_group_sums_kernel<vt.value><<<grid_of(tiles * o.mrows), SUM_COLS * slices_for(o.chunks), 0, (hipStream_t)stream>>>(
        a, o, d, (int)tiles, o.mrows == 1);
    const bool shared = dweight || dbias || dpost_weight || (dgate && !d.gate_rows) ||
                        (dscale && !d.scale_rows) || (dshift && !d.shift_rows);
    if (shared && o.mrows > 1)
      norm_shared_sums_kernel<vt.value><<<tiles, SUM_COLS * slices_for(o.mrows), 0, (hipStream_t)stream>>>(a, o, d);
  });
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
