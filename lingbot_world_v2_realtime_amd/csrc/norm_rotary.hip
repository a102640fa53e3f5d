// RMS norm of every head of q and k with the rotary turn (include/lbw_causal.h), forward and backward: y = turn(x r w), r =
// rsqrt(mean x^2 + eps). One pass over the rows, bound by memory.
//
// A row (a head of a token) belongs to a team of lanes, a power of two that holds its values two units a lane: partners of
// the turn, or two neighbouring units of the channels past it. The sum of squares is a few exchanges in the team, the weights
// of a lane's channels stay in registers for all of its rows, and a token's sines and cosines are formed once for all of its
// heads, in LDS. The gradient is the same walk: with u = x r, d = turn^-1(dy), g = d w,
//   dx = r (g - u mean(g u)),   dw = sum over rows of d u,
// where mean(g u) = r mean(g x) needs no second pass. A lane adds up its channels' weight gradients over its rows, a
// workgroup its teams, and a second kernel the workgroups, in one order.
//
// 6032 tokens, 12 + 12 heads of 128, bf16: 16.3 us, 4.5 TB/s of the 4.9 that a large copy reaches. 3998 tokens, 32 + 8 heads, fp32
// weights: forward 16.8 us (4.9 TB/s), gradients 30.5 (4.0) and 4.0 for the sums. The 6032 tokens in fp32: 44 us (3.4 TB/s),
// gradients 52.6 (4.2) and 4.9. 64 tokens of 12 + 2 heads: 6.8 us, a launch's latency.
#include <type_traits>

#include "lbw_causal.h"
#include "lbw_turn.h"

namespace lbw {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 8;   // of a step of a workgroup
constexpr int MAX_PAIRS = LBW_ROTARY_MAX_DIM / 2;
constexpr int MAX_GROUPS = 512;   // workgroups of a backward pass

template <int N>
using ic = std::integral_constant<int, N>;

struct Rows {
  const void *in, *grad;          // grad: of the outputs (backward), or null
  void* out;                      // or null
  const void* weight;             // or null
  int64_t heads, s_batch, s_tok, s_head, g_batch, g_tok, g_head, o_batch, o_tok, o_head;
};

struct NormRotaryArgs {
  Rows q, k;
  int64_t tokens, len;
  int dim, pairs, per_group, team, vec_fp32;
  const void* pos;
  int pos_is_i64;
  int64_t p_s_batch, p_s_tok, p_s_axis, pos_start;
  const double* freq;
  const int32_t* axis;
  int64_t axes;
  float factor, eps;
  float* partial;                 // [workgroups][2][dim], or null
};

// Sum over a team of 4 to 64 lanes, the same bits in each.
__device__ __forceinline__ float team_sum(float x, int team) {
  x += dpp<DPP_XOR1>(x);
  x += dpp<DPP_XOR2>(x);
  if (team > 4) x += dpp<DPP_HALF_MIRROR>(x);
  if (team > 8) x += dpp<DPP_MIRROR>(x);
  if (team > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (team > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// N weights from channel c on, in a load of their own type or of fp32.
template <int DT, int N>
__device__ __forceinline__ void load_weights(const void* v, int fp32, int c, float* w) {
  if (fp32) {
    constexpr int M = N < 4 ? N : 4;
#pragma unroll
    for (int i = 0; i < N; i += M) {
      Unit<LBW_DTYPE_FP32, M> u;
      u.load(v, c + i);
#pragma unroll
      for (int e = 0; e < M; ++e) w[i + e] = u.f[e];
    }
  } else {
    Unit<DT, N> u;
    u.load(v, c);
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = u.f[e];
  }
}

// N: values of a unit; U: items of a lane (4 where 64 lanes of one do not hold a row: single values of wide heads)
template <int DT, int N, bool INTER, int U, bool BWD>
__global__ __launch_bounds__(THREADS) void norm_rotary_kernel(NormRotaryArgs a) {
  __shared__ float2 cs[MAX_TOKENS * MAX_PAIRS];
  __shared__ int64_t at_tok[MAX_TOKENS][6];   // where a token's rows start: q, k, their gradients, the outputs
  const int team = a.team, it0 = threadIdx.x & (team - 1), mine = threadIdx.x / team, teams = THREADS / team;
  const int pair_items = a.pairs / N, rest = (a.dim - 2 * a.pairs) / N, items = pair_items + (rest + 1) / 2;

  int c0[U], c1[U];   // where a lane's two units lie in a head; -1: nothing there
  float sums[BWD ? 2 : 1][U][2 * N];
#pragma unroll
  for (int n = 0; n < U; ++n) {
    const int it = it0 + n * team, p = it * N, r0 = 2 * a.pairs + 2 * (it - pair_items) * N;
    const bool turned = it < pair_items;
    c0[n] = it < items ? (turned ? (INTER ? 2 * p : p) : r0) : -1;
    c1[n] = turned ? (INTER ? 2 * p + N : a.pairs + p) : it < items && r0 + N < a.dim ? r0 + N : -1;
    if constexpr (BWD) {
#pragma unroll
      for (int e = 0; e < 2 * N; ++e) sums[0][n][e] = sums[1][n][e] = 0.f;
    }
  }

  const int64_t groups = (a.tokens + a.per_group - 1) / a.per_group;
  for (int64_t group = group_id(); group < groups; group += BWD ? gridDim.x : groups) {
    const int64_t tok0 = group * a.per_group;
    const int ntok = (int)min((int64_t)a.per_group, a.tokens - tok0);
    if (BWD) __syncthreads();   // (the step before is done with what lies there)
    if (threadIdx.x < ntok) {
      const uint32_t tok = (uint32_t)(tok0 + threadIdx.x), b = tok / (uint32_t)a.len, t = tok - b * (uint32_t)a.len;
      at_tok[threadIdx.x][0] = b * a.q.s_batch + t * a.q.s_tok;
      at_tok[threadIdx.x][1] = b * a.k.s_batch + t * a.k.s_tok;
      at_tok[threadIdx.x][2] = b * a.q.g_batch + t * a.q.g_tok;
      at_tok[threadIdx.x][3] = b * a.k.g_batch + t * a.k.g_tok;
      at_tok[threadIdx.x][4] = b * a.q.o_batch + t * a.q.o_tok;
      at_tok[threadIdx.x][5] = b * a.k.o_batch + t * a.k.o_tok;
    }
    __syncthreads();
    // The rows of q, then those of k: a team's next row, loaded while the one before it is worked on (the first ones while the
    // angles are formed).
    typedef typename Unit<DT, N>::Raw Raw;
    struct Ahead {
      Raw x[U][2], d[BWD ? U : 1][2];
      char* out;
      uint32_t j;
    };
    const auto fetch = [&](auto which, uint32_t row) {
      constexpr int X = decltype(which)::value;
      const Rows& t = X ? a.k : a.q;
      const uint32_t heads = (uint32_t)t.heads;
      const bool live = row < ntok * heads;   // (lanes without a row take part in the exchanges)
      Ahead r;
      r.j = live ? row / heads : 0;
      const uint32_t h = live ? row - r.j * heads : 0;
      const char* in = (const char*)t.in + (at_tok[r.j][X] + h * t.s_head) * elem_size(DT);
      const char* grad = BWD && t.grad ? (const char*)t.grad + (at_tok[r.j][2 + X] + h * t.g_head) * elem_size(DT) : nullptr;
      r.out = t.out && live ? (char*)t.out + (at_tok[r.j][4 + X] + h * t.o_head) * elem_size(DT) : nullptr;
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = k ? c1[n] : c0[n];
          const bool there = live && c >= 0;
          r.x[n][k] = there ? Unit<DT, N>::raw(in, c) : Raw(0);
          if constexpr (BWD) r.d[n][k] = there && grad ? Unit<DT, N>::raw(grad, c) : Raw(0);
        }
      return r;
    };
    Ahead first[2];
    first[0] = fetch(ic<0>{}, mine);
    if (a.k.heads) first[1] = fetch(ic<1>{}, mine);
    for (int i = threadIdx.x; i < ntok * a.pairs; i += THREADS) {
      const int j = i / a.pairs, p = i - j * a.pairs;
      const uint32_t tok = (uint32_t)(tok0 + j), b = tok / (uint32_t)a.len, t = tok - b * (uint32_t)a.len;
      int64_t ax = 0;
      double freq = a.freq[p];
      if (a.axis) {   // an axis that the positions do not have: they are read inside, and the pair becomes NaN
        const int want = a.axis[p];
        ax = max((int64_t)0, min((int64_t)want, a.axes - 1));
        if (a.pos && ax != want) freq = __longlong_as_double(0x7FF8000000000000ll);
      }
      const int64_t at = b * a.p_s_batch + t * a.p_s_tok + ax * a.p_s_axis;
      const int64_t pos = !a.pos ? a.pos_start + t : a.pos_is_i64 ? ((const int64_t*)a.pos)[at] : ((const int32_t*)a.pos)[at];
      float s, c;
      turn_of<DT>(pos, freq, s, c);
      cs[i] = make_float2(a.factor * c, (BWD ? -a.factor : a.factor) * s);   // (the gradient's turn is the opposite one)
    }
    __syncthreads();
    const auto section = [&](auto which) {
      constexpr int X = decltype(which)::value;
      const Rows& t = X ? a.k : a.q;
      float w[U][2 * N];
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = k ? c1[n] : c0[n];
#pragma unroll
          for (int e = 0; e < N; ++e) w[n][k * N + e] = 1.f;
          if (c >= 0 && t.weight) load_weights<DT, N>(t.weight, a.vec_fp32, c, w[n] + k * N);
        }
      const uint32_t total = ntok * (uint32_t)t.heads;
      Ahead next = first[X];
      for (uint32_t row0 = 0; row0 < total; row0 += teams) {
        const Ahead now = next;
        const bool live = row0 + mine < total;
        if (row0 + teams < total) next = fetch(which, row0 + teams + mine);
        Unit<DT, N> x[U][2], d[BWD ? U : 1][2];
        float squares = 0.f, dots = 0.f;
#pragma unroll
        for (int n = 0; n < U; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            x[n][k].set(now.x[n][k]);
            if constexpr (BWD) d[n][k].set(now.d[n][k]);
          }
        // pair e of an item: in a row the values 2 e, 2 e + 1 of both units, else value e of each
        const auto turn = [&](Unit<DT, N> (&u)[2], int n) {
          if (c0[n] < 0 || it0 + n * team >= pair_items) return;
          const float2* at = cs + now.j * a.pairs + (it0 + n * team) * N;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            float& f0 = INTER && N > 1 ? (2 * e < N ? u[0].f[2 * e % N] : u[1].f[2 * e % N]) : u[0].f[e];
            float& f1 = INTER && N > 1 ? (2 * e < N ? u[0].f[(2 * e + 1) % N] : u[1].f[(2 * e + 1) % N]) : u[1].f[e];
            const float x0 = f0, x1 = f1;
            const float2 v = at[e];
            f0 = x0 * v.x - x1 * v.y;
            f1 = x1 * v.x + x0 * v.y;
          }
        };
#pragma unroll
        for (int n = 0; n < U; ++n) {
          if constexpr (BWD) turn(d[n], n);
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float v = x[n][k].f[e];
              squares = fmaf(v, v, squares);
              if constexpr (BWD) dots = fmaf(d[n][k].f[e] * w[n][k * N + e], v, dots);
            }
        }
        const float r = rsqrtf(team_sum(squares, team) / (float)a.dim + a.eps);
        if constexpr (BWD) dots = team_sum(dots, team) / (float)a.dim * r * r;
#pragma unroll
        for (int n = 0; n < U; ++n) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) {
              float& f = x[n][k].f[e];
              if constexpr (!BWD) {
                f = f * r * w[n][k * N + e];
              } else {
                const float dv = d[n][k].f[e];
                sums[X][n][k * N + e] += live ? dv * (f * r) : 0.f;
                f = r * (dv * w[n][k * N + e] - f * dots);
              }
            }
          if constexpr (!BWD) turn(x[n], n);
          if (now.out) {
            if (c0[n] >= 0) x[n][0].store(now.out, c0[n]);
            if (c1[n] >= 0) x[n][1].store(now.out, c1[n]);
          }
        }
      }
    };
    section(ic<0>{});
    if (a.k.heads) section(ic<1>{});
  }
  if constexpr (BWD) {
    if (!a.partial) return;
    // the teams of the workgroup, a tensor at a time: every team's values side by side, then a thread for each channel
    __shared__ float part[THREADS * 2 * N * U];
    for (int x = 0; x < 2; ++x) {
      __syncthreads();
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int e = 0; e < 2 * N; ++e) {
          const int c = e < N ? c0[n] : c1[n];
          if (c >= 0) part[mine * a.dim + c + e % N] = x ? sums[1][n][e] : sums[0][n][e];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.dim; c += THREADS) {
        float s = 0.f;
        for (int i = 0; i < teams; ++i) s += part[i * a.dim + c];
        a.partial[((int64_t)blockIdx.x * 2 + x) * a.dim + c] = s;
      }
    }
  }
}

// The workgroups' sums of the weights' gradients: 4 columns of [2][dim] by 64 slices of the workgroups.
template <int DT>
__global__ __launch_bounds__(THREADS) void norm_rotary_sums_kernel(const float* partial, int groups, int dim, int vec_fp32, void* dq, void* dk) {
  __shared__ float part[64][5];
  const int x = threadIdx.x & 3, col = blockIdx.x * 4 + x, slice = threadIdx.x >> 2;
  float s = 0.f;
  if (col < 2 * dim) {
#pragma unroll
    for (int i = 0; i < MAX_GROUPS / 64; ++i)
      if (i * 64 + slice < groups) s += partial[(int64_t)(i * 64 + slice) * 2 * dim + col];
  }
  part[slice][x] = s;
  __syncthreads();
  if (threadIdx.x >= 64) return;   // (the first wave: 16 lanes a column, four slices each)
  const int c = threadIdx.x >> 4, l = threadIdx.x & 15;
  s = (part[l][c] + part[l + 16][c]) + (part[l + 32][c] + part[l + 48][c]);
  s = row16_sum(s);
  const int out_col = blockIdx.x * 4 + c, at = out_col < dim ? out_col : out_col - dim;
  void* out = out_col < dim ? dq : dk;
  if (l || out_col >= 2 * dim || !out) return;
  if (vec_fp32) ((float*)out)[at] = s;
  else store1<DT>(out, at, s);
}

template <int DT, int N, bool BWD>
void launch(const NormRotaryArgs& a, bool inter, int64_t grid, hipStream_t stream) {
  const bool wide = N == 1 && a.dim > 128;   // (items past a wave's lanes)
  if constexpr (N == 1) {
    if (wide) {
      if (inter) norm_rotary_kernel<DT, N, true, 4, BWD><<<grid_of(grid), THREADS, 0, stream>>>(a);
      else norm_rotary_kernel<DT, N, false, 4, BWD><<<grid_of(grid), THREADS, 0, stream>>>(a);
      return;
    }
  }
  if (inter) norm_rotary_kernel<DT, N, true, 1, BWD><<<grid_of(grid), THREADS, 0, stream>>>(a);
  else norm_rotary_kernel<DT, N, false, 1, BWD><<<grid_of(grid), THREADS, 0, stream>>>(a);
}

template <int DT, bool BWD>
void launch_by_unit(const NormRotaryArgs& a, int unit, bool inter, int64_t grid, hipStream_t stream) {
  if (unit == 8) {
    if constexpr (DT != LBW_DTYPE_FP32) launch<DT, 8, BWD>(a, inter, grid, stream);
  } else if (unit == 4) {
    launch<DT, 4, BWD>(a, inter, grid, stream);
  } else {
    launch<DT, 1, BWD>(a, inter, grid, stream);
  }
}

template <bool BWD>
int run(NormRotaryArgs a, int dtype, int vec_dtype, int64_t batch, bool inter, void* dq_weight, void* dk_weight, hipStream_t stream) {
  const int es = elem_size(dtype);
  if (dtype < 0 || dtype > LBW_DTYPE_FP32 || (vec_dtype != dtype && vec_dtype != LBW_DTYPE_FP32) || batch < 1 || a.len < 1 ||
      batch > 1 << 30 || a.len > 1 << 30 || batch * a.len > 1 << 30 || a.q.heads < 1 || a.k.heads < 0 || a.q.heads > 4096 ||
      a.k.heads > 4096 || a.dim < 2 || a.dim > LBW_ROTARY_MAX_DIM || a.pairs < 1 || 2 * a.pairs > a.dim || a.axes < 1 || !(a.eps >= 0.f))
    return LBW_E_SHAPE;
  // the widest unit that sizes, strides and addresses are multiples of
  const auto fits = [&](int64_t n) {
    bool ok = a.dim % n == 0 && a.pairs % n == 0;
    for (const Rows* t : {&a.q, &a.k}) {
      if (!t->heads) continue;
      ok = ok && t->s_batch % n == 0 && t->s_tok % n == 0 && t->s_head % n == 0 && (uintptr_t)t->in % (n * es) == 0;
      if (t->grad) ok = ok && t->g_batch % n == 0 && t->g_tok % n == 0 && t->g_head % n == 0 && (uintptr_t)t->grad % (n * es) == 0;
      if (t->out) ok = ok && t->o_batch % n == 0 && t->o_tok % n == 0 && t->o_head % n == 0 && (uintptr_t)t->out % (n * es) == 0;
    }
    return ok;
  };
  if (!fits(1) || (uintptr_t)a.freq % 8 || (uintptr_t)a.axis % 4 || (uintptr_t)a.pos % (a.pos_is_i64 ? 8 : 4)) return LBW_E_ALIGN;
  for (const void* p : {a.q.weight, a.k.weight, (const void*)dq_weight, (const void*)dk_weight})
    if ((uintptr_t)p % 16) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const int unit = es == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
  const int items = a.pairs / unit + ((a.dim - 2 * a.pairs) / unit + 1) / 2;
  a.tokens = batch * a.len;
  a.vec_fp32 = vec_dtype == LBW_DTYPE_FP32;
  a.team = 4;
  while (a.team < 64 && a.team < items) a.team *= 2;
  // The tokens of a workgroup's step whose rows fill its teams best, q's and k's each by themselves, as long as there are
  // workgroups for every CU (6032 tokens of 12 + 12 heads: 17 us with eight, 21 with four).
  const int64_t teams = THREADS / a.team;
  double best = 0;
  a.per_group = 1;
  for (int n = 1; n <= MAX_TOKENS; n *= 2) {
    if (n > 1 && a.tokens / n < 512) break;
    const int64_t passes = (n * a.q.heads + teams - 1) / teams + (n * a.k.heads + teams - 1) / teams;
    const double filled = (double)(n * (a.q.heads + a.k.heads)) / (double)(passes * teams);
    if (filled > 1.05 * best) best = filled, a.per_group = n;
  }
  const int64_t groups = (a.tokens + a.per_group - 1) / a.per_group, grid = BWD ? std::min<int64_t>(groups, MAX_GROUPS) : groups;
  if (dtype == LBW_DTYPE_BF16) launch_by_unit<LBW_DTYPE_BF16, BWD>(a, unit, inter, grid, stream);
  else if (dtype == LBW_DTYPE_FP16) launch_by_unit<LBW_DTYPE_FP16, BWD>(a, unit, inter, grid, stream);
  else launch_by_unit<LBW_DTYPE_FP32, BWD>(a, unit, inter, grid, stream);
  if (BWD && a.partial) {
    const unsigned n = (2 * a.dim + 3) / 4;
    if (dtype == LBW_DTYPE_BF16) norm_rotary_sums_kernel<LBW_DTYPE_BF16><<<n, THREADS, 0, stream>>>(a.partial, (int)grid, a.dim, a.vec_fp32, dq_weight, dk_weight);
    else if (dtype == LBW_DTYPE_FP16) norm_rotary_sums_kernel<LBW_DTYPE_FP16><<<n, THREADS, 0, stream>>>(a.partial, (int)grid, a.dim, a.vec_fp32, dq_weight, dk_weight);
    else norm_rotary_sums_kernel<LBW_DTYPE_FP32><<<n, THREADS, 0, stream>>>(a.partial, (int)grid, a.dim, a.vec_fp32, dq_weight, dk_weight);
  }
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}

}  // namespace
}  // namespace lbw

using namespace lbw;

extern "C" int lbw_norm_rotary(const void* q, const void* k, int dtype, int vec_dtype, int64_t batch, int64_t len, int64_t q_heads,
                               int64_t k_heads, int64_t dim, int64_t pairs, int64_t q_s_batch, int64_t q_s_tok, int64_t q_s_head,
                               int64_t k_s_batch, int64_t k_s_tok, int64_t k_s_head, const void* q_weight, const void* k_weight,
                               float eps, const void* positions, int pos_is_i64, int64_t p_s_batch, int64_t p_s_tok,
                               int64_t p_s_axis, int64_t pos_start, const double* freq, const int32_t* axis, int64_t axes,
                               int interleaved, float factor, void* q_out, void* k_out, int64_t qo_s_batch, int64_t qo_s_tok,
                               int64_t qo_s_head, int64_t ko_s_batch, int64_t ko_s_tok, int64_t ko_s_head, void* stream) {
  if (!q || !q_out || !freq || (k_heads > 0 && (!k || !k_out))) return LBW_E_NULL;
  if (dim > LBW_ROTARY_MAX_DIM || pairs > LBW_ROTARY_MAX_DIM) return LBW_E_SHAPE;
  const NormRotaryArgs a = {{q, nullptr, q_out, q_weight, q_heads, q_s_batch, q_s_tok, q_s_head, 0, 0, 0, qo_s_batch, qo_s_tok, qo_s_head},
                            {k, nullptr, k_out, k_weight, k_heads, k_s_batch, k_s_tok, k_s_head, 0, 0, 0, ko_s_batch, ko_s_tok, ko_s_head},
                            0, len, (int)dim, (int)pairs, 1, 4, 0, positions, pos_is_i64, p_s_batch, p_s_tok, p_s_axis, pos_start,
                            freq, axis, axes, factor, eps, nullptr};
  return run<false>(a, dtype, vec_dtype, batch, interleaved, nullptr, nullptr, (hipStream_t)stream);
}

extern "C" int64_t lbw_norm_rotary_bwd_workspace_bytes(int64_t dim) { return (int64_t)MAX_GROUPS * 2 * dim * 4; }

extern "C" int lbw_norm_rotary_bwd(const void* dq, const void* dk, const void* q, const void* k, int dtype, int vec_dtype,
                                   int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t pairs,
                                   int64_t dq_s_batch, int64_t dq_s_tok, int64_t dq_s_head, int64_t dk_s_batch, int64_t dk_s_tok,
                                   int64_t dk_s_head, int64_t q_s_batch, int64_t q_s_tok, int64_t q_s_head, int64_t k_s_batch,
                                   int64_t k_s_tok, int64_t k_s_head, const void* q_weight, const void* k_weight, float eps,
                                   const void* positions, int pos_is_i64, int64_t p_s_batch, int64_t p_s_tok, int64_t p_s_axis,
                                   int64_t pos_start, const double* freq, const int32_t* axis, int64_t axes, int interleaved,
                                   float factor, void* dq_in, void* dk_in, int64_t qo_s_batch, int64_t qo_s_tok, int64_t qo_s_head,
                                   int64_t ko_s_batch, int64_t ko_s_tok, int64_t ko_s_head, void* dq_weight, void* dk_weight,
                                   void* workspace, void* stream) {
  const bool sums = dq_weight || dk_weight;
  if (!q || !freq || (k_heads > 0 && !k) || (sums && !workspace)) return LBW_E_NULL;
  if (dim > LBW_ROTARY_MAX_DIM || pairs > LBW_ROTARY_MAX_DIM) return LBW_E_SHAPE;
  if ((uintptr_t)workspace % 16) return LBW_E_ALIGN;
  const NormRotaryArgs a = {{q, dq, dq_in, q_weight, q_heads, q_s_batch, q_s_tok, q_s_head, dq_s_batch, dq_s_tok, dq_s_head, qo_s_batch, qo_s_tok, qo_s_head},
                            {k, dk, dk_in, k_weight, k_heads, k_s_batch, k_s_tok, k_s_head, dk_s_batch, dk_s_tok, dk_s_head, ko_s_batch, ko_s_tok, ko_s_head},
                            0, len, (int)dim, (int)pairs, 1, 4, 0, positions, pos_is_i64, p_s_batch, p_s_tok, p_s_axis, pos_start,
                            freq, axis, axes, factor, eps, sums ? (float*)workspace : nullptr};
  return run<true>(a, dtype, vec_dtype, batch, interleaved, dq_weight, dk_weight, (hipStream_t)stream);
}
