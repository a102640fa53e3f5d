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
#include "lbw_causal.h"
#include "lbw_turn.h"

namespace lbw {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 8;   // of a step of a workgroup
constexpr int MAX_PAIRS = LBW_ROTARY_MAX_DIM / 2;
constexpr int MAX_GROUPS = 1024;   // workgroups of a backward pass

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

// N: values of a unit; U: items of a lane (4 where 64 lanes of one do not hold a row: single values of wide heads)
template <int DT, int N, bool INTER, int U, bool BWD>
__global__ __launch_bounds__(THREADS) void norm_rotary_kernel(NormRotaryArgs a) {
  __shared__ float2 cs[MAX_TOKENS * MAX_PAIRS];
  __shared__ int64_t at_tok[MAX_TOKENS][6];   // where a token's rows start: q, k, their gradients, the outputs
  const int team = a.team, it0 = threadIdx.x & (team - 1), mine = threadIdx.x / team, teams = THREADS / team;
  const int pair_items = a.pairs / N, rest = (a.dim - 2 * a.pairs) / N, items = pair_items + (rest + 1) / 2;
  const uint32_t heads = (uint32_t)(a.q.heads + a.k.heads);

  // a lane's channels: where its two units lie, and their weights for q and k
  int c0[U], c1[U];   // -1: nothing there
  float w[2][U][2 * N], sums[BWD ? 2 : 1][U][2 * N];
#pragma unroll
  for (int n = 0; n < U; ++n) {
    const int it = it0 + n * team, p = it * N, r0 = 2 * a.pairs + 2 * (it - pair_items) * N;
    const bool turned = it < pair_items;
    c0[n] = it < items ? (turned ? (INTER ? 2 * p : p) : r0) : -1;
    c1[n] = turned ? (INTER ? 2 * p + N : a.pairs + p) : it < items && r0 + N < a.dim ? r0 + N : -1;
#pragma unroll
    for (int e = 0; e < 2 * N; ++e) {
      const int c = e < N ? c0[n] : c1[n], at = c + e % N;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const void* v = x ? a.k.weight : a.q.weight;
        w[x][n][e] = c < 0 || !v ? 1.f : a.vec_fp32 ? ((const float*)v)[at] : load1<DT>(v, at);
        if constexpr (BWD) sums[x][n][e] = 0.f;
      }
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
    const uint32_t total = ntok * heads;
    for (uint32_t row0 = 0; row0 < total; row0 += teams) {
      const uint32_t row = row0 + mine;
      const bool live = row < total;   // (lanes without a row take part in the exchanges)
      const uint32_t j = live ? row / heads : 0, h = live ? row - j * heads : 0;
      const bool is_q = h < (uint32_t)a.q.heads;
      const Rows& t = is_q ? a.q : a.k;
      const int64_t hh = is_q ? h : h - a.q.heads;
      const char* in = (const char*)t.in + (at_tok[j][is_q ? 0 : 1] + hh * t.s_head) * elem_size(DT);
      const char* grad = BWD && t.grad ? (const char*)t.grad + (at_tok[j][is_q ? 2 : 3] + hh * t.g_head) * elem_size(DT) : nullptr;
      char* out = t.out ? (char*)t.out + (at_tok[j][is_q ? 4 : 5] + hh * t.o_head) * elem_size(DT) : nullptr;
      Unit<DT, N> x[U][2], d[BWD ? U : 1][2];
      float squares = 0.f, dots = 0.f;
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = k ? c1[n] : c0[n];
          if (live && c >= 0) {
            x[n][k].load(in, c);
            if constexpr (BWD) {
              if (grad) d[n][k].load(grad, c);
            }
          }
          if (!(live && c >= 0)) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[n][k].f[e] = 0.f;
          }
          if constexpr (BWD) {
            if (!(live && c >= 0 && grad)) {
#pragma unroll
              for (int e = 0; e < N; ++e) d[n][k].f[e] = 0.f;
            }
          }
        }
      // pair e of an item: in a row the values 2 e, 2 e + 1 of both units, else value e of each
      const auto turn = [&](Unit<DT, N> (&u)[2], int n) {
        if (c0[n] < 0 || it0 + n * team >= pair_items) return;
        const float2* at = cs + j * a.pairs + (it0 + n * team) * N;
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
            if constexpr (BWD) dots = fmaf(d[n][k].f[e] * (is_q ? w[0][n][k * N + e] : w[1][n][k * N + e]), v, dots);
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
            const float wt = is_q ? w[0][n][k * N + e] : w[1][n][k * N + e];
            if constexpr (!BWD) {
              f = f * r * wt;
            } else {
              const float dv = d[n][k].f[e], du = live ? dv * (f * r) : 0.f;
              sums[0][n][k * N + e] += is_q ? du : 0.f;
              sums[1][n][k * N + e] += is_q ? 0.f : du;
              f = r * (dv * wt - f * dots);
            }
          }
        if constexpr (!BWD) turn(x[n], n);
        if (live && out) {
          if (c0[n] >= 0) x[n][0].store(out, c0[n]);
          if (c1[n] >= 0) x[n][1].store(out, c1[n]);
        }
      }
    }
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

// The workgroups' sums of the weights' gradients: 16 columns of [2][dim] by 16 slices of the workgroups.
template <int DT>
__global__ __launch_bounds__(THREADS) void norm_rotary_sums_kernel(const float* partial, int groups, int dim, int vec_fp32, void* dq, void* dk) {
  __shared__ float part[16][17];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), slice = threadIdx.x >> 4;
  float s = 0.f;
  if (col < 2 * dim)
    for (int i = slice; i < groups; i += 16) s += partial[(int64_t)i * 2 * dim + col];
  part[slice][threadIdx.x & 15] = s;
  __syncthreads();
  if (threadIdx.x >= 16 || col >= 2 * dim) return;
  s = 0.f;
  for (int i = 0; i < 16; ++i) s += part[i][threadIdx.x];
  void* out = col < dim ? dq : dk;
  const int c = col < dim ? col : col - dim;
  if (!out) return;
  if (vec_fp32) ((float*)out)[c] = s;
  else store1<DT>(out, c, s);
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
    if ((uintptr_t)p % elem_size(vec_dtype)) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  const int unit = es == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
  const int items = a.pairs / unit + ((a.dim - 2 * a.pairs) / unit + 1) / 2;
  a.tokens = batch * a.len;
  a.vec_fp32 = vec_dtype == LBW_DTYPE_FP32;
  a.team = 4;
  while (a.team < 64 && a.team < items) a.team *= 2;
  // a few rows a team, as long as there are workgroups for every CU
  const int64_t rows = a.q.heads + a.k.heads;
  a.per_group = 1;
  while (a.per_group < MAX_TOKENS && a.per_group * rows * a.team < 4 * THREADS && a.tokens / (2 * a.per_group) >= 1024) a.per_group *= 2;
  const int64_t groups = (a.tokens + a.per_group - 1) / a.per_group, grid = BWD ? std::min<int64_t>(groups, MAX_GROUPS) : groups;
  if (dtype == LBW_DTYPE_BF16) launch_by_unit<LBW_DTYPE_BF16, BWD>(a, unit, inter, grid, stream);
  else if (dtype == LBW_DTYPE_FP16) launch_by_unit<LBW_DTYPE_FP16, BWD>(a, unit, inter, grid, stream);
  else launch_by_unit<LBW_DTYPE_FP32, BWD>(a, unit, inter, grid, stream);
  if (BWD && a.partial) {
    const unsigned n = (2 * a.dim + 15) / 16;
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
