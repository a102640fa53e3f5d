// Rotary positions (include/lbw_block.h): q and k read once, rotated in registers, written once. Bound by memory.
//
// A workgroup takes a few tokens. Their angles are formed once for all heads: position * frequency in 64 bits,
// reduced to (-1/2, 1/2] turns there (far positions lose nothing: an angle of 1e6 radians is still good to 1e-10),
// then sine and cosine in fp32 of the reduced angle rounded to fp32, into LDS. 16-bit values do not see that rounding;
// for fp32 values both are moved by what it took off (standard normal values: 4.1e-8 rms off, 5.4e-8 without; sine and
// cosine in 64 bits 3.7e-8, but 64 tokens of 14 heads 3.27 us against 3.07). The heads' values then pass through
// registers, 16 bytes a load: with neighbouring pairs a load holds whole pairs; with halves a thread takes the 16
// bytes of both partners. 6032 tokens of 24 heads of 128 in bf16 take 13.4 us (5.5 TB/s; a copy of 1 GiB reaches 5.1), 24 of
// their 96 channels turned 11.6 with 8-byte units (53 value by value).
#include "lbw_turn.h"

namespace lbw {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_TOKENS = 8;   // of a workgroup
constexpr int MAX_PAIRS = LBW_ROTARY_MAX_DIM / 2;

struct Tensor {
  const void* in;
  void* out;
  int64_t heads, s_batch, s_tok, s_head, o_batch, o_tok, o_head;
};

struct RotaryArgs {
  Tensor q, k;
  int64_t tokens, len;            // tokens of all entries, and of one
  int dim, pairs, per_group;      // per_group: tokens of a workgroup
  const void* pos;
  int pos_is_i64;
  int64_t p_s_batch, p_s_tok, p_s_axis, pos_start;
  const double* freq;
  const int32_t* axis;
  int64_t axes;
  float factor, sign;             // sign -1: the inverse rotation
  int copy;                       // whether the channels past the pairs have to be written (not in place)
};

// N: values of a unit (16 bytes of the format, 8, or one value, as strides, sizes and addresses allow). An item is
// two units: those of partners (with INTER N pairs, 2 N channels in a row, else N channels in each half), or two
// neighbouring ones of the channels past the pairs, which are copied.
template <int DT, int N, bool INTER>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryArgs a) {
  // Items whose loads are in flight together: with whole units more waves do better than more loads a wave (bf16,
  // 6032 tokens of 24 heads of 128: 13.4 us with one, 13.9 with two, 16.4 with four), single values need them (8
  // heads of 80: 10.7 with four, 15.2).
  constexpr int U = N == 1 ? 4 : 1;
  __shared__ float2 cs[MAX_TOKENS * MAX_PAIRS];
  __shared__ int64_t at_tok[MAX_TOKENS][4];   // where a token's rows start: q, k, and in the outputs
  const int64_t tok0 = (int64_t)group_id() * a.per_group;
  if (tok0 >= a.tokens) return;
  const int ntok = (int)min((int64_t)a.per_group, a.tokens - tok0);
  if (threadIdx.x < ntok) {
    const uint32_t tok = (uint32_t)(tok0 + threadIdx.x), b = tok / (uint32_t)a.len, t = tok - b * (uint32_t)a.len;
    at_tok[threadIdx.x][0] = b * a.q.s_batch + t * a.q.s_tok;
    at_tok[threadIdx.x][1] = b * a.k.s_batch + t * a.k.s_tok;
    at_tok[threadIdx.x][2] = b * a.q.o_batch + t * a.q.o_tok;
    at_tok[threadIdx.x][3] = b * a.k.o_batch + t * a.k.o_tok;
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
    cs[i] = make_float2(a.factor * c, a.sign * a.factor * s);
  }
  __syncthreads();
  const int pair_items = a.pairs / N, rest = a.copy ? (a.dim - 2 * a.pairs) / N : 0;   // (units of the rest)
  const uint32_t items = pair_items + (rest + 1) / 2;
  const uint32_t heads = (uint32_t)(a.q.heads + a.k.heads), total = ntok * heads * items;
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += U * THREADS) {
    Unit<DT, N> u[U], v[U];
    char *out0[U], *out1[U];   // null: nothing there
    int pair[U];               // the item's first pair in cs, or -1
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const uint32_t i = i0 + n * THREADS;
      out0[n] = out1[n] = nullptr;
      pair[n] = -1;
      if (i >= total) continue;
      const uint32_t row = i / items, j = row / heads, h = row - j * heads;
      const int it = (int)(i - row * items);
      const bool is_q = h < (uint32_t)a.q.heads;
      const int64_t src = at_tok[j][is_q ? 0 : 1] + (is_q ? h * a.q.s_head : (h - a.q.heads) * a.k.s_head);
      const int64_t dst = at_tok[j][is_q ? 2 : 3] + (is_q ? h * a.q.o_head : (h - a.q.heads) * a.k.o_head);
      const char* in = (const char*)(is_q ? a.q.in : a.k.in) + src * elem_size(DT);
      char* out = (char*)(is_q ? a.q.out : a.k.out) + dst * elem_size(DT);
      const bool turned = it < pair_items;
      const int p = it * N, r0 = 2 * a.pairs + 2 * (it - pair_items) * N;
      const int c0 = turned ? (INTER ? 2 * p : p) : r0, c1 = turned && !INTER ? a.pairs + p : c0 + N;
      u[n].load(in, c0);
      out0[n] = out + c0 * elem_size(DT);
      if (turned || c1 < a.dim) {
        v[n].load(in, c1);
        out1[n] = out + c1 * elem_size(DT);
      }
      if (turned) pair[n] = (int)j * a.pairs + p;
    }
#pragma unroll
    for (int n = 0; n < U; ++n) {
      if (!out0[n]) continue;
      if (pair[n] >= 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          // pair e: in a row the values 2 e, 2 e + 1 of both units, else value e of each
          float& f0 = INTER && N > 1 ? (2 * e < N ? u[n].f[2 * e % N] : v[n].f[2 * e % N]) : u[n].f[e];
          float& f1 = INTER && N > 1 ? (2 * e < N ? u[n].f[(2 * e + 1) % N] : v[n].f[(2 * e + 1) % N]) : v[n].f[e];
          const float x0 = f0, x1 = f1;
          const float2 w = cs[pair[n] + e];
          f0 = x0 * w.x - x1 * w.y;
          f1 = x1 * w.x + x0 * w.y;
        }
      }
      u[n].store(out0[n], 0);
      if (out1[n]) v[n].store(out1[n], 0);
    }
  }
}

template <int DT, int N>
void launch(const RotaryArgs& a, bool inter, int64_t grid, hipStream_t stream) {
  if (inter) rotary_kernel<DT, N, true><<<grid_of(grid), THREADS, 0, stream>>>(a);
  else rotary_kernel<DT, N, false><<<grid_of(grid), THREADS, 0, stream>>>(a);
}

template <int DT>
void launch_by_unit(const RotaryArgs& a, int unit, bool inter, int64_t grid, hipStream_t stream) {
  if (unit == 8) {
    if constexpr (DT != LBW_DTYPE_FP32) launch<DT, 8>(a, inter, grid, stream);
  } else if (unit == 4) {
    launch<DT, 4>(a, inter, grid, stream);
  } else {
    launch<DT, 1>(a, inter, grid, stream);
  }
}

}  // namespace
}  // namespace lbw

using namespace lbw;

extern "C" int lbw_rotary(const void* q, const void* k, int dtype, int64_t batch, int64_t len, int64_t q_heads,
                          int64_t k_heads, int64_t dim, int64_t pairs, int64_t q_s_batch, int64_t q_s_tok,
                          int64_t q_s_head, int64_t k_s_batch, int64_t k_s_tok, int64_t k_s_head,
                          const void* positions, int pos_is_i64, int64_t p_s_batch, int64_t p_s_tok, int64_t p_s_axis,
                          int64_t pos_start, const double* freq, const int32_t* axis, int64_t axes, int interleaved,
                          int inverse, float factor, void* q_out, void* k_out, int64_t qo_s_batch, int64_t qo_s_tok,
                          int64_t qo_s_head, int64_t ko_s_batch, int64_t ko_s_tok, int64_t ko_s_head, void* stream) {
  if (!q || !q_out || !freq || (k_heads > 0 && (!k || !k_out))) return LBW_E_NULL;
  if (dtype < 0 || dtype > LBW_DTYPE_FP32 || batch < 1 || len < 1 || batch > (1 << 30) || len > (1 << 30) ||
      batch * len > (1 << 30) || q_heads < 1 || k_heads < 0 || q_heads > 4096 || k_heads > 4096 || dim < 2 ||
      dim > LBW_ROTARY_MAX_DIM || pairs < 1 || 2 * pairs > dim || axes < 1)
    return LBW_E_SHAPE;
  const int es = elem_size(dtype);
  const int64_t strides[] = {q_s_batch, q_s_tok, q_s_head, k_s_batch, k_s_tok, k_s_head,
                             qo_s_batch, qo_s_tok, qo_s_head, ko_s_batch, ko_s_tok, ko_s_head};
  // the widest unit that sizes, strides and addresses are multiples of
  const auto fits = [&](int64_t n) {
    bool ok = dim % n == 0 && pairs % n == 0;
    for (int i = 0; i < 12; ++i)
      if (k_heads || i % 6 < 3) ok = ok && strides[i] % n == 0;
    for (const void* p : {q, (const void*)q_out, k_heads ? k : nullptr, k_heads ? (const void*)k_out : nullptr})
      ok = ok && (uintptr_t)p % (n * es) == 0;
    return ok;
  };
  if (!fits(1)) return LBW_E_ALIGN;
  const int unit = es == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
  if ((uintptr_t)freq % 8 || (uintptr_t)axis % 4 || (uintptr_t)positions % (pos_is_i64 ? 8 : 4)) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  RotaryArgs a = {{q, q_out, q_heads, q_s_batch, q_s_tok, q_s_head, qo_s_batch, qo_s_tok, qo_s_head},
                  {k, k_out, k_heads, k_s_batch, k_s_tok, k_s_head, ko_s_batch, ko_s_tok, ko_s_head},
                  batch * len, len, (int)dim, (int)pairs, 1, positions, pos_is_i64, p_s_batch, p_s_tok, p_s_axis,
                  pos_start, freq, axis, axes, factor, inverse ? -1.f : 1.f, q != q_out || (k_heads && k != k_out)};
  // a few items a thread, as long as there are workgroups for every CU
  const int64_t items = (q_heads + k_heads) * dim / (2 * unit);
  while (a.per_group < MAX_TOKENS && a.per_group * items < 4 * THREADS && a.tokens / (2 * a.per_group) >= 1024)
    a.per_group *= 2;
  const int64_t grid = (a.tokens + a.per_group - 1) / a.per_group;
  if (dtype == LBW_DTYPE_BF16) launch_by_unit<LBW_DTYPE_BF16>(a, unit, interleaved, grid, (hipStream_t)stream);
  else if (dtype == LBW_DTYPE_FP16) launch_by_unit<LBW_DTYPE_FP16>(a, unit, interleaved, grid, (hipStream_t)stream);
  else launch_by_unit<LBW_DTYPE_FP32>(a, unit, interleaved, grid, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
