// Rotary positions (include/lbw_block.h): q and k read once, rotated in registers, written once. Bound by memory.
//
// A workgroup takes a few tokens. Their angles are formed once for all heads: position * frequency in 64 bits, reduced to
// (-1/2, 1/2] turns there (far positions lose nothing: an angle of 1e6 radians is still good to 1e-10), then sine and cosine of
// the reduced angle in fp32, into LDS. The heads' values then pass through registers, 16 bytes a load: with neighbouring pairs
// a load holds whole pairs; with halves a thread takes the 16 bytes of both partners.
#include "lbw_rows.h"

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

// N consecutive values (16 bytes, or one)
template <int DT, int N>
struct Unit {
  float f[N];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (N == 1) {
      f[0] = load1<DT>(p, i);
    } else {
      const v4i w = *(const v4i*)((const char*)p + i * elem_size(DT));
      if constexpr (DT == LBW_DTYPE_FP32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __int_as_float(w[e]);
      } else {
        unpack8t<DT == LBW_DTYPE_FP16>(w, f);
      }
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t i) const {
    if constexpr (N == 1) {
      store1<DT>(p, i, f[0]);
    } else {
      v4i w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == LBW_DTYPE_FP32) w[e] = __float_as_int(f[e]);
        else w[e] = (int)pack2<DT>(f[2 * e], f[2 * e + 1]);
      }
      *(v4i*)((char*)p + i * elem_size(DT)) = w;
    }
  }
};

// N: values of a unit (16 bytes of the format, or 1 where strides, sizes or addresses do not allow that). An item is one unit
// of channels past the pairs, or the units a, b of partners: with INTER those of N pairs (2 N channels in a row), else of N
// channels in each half.
template <int DT, int N, bool INTER>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 cs[MAX_TOKENS * MAX_PAIRS];
  const int64_t tok0 = (int64_t)blockIdx.x * a.per_group;
  const int ntok = (int)min((int64_t)a.per_group, a.tokens - tok0);
  for (int i = threadIdx.x; i < ntok * a.pairs; i += THREADS) {
    const int j = i / a.pairs, p = i - j * a.pairs;
    const int64_t tok = tok0 + j, b = tok / a.len, t = tok - b * a.len;
    // an axis outside the positions' would read past them: held inside
    const int64_t ax = a.axis ? max((int64_t)0, min((int64_t)a.axis[p], a.axes - 1)) : 0;
    const int64_t at = b * a.p_s_batch + t * a.p_s_tok + ax * a.p_s_axis;
    const int64_t pos = !a.pos ? a.pos_start + t : a.pos_is_i64 ? ((const int64_t*)a.pos)[at] : ((const int32_t*)a.pos)[at];
    const double turns = (double)pos * a.freq[p] * 0.15915494309189533577;   // 1 / (2 pi)
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[i] = make_float2(a.factor * c, a.sign * a.factor * s);
  }
  __syncthreads();
  const int pair_items = a.pairs / N;
  const int items = pair_items + (a.copy ? (a.dim - 2 * a.pairs) / N : 0);
  const int heads = (int)(a.q.heads + a.k.heads);
  const int total = ntok * heads * items;
  for (int i = threadIdx.x; i < total; i += THREADS) {
    const int row = i / items, it = i - row * items, j = row / heads;
    int h = row - j * heads;
    const bool is_q = h < a.q.heads;
    const Tensor& x = is_q ? a.q : a.k;
    if (!is_q) h -= (int)a.q.heads;
    const int64_t tok = tok0 + j, b = tok / a.len, t = tok - b * a.len;
    const int64_t src = b * x.s_batch + t * x.s_tok + h * x.s_head, dst = b * x.o_batch + t * x.o_tok + h * x.o_head;
    if (it < pair_items) {
      const int p = it * N;
      const int c0 = INTER ? 2 * p : p, c1 = INTER ? c0 + N : a.pairs + p;
      Unit<DT, N> u, v;
      u.load(x.in, src + c0);
      v.load(x.in, src + c1);
      const float2* w = cs + j * a.pairs + p;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        // pair e: in a row the values 2 e, 2 e + 1 of both units, else value e of each
        float& f0 = INTER && N > 1 ? (2 * e < N ? u.f[2 * e % N] : v.f[2 * e % N]) : u.f[e];
        float& f1 = INTER && N > 1 ? (2 * e < N ? u.f[(2 * e + 1) % N] : v.f[(2 * e + 1) % N]) : v.f[e];
        const float x0 = f0, x1 = f1;
        f0 = x0 * w[e].x - x1 * w[e].y;
        f1 = x1 * w[e].x + x0 * w[e].y;
      }
      u.store(x.out, dst + c0);
      v.store(x.out, dst + c1);
    } else {
      const int c = 2 * a.pairs + (it - pair_items) * N;
      Unit<DT, N> u;
      u.load(x.in, src + c);
      u.store(x.out, dst + c);
    }
  }
}

template <int DT, int N>
void launch(const RotaryArgs& a, bool inter, int64_t grid, hipStream_t stream) {
  if (inter) rotary_kernel<DT, N, true><<<(unsigned)grid, THREADS, 0, stream>>>(a);
  else rotary_kernel<DT, N, false><<<(unsigned)grid, THREADS, 0, stream>>>(a);
}

template <int DT>
void launch_by_unit(const RotaryArgs& a, bool wide, bool inter, int64_t grid, hipStream_t stream) {
  if (wide) launch<DT, 16 / elem_size(DT)>(a, inter, grid, stream);
  else launch<DT, 1>(a, inter, grid, stream);
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
  const int64_t n = 16 / es;
  const int64_t strides[] = {q_s_batch, q_s_tok, q_s_head, k_s_batch, k_s_tok, k_s_head,
                             qo_s_batch, qo_s_tok, qo_s_head, ko_s_batch, ko_s_tok, ko_s_head};
  bool wide = dim % n == 0 && pairs % n == 0;
  for (int i = 0; i < 12; ++i)
    if (k_heads || i % 6 < 3) wide = wide && strides[i] % n == 0;
  for (const void* p : {q, (const void*)q_out, k_heads ? k : nullptr, k_heads ? (const void*)k_out : nullptr}) {
    if ((uintptr_t)p % es) return LBW_E_ALIGN;
    wide = wide && (uintptr_t)p % 16 == 0;
  }
  if ((uintptr_t)freq % 8 || (uintptr_t)axis % 4 || (uintptr_t)positions % (pos_is_i64 ? 8 : 4)) return LBW_E_ALIGN;
  if (const int st = check_device()) return st;
  RotaryArgs a = {{q, q_out, q_heads, q_s_batch, q_s_tok, q_s_head, qo_s_batch, qo_s_tok, qo_s_head},
                  {k, k_out, k_heads, k_s_batch, k_s_tok, k_s_head, ko_s_batch, ko_s_tok, ko_s_head},
                  batch * len, len, (int)dim, (int)pairs, 1, positions, pos_is_i64, p_s_batch, p_s_tok, p_s_axis,
                  pos_start, freq, axis, axes, factor, inverse ? -1.f : 1.f, q != q_out || (k_heads && k != k_out)};
  // a few items a thread, as long as there are workgroups for every CU
  const int64_t items = (q_heads + k_heads) * dim / (2 * (wide ? n : 1));
  while (a.per_group < MAX_TOKENS && a.per_group * items < 4 * THREADS && a.tokens / (2 * a.per_group) >= 1024)
    a.per_group *= 2;
  const int64_t grid = (a.tokens + a.per_group - 1) / a.per_group;
  if (dtype == LBW_DTYPE_BF16) launch_by_unit<LBW_DTYPE_BF16>(a, wide, interleaved, grid, (hipStream_t)stream);
  else if (dtype == LBW_DTYPE_FP16) launch_by_unit<LBW_DTYPE_FP16>(a, wide, interleaved, grid, (hipStream_t)stream);
  else launch_by_unit<LBW_DTYPE_FP32>(a, wide, interleaved, grid, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? LBW_OK : LBW_E_LAUNCH;
}
