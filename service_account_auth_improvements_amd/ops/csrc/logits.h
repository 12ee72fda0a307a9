// Shared pieces of the kernels that walk rows of logits (token_logprobs.hip, distill_topk.hip).
//
// A row of V logits (bf16, fp16 or fp32, any row stride, any alignment of the element type) is cut
// into pieces of 16 bytes: N = 8 or 4 logits each, V / N full ones and a tail of V % N.  A piece is
// one load or store per thread whatever the row's alignment: gfx950 takes global accesses of any
// alignment, and odd vocabularies put most rows off a 16-byte boundary (load_pieces: what is done
// about rows off a 4-byte one).
//
// Softmax arithmetic is base 2 with the temperature folded in: a = log2(e) / temperature, and for
// the row's greatest logit m,  s = sum 2^((x - m) a),  log2 p_j = (x_j - m) a - log2 s.  The
// difference x - m is formed first, though x a - m a would be one instruction less (1.5 % of the
// distillation's time): it is exact where it matters (x near m), however great m is, and stays
// finite for logits at the type's lowest value, where x a would overflow.
#pragma once
#include <tuple>
#include <type_traits>

#include "common.h"

namespace kf {

enum { DT_BF16 = 0, DT_FP16 = 1, DT_FP32 = 2 };
constexpr float LN2 = 0.69314718055994531f, LOG2E = 1.4426950408889634f;
// stands for x - m = -inf in products with 2^((x - m) a) = 0: far enough for that at every
// temperature taken (1e-4 to 1e4), and finite when multiplied by a sum over any row
constexpr float FAR = -1e25f;
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fc00000u); }

typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t u32x4_a2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;

template <int DT> struct Elem {
  static constexpr int bytes = DT == DT_FP32 ? 4 : 2;
  static constexpr int N = 16 / bytes;
  static constexpr u32 neg_inf = DT == DT_BF16 ? 0xff80ff80u : DT == DT_FP16 ? 0xfc00fc00u : 0xff800000u;   // a word of -inf
};

template <int DT>
__device__ __forceinline__ u32x4 load_piece(const char* row, int c) {
  return *(const u32x4_a2*)(row + 16L * c);
}
template <int DT>
__device__ __forceinline__ void unpack_piece(const u32x4& v, float* f) {
  if constexpr (DT == DT_BF16) {
    unpack8(v, f);
  } else if constexpr (DT == DT_FP16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2_t h = __builtin_bit_cast(f16x2_t, (u32)v[i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
  }
}
// one rounding, to nearest even, at the store
template <int DT>
__device__ __forceinline__ u32x4 pack_piece(const float* f) {
  if constexpr (DT == DT_BF16) return pack8(f);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == DT_FP16) r[i] = __builtin_bit_cast(u32, f16x2_t{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
    else r[i] = __float_as_uint(f[i]);
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void store_piece(char* row, int c, const float* f) {
  *(u32x4_a2*)(row + 16L * c) = pack_piece<DT>(f);
}

template <int DT>
__device__ __forceinline__ float load1(const void* row, long e) {
  if constexpr (DT == DT_BF16) return bf2f(((const bf16_t*)row)[e]);
  if constexpr (DT == DT_FP16) return (float)((const _Float16*)row)[e];
  return ((const float*)row)[e];
}
__device__ __forceinline__ float load1_as(int dt, const void* row, long e) {
  return dt == DT_BF16 ? load1<DT_BF16>(row, e) : dt == DT_FP16 ? load1<DT_FP16>(row, e) : load1<DT_FP32>(row, e);
}
template <int DT>
__device__ __forceinline__ void store1(void* row, long e, float f) {
  if constexpr (DT == DT_BF16) ((bf16_t*)row)[e] = f2bf(f);
  else if constexpr (DT == DT_FP16) ((_Float16*)row)[e] = (_Float16)f;
  else ((float*)row)[e] = f;
}

// piece c of a row of V logits; what lies behind the row's end reads as `fill`
template <int DT>
__device__ __forceinline__ void load_any(const char* row, int c, int V, float fill, float* f) {
  constexpr int N = Elem<DT>::N;
  if (c < V / N) {
    unpack_piece<DT>(load_piece<DT>(row, c), f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = (long)N * c + j < V ? load1<DT>(row, (long)N * c + j) : fill;
  }
}
// v[j] = full piece at(j) of a row.  Accesses off a 4-byte boundary run at half the rate, so where a
// row starts off one, a piece is put together from the 5 words it lies in: the values and their order
// are the same wherever the row lies.  Half the rows of an odd vocabulary: 1661 rows of 133153 bf16
// logits 81 us (97 without this; 133152: 79).
template <int DT, int UN, typename At>
__device__ __forceinline__ void load_pieces(const char* row, At at, u32x4 (&v)[UN]) {
  if (DT != DT_FP32 && ((u32)(size_t)row & 2)) {
    u32 last[UN];                                // right behind its piece, whose lines are in the L1 then
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      v[j] = load_piece<DT>(row - 2, at(j));
      last[j] = *(const u32*)(row - 2 + 16L * at(j) + 16);
    }
#pragma unroll
    for (int j = 0; j < UN; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) v[j][w] = __builtin_amdgcn_alignbit(w < 3 ? v[j][w + 1] : last[j], v[j][w], 16);
  } else {
#pragma unroll
    for (int j = 0; j < UN; ++j) v[j] = load_piece<DT>(row, at(j));
  }
}
template <int DT>
__device__ __forceinline__ void store_any(char* row, int c, int V, const float* f) {
  constexpr int N = Elem<DT>::N;
  if (c < V / N) {
    store_piece<DT>(row, c, f);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if ((long)N * c + j < V) store1<DT>(row, (long)N * c + j, f[j]);
  }
}
template <int DT>
__device__ __forceinline__ float max_piece(const float* f) {
  float m = fmaxf(f[0], f[1]);
#pragma unroll
  for (int j = 2; j < Elem<DT>::N; ++j) m = fmaxf(m, f[j]);
  return m;
}

// A barrier for what the block exchanges through LDS: loads from and stores to global memory stay in
// flight across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---- reductions by DPP moves: no LDS round trips inside a wave, no address registers; the results
// are uniform.  Every lane of the wave takes part.
struct OpMax { __device__ __forceinline__ float operator()(float p, float q) const { return fmaxf(p, q); } };
struct OpAdd { __device__ __forceinline__ float operator()(float p, float q) const { return p + q; } };
template <int CTRL, int ROWS, typename Op>
__device__ __forceinline__ float dpp_step(float v, float neutral, Op op) {
  return op(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(neutral), __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
// lane 15 of each row of 16 lanes holds the row's result
template <typename Op>
__device__ __forceinline__ float row_reduce(float v, float neutral, Op op) {
  v = dpp_step<0x111, 0xf>(v, neutral, op);      // row_shr by 1, 2, 4, 8
  v = dpp_step<0x112, 0xf>(v, neutral, op);
  v = dpp_step<0x114, 0xf>(v, neutral, op);
  return dpp_step<0x118, 0xf>(v, neutral, op);
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
template <typename Op>
__device__ __forceinline__ float wave_reduce(float v, float neutral, Op op) {
  v = row_reduce(v, neutral, op);
  v = dpp_step<0x142, 0xa>(v, neutral, op);      // row_bcast:15 into rows 1 and 3
  v = dpp_step<0x143, 0xc>(v, neutral, op);      // row_bcast:31 into rows 2 and 3
  return lane_value(v, 63);
}
__device__ __forceinline__ u32 wave_max(u32 v) {           // 0 is neutral
  const auto step = [&](auto ctrl, auto rows) {
    v = max(v, (u32)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return (u32)__builtin_amdgcn_readlane((int)v, 63);
}
// `red` holds NT / 64 values and is not written again before another barrier
template <int NT, typename Op>
__device__ __forceinline__ float block_reduce(float v, float neutral, float* red, Op op, int tid) {
  v = wave_reduce(v, neutral, op);
  if ((tid & 63) == 0) red[tid >> 6] = v;
  lds_barrier();
  const int l = tid & 15;
  return lane_value(row_reduce(l < NT / 64 ? red[l] : neutral, neutral, op), 15);
}
// a sum in 64 bits, of what the first `waves` waves (four at most) hold; the others skip it
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  const u32x2 p = __builtin_bit_cast(u32x2, v);
  u32x2 q;
#pragma unroll
  for (int i = 0; i < 2; ++i) q[i] = (u32)__builtin_amdgcn_update_dpp(0, (int)p[i], CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(double, q);
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  u32x2 p = __builtin_bit_cast(u32x2, v);
#pragma unroll
  for (int i = 0; i < 2; ++i) p[i] = (u32)__builtin_amdgcn_readlane((int)p[i], lane);
  return __builtin_bit_cast(double, p);
}
__device__ __forceinline__ double block_sum(double v, int waves, double* red, int tid) {
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (wave < waves) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    v = lane_value(dpp_add<0x143, 0xc>(v), 63);
    if ((tid & 63) == 0) red[wave] = v;
  }
  lds_barrier();
  v = (tid & 3) < waves ? red[tid & 3] : 0.0;
  return lane_value(dpp_add<0x112, 0xf>(dpp_add<0x111, 0xf>(v)), 3);
}

// Running softmax of a row part: m = greatest logit, s = sum 2^((x-m) a), and for the entropy (MOMENT)
// u = sum (x-m) 2^((x-m) a).  An empty part is {-inf, 0, 0}, and so is one whose logits are all -inf.
// A NaN or +inf logit makes s NaN.
enum { MOMENT = 0, PLAIN = 1 };
struct RowStat {
  float m, s, u;
};
__device__ __forceinline__ RowStat stat_empty() { return {-INFINITY, 0.f, 0.f}; }

// what x - m is formed with: 0 for m = -inf, so that -inf logits give 2^-inf = 0 and not NaN
__device__ __forceinline__ float stat_ref(float m) { return m == -INFINITY ? 0.f : m; }

// moves the part to the greater reference mn (>= r.m)
template <int KIND>
__device__ __forceinline__ void stat_move(RowStat& r, float mn, float a) {
  // r.m = -inf: nothing but zeros was summed; else the shift is finite, or -inf below a +inf mn
  const float d = r.m == -INFINITY ? 0.f : fmaxf(r.m - mn, FAR);
  const float f = __builtin_amdgcn_exp2f(d * a);
  if constexpr (KIND == MOMENT) r.u = f * fmaf(d, r.s, r.u);
  r.s *= f;
  r.m = mn;
}
// adds one logit to s (and u); ref = stat_ref(r.m)
template <int KIND>
__device__ __forceinline__ void stat_add(RowStat& r, float ref, float x, float a) {
  const float d = x - ref;
  const float e = __builtin_amdgcn_exp2f(d * a);
  r.s += e;
  if constexpr (KIND == MOMENT) r.u = fmaf(fmaxf(d, FAR), e, r.u);   // d = -inf: 0, not -inf * 0
}
template <int KIND, int LANES>
__device__ __forceinline__ RowStat lanes_stat(RowStat r, float a) {
  const float m = LANES == 64 ? wave_reduce(r.m, -INFINITY, OpMax{}) : lane_value(row_reduce(r.m, -INFINITY, OpMax{}), 15);
  stat_move<KIND>(r, m, a);
  if constexpr (LANES == 64)
    return {m, wave_reduce(r.s, 0.f, OpAdd{}), KIND == PLAIN ? 0.f : wave_reduce(r.u, 0.f, OpAdd{})};
  else
    return {m, lane_value(row_reduce(r.s, 0.f, OpAdd{}), 15), KIND == PLAIN ? 0.f : lane_value(row_reduce(r.u, 0.f, OpAdd{}), 15)};
}
template <int KIND, int NT>
__device__ __forceinline__ RowStat block_stat(RowStat r, float a, RowStat* red, int tid) {
  r = lanes_stat<KIND, 64>(r, a);
  if ((tid & 63) == 0) red[tid >> 6] = r;
  lds_barrier();
  const int l = tid & 15;
  return lanes_stat<KIND, 16>(l < NT / 64 ? red[l] : stat_empty(), a);
}

// two parts at once; in waves from `waves` on p is q
template <int NT>
__device__ __forceinline__ void block_stat2(RowStat& p, RowStat& q, int waves, float a, RowStat (*red)[2], int tid) {
  q = lanes_stat<PLAIN, 64>(q, a);
  p = __builtin_amdgcn_readfirstlane(tid >> 6) < waves ? lanes_stat<PLAIN, 64>(p, a) : q;
  if ((tid & 63) == 0) { red[tid >> 6][0] = p; red[tid >> 6][1] = q; }
  lds_barrier();
  const int l = tid & 15;
  p = lanes_stat<PLAIN, 16>(l < NT / 64 ? red[l][0] : stat_empty(), a);
  q = lanes_stat<PLAIN, 16>(l < NT / 64 ? red[l][1] : stat_empty(), a);
}

constexpr long ROWS_PER_LAUNCH = 1 << 20;   // a launch holds less than 2^32 threads

// Launches kernels; rc is 0 or, from LAUNCH_RC on, the first launch's error.
constexpr int LAUNCH_RC = 1000;
struct Launcher {
  int rc = 0;
  template <typename... P, typename... A>
  void operator()(void (*kernel)(P...), unsigned grid, unsigned block, size_t lds, hipStream_t s, A... a) {
    std::tuple<P...> args(static_cast<P>(a)...);
    const hipError_t e = std::apply([&](P&... p) {
      void* at[] = {(void*)&p...};
      return hipLaunchKernel((const void*)kernel, dim3(grid), dim3(block), at, lds, s);
    }, args);
    if (rc == 0 && e != hipSuccess) rc = LAUNCH_RC + (int)e;
  }
};

// f(std::integral_constant<int, DT>) for the type dt
template <typename F>
inline void by_type(int dt, F f) {
  if (dt == DT_BF16) f(std::integral_constant<int, DT_BF16>{});
  else if (dt == DT_FP16) f(std::integral_constant<int, DT_FP16>{});
  else f(std::integral_constant<int, DT_FP32>{});
}

}  // namespace kf
