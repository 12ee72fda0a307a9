// Shared pieces of the kernels that walk rows of logits (token_logprobs.hip, distill_topk.hip).
//
// A row of V logits (bf16, fp16 or fp32, any row stride, any alignment of the element type) is cut
// into chunks of 8 elements; chunk c holds elements [8c, 8c + 8), the last one possibly fewer.  A
// thread's loads are 16 bytes whatever the row's alignment: gfx950 takes global accesses of any
// alignment, and odd vocabularies put most rows off a 16-byte boundary.
//
// Softmax arithmetic is base 2 with the temperature folded in: a = log2(e) / temperature, and for
// the row's greatest logit m,  s = sum 2^((x - m) a),  log2 p_j = (x_j - m) a - log2 s.  The
// difference x - m is formed first: it is exact where it matters (x near m) and stays finite for
// logits at the type's lowest value, where x * a would overflow.
#pragma once
#include "common.h"

namespace kf {

enum { DT_BF16 = 0, DT_FP16 = 1, DT_FP32 = 2 };
constexpr float LN2 = 0.69314718055994531f;
// stands for x - m = -inf in products with 2^((x - m) a) = 0: far enough for that at every
// temperature taken (1e-4 to 1e4), and finite when multiplied by a sum over any row
constexpr float FAR = -1e25f;

typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t u32x4_a2;
typedef __attribute__((ext_vector_type(4), aligned(4))) float f32x4_a4;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;

template <int DT> struct Elem { static constexpr int bytes = DT == DT_FP32 ? 4 : 2; };

// 8 logits as they lie in memory: 4 registers for the 16-bit types, 8 for fp32
template <int DT> struct Raw8 { u32x4 v[DT == DT_FP32 ? 2 : 1]; };

template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* row, long e) {
  Raw8<DT> r;
  const char* p = (const char*)row + e * Elem<DT>::bytes;
  if constexpr (DT == DT_FP32) {
    r.v[0] = __builtin_bit_cast(u32x4, *(const f32x4_a4*)p);
    r.v[1] = __builtin_bit_cast(u32x4, *(const f32x4_a4*)(p + 16));
  } else {
    r.v[0] = *(const u32x4_a2*)p;
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack_raw(const Raw8<DT>& r, float* f) {
  if constexpr (DT == DT_BF16) {
    unpack8(r.v[0], f);
  } else if constexpr (DT == DT_FP16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2_t h = __builtin_bit_cast(f16x2_t, (u32)r.v[0][i]);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(r.v[i >> 2][i & 3]);
  }
}

template <int DT>
__device__ __forceinline__ float load1(const void* row, long e) {
  if constexpr (DT == DT_BF16) return bf2f(((const bf16_t*)row)[e]);
  if constexpr (DT == DT_FP16) return (float)((const _Float16*)row)[e];
  return ((const float*)row)[e];
}

// one rounding, to nearest even, at the store
template <int DT>
__device__ __forceinline__ void store1(void* row, long e, float f) {
  if constexpr (DT == DT_BF16) ((bf16_t*)row)[e] = f2bf(f);
  else if constexpr (DT == DT_FP16) ((_Float16*)row)[e] = (_Float16)f;
  else ((float*)row)[e] = f;
}

template <int DT>
__device__ __forceinline__ void store8(void* row, long e, const float* f) {
  char* p = (char*)row + e * Elem<DT>::bytes;
  if constexpr (DT == DT_FP32) {
    *(f32x4_a4*)p = f32x4{f[0], f[1], f[2], f[3]};
    *(f32x4_a4*)(p + 16) = f32x4{f[4], f[5], f[6], f[7]};
  } else if constexpr (DT == DT_BF16) {
    *(u32x4_a2*)p = pack8(f);
  } else {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = __builtin_bit_cast(u32, f16x2_t{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
    *(u32x4_a2*)p = r;
  }
}

// chunk c of a row of V elements; elements behind the row's end read as `fill`
template <int DT>
__device__ __forceinline__ void load_chunk(const void* row, int c, int V, float fill, float* f) {
  const long e = 8L * c;
  if (e + 8 <= V) {
    unpack_raw<DT>(load8<DT>(row, e), f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = e + j < V ? load1<DT>(row, e + j) : fill;
  }
}
template <int DT>
__device__ __forceinline__ void store_chunk(void* row, int c, int V, const float* f) {
  const long e = 8L * c;
  if (e + 8 <= V) {
    store8<DT>(row, e, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e + j < V) store1<DT>(row, e + j, f[j]);
  }
}

__device__ __forceinline__ float max8(const float* f) {
  float m = fmaxf(f[0], f[1]);
#pragma unroll
  for (int j = 2; j < 8; ++j) m = fmaxf(m, f[j]);
  return m;
}

// Running softmax of a row part: m = greatest logit, s = sum 2^((x-m) a), u = sum (x-m) 2^((x-m) a)
// (the entropy's sum).  An empty part is {-inf, 0, 0}; a part whose logits are all -inf is too.
// A NaN or +inf logit makes s NaN.
struct RowStat {
  float m, s, u;
};
__device__ __forceinline__ RowStat stat_empty() { return {-INFINITY, 0.f, 0.f}; }

// what x - m is formed with: 0 for m = -inf, so that -inf logits give 2^-inf = 0 and not NaN
__device__ __forceinline__ float stat_ref(float m) { return m == -INFINITY ? 0.f : m; }

// moves the part to the greater reference mn (>= r.m)
__device__ __forceinline__ void stat_move(RowStat& r, float mn, float a) {
  if (mn == r.m) return;
  // r.m = -inf: nothing but zeros was summed; else the shift is finite, or -inf below a +inf mn
  const float d = r.m == -INFINITY ? 0.f : fmaxf(r.m - mn, FAR);
  const float f = __builtin_amdgcn_exp2f(d * a);
  r.u = f * fmaf(d, r.s, r.u);
  r.s *= f;
  r.m = mn;
}
__device__ __forceinline__ RowStat stat_join(RowStat x, RowStat y, float a) {
  const float mn = fmaxf(x.m, y.m);
  stat_move(x, mn, a);
  stat_move(y, mn, a);
  return {mn, x.s + y.s, x.u + y.u};
}
// adds one logit: ref = stat_ref(r.m)
__device__ __forceinline__ void stat_add(RowStat& r, float ref, float x, float a) {
  const float d = x - ref;
  const float e = __builtin_amdgcn_exp2f(d * a);
  r.s += e;
  r.u = fmaf(fmaxf(d, FAR), e, r.u);   // d = -inf: 0, not -inf * 0
}

template <int NT>
__device__ __forceinline__ RowStat block_stat(RowStat r, float a, RowStat* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    r = stat_join(r, RowStat{__shfl_xor(r.m, o, 64), __shfl_xor(r.s, o, 64), __shfl_xor(r.u, o, 64)}, a);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = r;
    __syncthreads();
    r = red[0];
#pragma unroll
    for (int k = 1; k < NT / 64; ++k) r = stat_join(r, red[k], a);
  }
  return r;
}

}  // namespace kf
