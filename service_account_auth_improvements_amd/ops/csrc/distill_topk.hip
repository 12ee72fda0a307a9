// Distillation from a teacher's top logits: the divergence of a row's softmax p (over V logits x,
// at a temperature) from the teacher's distribution q over K given ids, and its gradient.
//
//   q = softmax(z / temperature) over the row's entries, r = 0                (no teacher lse)
//   q = exp(z / temperature - lse), r = max(0, 1 - sum q) the teacher's rest  (with it)
//   loss = sum q (ln q - ln p_id) + r (ln r - ln R),      R = sum of p outside the ids
//   dx_j = (p_j W - q_j) / temperature          inside,   W = sum q + r
//   dx_j = p_j (W - r / R) / temperature        outside
//
// An entry with a negative id is no entry; a row without entries (or with q = 0 throughout) has
// loss 0 and gradient 0 and is not read.  Where the student has no mass outside (R = 0) the rest is
// left out.  An id at or behind the vocabulary's end makes its row NaN.
//
// One block per row.  The outside sum is summed over the outside elements (one bit per element in
// LDS tells them), not formed as 1 - sum p_id, which loses everything when the student is sure.
#include "logits.h"

#include <type_traits>

using namespace kf;

namespace {

enum { KD_FUSED = 0, KD_STATS = 1, KD_GRAD = 2 };
constexpr int K_MAX = 256;           // one thread per entry in the smallest block
constexpr size_t BITS_MAX = 61440;   // bytes of LDS for the bit per element: 491520 logits

struct Teacher {
  const void* ids;       // int64 or int32 [T, K], rows ldi apart
  const void* z;         // logits' row of any of the three types, rows ldz apart
  const float* lse;      // [T] or null
  long ldi, ldz;
  int ids32, zt, K;
};

template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) t = fmaxf(t, red[i]);
  return t;
}

// the row's sums without the entropy's; `u` is the sum outside the ids
__device__ __forceinline__ void sums_move(RowStat& r, float mn, float a) {
  if (mn == r.m) return;
  const float f = __builtin_amdgcn_exp2f((r.m == -INFINITY ? 0.f : fmaxf(r.m - mn, FAR)) * a);
  r.u *= f;
  r.s *= f;
  r.m = mn;
}
__device__ __forceinline__ RowStat sums_join(RowStat x, RowStat y, float a) {
  const float mn = fmaxf(x.m, y.m);
  sums_move(x, mn, a);
  sums_move(y, mn, a);
  return {mn, x.s + y.s, x.u + y.u};
}

constexpr int UN = 4;

template <int DT, int NT, bool REST>
__device__ __forceinline__ RowStat walk_sums(const void* row, int V, float a, const unsigned char* inside) {
  const int nfull = V >> 3;
  RowStat st = stat_empty();
  float f[UN][8];
  auto eat = [&](int c0, int n) {
    float bm = -INFINITY;
#pragma unroll
    for (int j = 0; j < UN; ++j)
      if (j < n) bm = fmaxf(bm, max8(f[j]));
    sums_move(st, fmaxf(st.m, bm), a);
    const float ref = stat_ref(st.m);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (j >= n) continue;
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[j][i] = __builtin_amdgcn_exp2f((f[j][i] - ref) * a);
        part += f[j][i];
      }
      st.s += part;
      if constexpr (REST) {
        const int c = c0 + j * NT;
        const u32 bits = 8 * c < V ? inside[c] : 0u;
        if (bits) {                                  // few chunks hold an id
          part = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) part += (bits >> i & 1) ? 0.f : f[j][i];
        }
        st.u += part;
      }
    }
  };
  int c = threadIdx.x;
  for (; c + (UN - 1) * NT < nfull; c += UN * NT) {
    Raw8<DT> r[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j) r[j] = load8<DT>(row, 8L * (c + j * NT));
#pragma unroll
    for (int j = 0; j < UN; ++j) unpack_raw<DT>(r[j], f[j]);
    eat(c, UN);
  }
  if (c < nfull) {
    Raw8<DT> r[UN];
#pragma unroll
    for (int j = 0; j < UN; ++j) r[j] = load8<DT>(row, 8L * (c + j * NT < nfull ? c + j * NT : nfull - 1));
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      unpack_raw<DT>(r[j], f[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = c + j * NT < nfull ? f[j][i] : -INFINITY;
    }
    eat(c, UN);
  }
  if ((V & 7) && (int)threadIdx.x == nfull % NT) {
    load_chunk<DT>(row, nfull, V, -INFINITY, f[0]);
    eat(nfull, 1);
  }
  return st;
}

template <int DT, int NT, int MODE, bool REST>
__global__ __launch_bounds__(NT) void distill_kernel(const void* logits, long ld, void* out, long ldo, int V, long vstart,
                                                     long vtotal, Teacher te, float temp, const float* scale_ptr,
                                                     float scale_h, const float* rows, float* loss, float* stats,
                                                     long lds) {
  __shared__ RowStat red3[NT / 64];
  __shared__ float red[NT / 64];
  __shared__ int sid[K_MAX];
  __shared__ float sq[K_MAX];
  __shared__ float sx[K_MAX];                      // the student's logits at the ids, read before any store
  extern __shared__ u32 bits[];                    // REST: one bit per element
  const float inv_temp = 1.f / temp, a = 1.4426950408889634f * inv_temp;
  const float NaN = __uint_as_float(0x7fc00000u);
  const long r = blockIdx.x;
  const int tid = threadIdx.x, K = te.K;
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  char* orow = (char*)out + r * ldo * Elem<DT>::bytes;
  const int nchunk = (V + 7) >> 3, nword = (nchunk + 3) >> 2;

  // ---- the teacher's row: thread k holds entry k
  long id = -1;
  float z = -INFINITY;
  if (tid < K) {
    id = te.ids32 ? ((const int*)te.ids)[r * te.ldi + tid] : ((const long*)te.ids)[r * te.ldi + tid];
    if (id >= 0)
      z = te.zt == DT_BF16 ? load1<DT_BF16>(te.z, r * te.ldz + tid)
          : te.zt == DT_FP16 ? load1<DT_FP16>(te.z, r * te.ldz + tid) : load1<DT_FP32>(te.z, r * te.ldz + tid);
  }
  if constexpr (REST)
    for (int i = tid; i < nword; i += NT) bits[i] = 0;
  const bool bad = __syncthreads_or(id >= vtotal);
  const bool mine = id >= vstart && id < vstart + V;       // inside this part of the vocabulary
  const int col = mine ? (int)(id - vstart) : -1;
  float lq, q;                                              // ln q and q
  if constexpr (REST) {
    lq = fmaf(z, inv_temp, -te.lse[r]);
    q = id >= 0 ? __builtin_amdgcn_exp2f(lq * 1.4426950408889634f) : 0.f;
    if (mine) atomicOr(&bits[col >> 5], 1u << (col & 31));
  } else {
    const float mz = block_max<NT>(z, red);
    z -= stat_ref(mz);
    q = id >= 0 ? __builtin_amdgcn_exp2f(z * a) : 0.f;
    const float n = block_sum<NT>(q, red);
    lq = z * inv_temp - LN2 * __log2f(n);
    q = n == 0.f ? 0.f : q / n;
  }
  const bool some = __syncthreads_or(q != 0.f);
  const float sc = (rows ? rows[r] : 1.f) * (scale_ptr ? scale_ptr[0] : scale_h) / temp;
  if (!some || bad) {
    const float v = bad ? NaN : 0.f;
    if (tid == 0 && loss) loss[r] = v;
    if (MODE == KD_STATS) {
      if (tid < 5) stats[5 * r + tid] = v;
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v;
      for (int c = tid; c < nchunk; c += NT) store_chunk<DT>(orow, c, V, f);
    }
    return;
  }
  const float x = mine ? load1<DT>(row, col) : 0.f;
  if (tid < K) { sid[tid] = col; sq[tid] = q; sx[tid] = x; }
  const float Q = block_sum<NT>(q, red);
  const float rest = REST ? fmaxf(1.f - Q, 0.f) : 0.f;
  const float W = Q + rest;

  // ---- the student's row
  float m, s, u;
  if constexpr (MODE == KD_GRAD) {
    m = stats[r * lds];
    s = stats[r * lds + 1];
    u = stats[r * lds + 2];
    __syncthreads();
  } else {
    RowStat st = walk_sums<DT, NT, REST>(row, V, a, (const unsigned char*)bits);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      st = sums_join(st, RowStat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.u, o, 64)}, a);
    if ((tid & 63) == 0) red3[tid >> 6] = st;
    __syncthreads();
    st = red3[0];
#pragma unroll
    for (int k = 1; k < NT / 64; ++k) st = sums_join(st, red3[k], a);
    m = st.m;
    s = st.s;
    u = st.u;
  }
  const float L = __log2f(s);
  const bool use_rest = REST && rest > 0.f && !(u == 0.f);
  if (MODE == KD_STATS || loss) {
    // entries of q = 0 add nothing, whatever the student gives them
    const bool own = MODE != KD_GRAD && mine;
    const float xq = block_sum<NT>(own && q != 0.f ? q * (x - m) : 0.f, red);
    if constexpr (MODE == KD_STATS) {
      const float ql = block_sum<NT>(own ? q : 0.f, red);
      if (tid == 0) {
        stats[5 * r] = m;
        stats[5 * r + 1] = s;
        stats[5 * r + 2] = u;
        stats[5 * r + 3] = xq;
        stats[5 * r + 4] = ql;
      }
    }
    if (loss) {
      float l;
      if constexpr (MODE == KD_GRAD) {
        l = block_sum<NT>(q != 0.f ? q * (lq + LN2 * L) : 0.f, red) - inv_temp * stats[r * lds + 3];
      } else {
        l = block_sum<NT>(q != 0.f ? q * (lq - ((x - m) * inv_temp - LN2 * L)) : 0.f, red);
      }
      if (use_rest) l += rest * LN2 * (__log2f(rest) - (__log2f(u) - L));
      if (tid == 0) loss[r] = l;
    }
  }
  if constexpr (MODE == KD_STATS) return;

  // ---- gradient: every element as one outside, then the ids' own
  const float cout = sc * (use_rest ? W - rest * s / u : W);
  for (int c = tid; c < nchunk; c += NT) {
    float f[8];
    load_chunk<DT>(row, c, V, 0.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = cout * __builtin_amdgcn_exp2f(fmaf(f[i] - m, a, -L));
    store_chunk<DT>(orow, c, V, f);
  }
  __syncthreads();
  if (mine) {
    float qs = 0.f;                      // an id given twice: both entries, stored twice alike
    for (int k = 0; k < K; ++k) qs += sid[k] == col ? sq[k] : 0.f;
    store1<DT>(orow, col, sc * (W * __builtin_amdgcn_exp2f(fmaf(sx[tid] - m, a, -L)) - qs));
  }
}

constexpr long ROWS_PER_LAUNCH = 1 << 20;   // a launch holds less than 2^32 threads

}  // namespace

extern "C" {

int kf_distill_k_max() { return K_MAX; }
long kf_distill_rest_v_max() { return 8L * BITS_MAX; }

// mode 0: loss rows and gradient; 1: local statistics [T, 5] (m, s, outside sum, sum q (x - m), sum
// q of the ids of this part) and, with `loss`, the loss of an undivided vocabulary; 2: gradient
// (and loss) from the joined statistics [T, 4],
// or [T, 5] of an undivided vocabulary (ld_stats)
int kf_distill_topk(const void* logits, int dt, long ld, void* out, long ldo, long rows, int V, long vstart, long vtotal,
                    const void* ids, int ids32, long ldi, const void* z, int zt, long ldz, const float* lse, int K,
                    float temp, const float* scale_ptr, float scale_h, const float* row_scale, float* loss, float* stats,
                    long ld_stats, int mode, hipStream_t s) {
  if (V < 1 || K < 0 || K > K_MAX || dt < DT_BF16 || dt > DT_FP32 || zt < DT_BF16 || zt > DT_FP32) return 1;
  const size_t lds = lse ? ((size_t)(V + 7) / 8 + 3) / 4 * 4 : 0;
  if (lds > BITS_MAX) return 2;
  for (long r0 = 0; r0 < rows; r0 += ROWS_PER_LAUNCH) {
    const int n = (int)std::min(ROWS_PER_LAUNCH, rows - r0);
    auto go = [&](auto DTc, auto NTc, auto Mc, auto Rc) {
      constexpr int DT = decltype(DTc)::value, NT = decltype(NTc)::value, MODE = decltype(Mc)::value;
      constexpr bool REST = decltype(Rc)::value;
      const Teacher te{(const char*)ids + r0 * ldi * (ids32 ? 4 : 8), (const char*)z + r0 * ldz * (zt == DT_FP32 ? 4 : 2),
                       lse ? lse + r0 : nullptr, ldi, ldz, ids32, zt, K};
      distill_kernel<DT, NT, MODE, REST><<<n, NT, lds, s>>>(
          (const char*)logits + r0 * ld * Elem<DT>::bytes, ld, out ? (char*)out + r0 * ldo * Elem<DT>::bytes : nullptr, ldo,
          V, vstart, vtotal, te, temp, scale_ptr, scale_h, row_scale ? row_scale + r0 : nullptr, loss ? loss + r0 : nullptr,
          stats ? stats + r0 * ld_stats : nullptr, ld_stats);
    };
    auto by_rest = [&](auto DTc, auto NTc, auto Mc) {
      if (lse) go(DTc, NTc, Mc, std::true_type{});
      else go(DTc, NTc, Mc, std::false_type{});
    };
    auto by_mode = [&](auto DTc, auto NTc) {
      if (mode == KD_FUSED) by_rest(DTc, NTc, std::integral_constant<int, KD_FUSED>{});
      else if (mode == KD_STATS) by_rest(DTc, NTc, std::integral_constant<int, KD_STATS>{});
      else by_rest(DTc, NTc, std::integral_constant<int, KD_GRAD>{});
    };
    auto by_size = [&](auto DTc) {
      if (V > 16384) by_mode(DTc, std::integral_constant<int, 1024>{});
      else by_mode(DTc, std::integral_constant<int, 256>{});
    };
    if (dt == DT_BF16) by_size(std::integral_constant<int, DT_BF16>{});
    else if (dt == DT_FP16) by_size(std::integral_constant<int, DT_FP16>{});
    else by_size(std::integral_constant<int, DT_FP32>{});
  }
  return 0;
}

}  // extern "C"
