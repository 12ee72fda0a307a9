// Distillation from a teacher's top logits: the divergence of a row's softmax p (over V logits x,
// at a temperature) from the teacher's distribution q over K given ids, and its gradient.
//
//   q = softmax(z / temperature) over the row's entries, r = 0                (no teacher lse)
//   q = exp(z / temperature - lse), r = max(0, 1 - sum q) the teacher's rest  (with it)
//   loss = sum q (ln q - ln p_id) + r (ln r - ln R),      R = sum of p outside the ids
//   dx_j = (p_j W - q_j) / temperature          inside,   W = sum q + r
//   dx_j = o_j (W R - r) / temperature          outside,  o_j = p_j / R
//
// An entry with a negative id is no entry; a row without entries (or with q = 0 throughout) has
// loss 0 and gradient 0.  Where the student has no mass outside (nothing but -inf) the rest is left
// out.  An id at or behind the vocabulary's end makes its row NaN.
//
// The outside sum is summed over the outside elements, not formed as 1 - sum p_id, which loses
// everything when the student is sure, and against their own greatest logit mo:  u = sum 2^((x - mo) a),
// R = u 2^((mo - m) a) / s.  Against the row's, u would be flushed to 0, and 1 / R overflow, from a
// distance of 87 nats on; so R may vanish, o and ln R = (mo - m) / temperature + ln u - ln s do not.
#include "logits.h"

using namespace kf;

namespace {

typedef unsigned long long u64;
enum { KD_FUSED = 0, KD_STATS = 1, KD_GRAD = 2 };
constexpr int K_MAX = 256;           // one thread per entry in the smallest block
constexpr size_t BITS_MAX = 61440;   // bytes of LDS for a bit per element: 491520 logits
constexpr int BAD = 0x7fffffff;      // an id behind the vocabulary

// a row's statistics between the two halves: the student's (m, s, mo, u, sum q (x - m), sum q of this
// part's ids) and the teacher's (greatest z and sum without lse, else r and sum q) and the row's state
// (0 no entries, 1 entries, NaN an id behind the vocabulary)
enum { ST_M, ST_S, ST_MO, ST_U, ST_XQ, ST_QL, ST_ZM, ST_ZN, ST_LIVE, ST_COLS, ST_REST = ST_ZM };

// k = (W R - r) / u, with  dx_j = k 2^((x_j - mo) a) / temperature  outside.  u and s are 0 (nothing but
// -inf), 1 or more, or NaN; k is 0 where u is, and NaN where s is 0.
__device__ __forceinline__ float outside_factor(float m, float s, float mo, float u, float W, float rest, float a) {
  const float R = u * __builtin_amdgcn_exp2f((mo - m) * a) * __builtin_amdgcn_rcpf(s);
  return (W * R - (u == 0.f ? 0.f : rest)) * __builtin_amdgcn_rcpf(fmaxf(u, 1.f));
}
// r (ln r - ln R): the rest's share of the loss
__device__ __forceinline__ float rest_loss(float m, float L, float mo, float u, float rest, float inv_temp) {
  if (!(rest > 0.f) || u == 0.f) return 0.f;
  return rest * (LN2 * (__log2f(rest) - __log2f(u) + L) - (mo - m) * inv_temp);
}

// e^x in 64 bits, to a relative 1e-12: (e^(f / 8))^8 2^n with x = n ln 2 + f and six terms of the series.
// It needs few constants: those of exp() would take 24 scalar registers from row to row, and one of the
// fused kernel's would be spilled.
__device__ __forceinline__ double exp64(double x) {
  x = x < -800.0 ? -800.0 : x > 800.0 ? 800.0 : x;       // 0 and infinity; NaN passes
  const double n = rint(x * 1.4426950408889634);
  const double g = ldexp(fma(n, -0.69314718055994531, x), -3);
  double p = fma(g, 1.0 / 720, 1.0 / 120);
  p = fma(g, p, 1.0 / 24);
  p = fma(g, p, 1.0 / 6);
  p = fma(g, p, 0.5);
  p = fma(g, p, 1.0);
  p = fma(g, p, 1.0);
  p *= p;
  p *= p;
  return ldexp(p * p, (int)n);
}

struct Teacher {
  const void* ids;       // int64 or int32 [T, K], rows ldi apart
  const void* z;         // logits' row of any of the three types, rows ldz apart
  const float* lse;      // [T] or null
  double inv_temp;
  long ldi, ldz, vocab;
  int ids32, zt, K;
  // entry k of row r: -1 none, BAD behind the vocabulary
  __device__ __forceinline__ void entry(long r, int k, int& id, float& v) const {
    id = -1;
    v = -INFINITY;
    if (k < K) {
      const long i = ids32 ? ((const int*)ids)[r * ldi + k] : ((const long*)ids)[r * ldi + k];
      v = load1_as(zt, z, r * ldz + k);
      id = i < 0 ? -1 : i >= vocab ? BAD : (int)i;
    }
    if (id < 0) v = -INFINITY;
  }
  // q against the teacher's whole mass, and ln q.  In 64 bits: r = 1 - sum q is often small, and at
  // r = 1e-6 would be off by some per cent, and the outside's gradient with it, were q an fp32 exponential.
  __device__ __forceinline__ double mass(long r, int id, float v, float& lq) const {
    lq = -INFINITY;
    if (id < 0) return 0.0;
    const double l = (double)v * inv_temp - (double)lse[r];
    lq = (float)l;
    return exp64(l);
  }
};

// ---------------------------------------------------------------- rows of up to 256 KB: read once
//
// The row stays in the block's registers (16 pieces a thread) between the sums and the gradient, and
// the block walks rows, reading each piece of its next row as the piece of this row leaves: the
// loads of one row and the stores of another are in flight while the exponentials are computed.
// 4096 rows of 128256 bf16 logits: 443 us (4.7 TB/s; a copy of the same bytes takes 365), where
// two passes over rows, the second from the caches, take 525 and a block per row without the
// reads ahead takes 600.  Groups of pieces behind a row's end are jumped over by the whole block:
// 4096 rows of 4000 bf16 logits take 25 us, and 70 where every thread goes through all sixteen.
// Rows that four pieces a thread of the smallest block hold leave registers for half as many
// blocks more on a CU: 20 us.
constexpr int RES_MAX = 16, RES_SHORT = 4;       // pieces of a thread
constexpr int GRP = 2;               // pieces summed together

// piece j of thread t; behind the last full piece: some full piece
template <int NT>
__device__ __forceinline__ u32x4 load_mine(const char* row, int j, int nfull, int t) {
  const int rem = nfull - j * NT;
  const int last = rem < 1 ? 0 : rem > NT ? NT - 1 : rem - 1;
  const char* base = row + (rem > 0 ? j * NT * 16 : 0);
  return *(const u32x4_a2*)(base + (size_t)(u32)(min(t, last) * 16));
}

// 128 registers a thread: 16 waves fill a CU; of rows of RES_SHORT 24 (32 would be as fast, with
// scalar registers spilled)
constexpr int fused_waves(int res) { return res == RES_SHORT ? 6 : 4; }

template <int DT, int NT, int RES, bool REST>
__global__ __launch_bounds__(NT, fused_waves(RES)) void distill_fused_kernel(
    const void* logits, long ld, void* out, long ldo, long T, int V, Teacher te, float temp, const float* scale_ptr,
    float scale_h, float* loss, int keep) {
  constexpr int N = Elem<DT>::N;
  __shared__ float red[5][NT / 64];
  __shared__ RowStat red3[NT / 64][2];
  __shared__ int head[NT];                               // a thread's own ids: a list through next
  __shared__ int sid[K_MAX], next[K_MAX];
  __shared__ float sq[K_MAX], slq[K_MAX], sx[K_MAX], sqs[K_MAX];
  __shared__ double redq[NT / 64];
  const float inv_temp = 1.f / temp, a = LOG2E * inv_temp;
  const int tid0 = threadIdx.x, K = te.K, kwaves = (K + 63) / 64;      // waves whose threads hold entries
  const int nfull0 = V / N, ntail = V % N;
  const float sc = (scale_ptr ? scale_ptr[0] : scale_h) * inv_temp;
  auto row_at = [&](long r) { return (const char*)logits + r * ld * Elem<DT>::bytes; };
  long r = blockIdx.x;
  int id;
  float z, x = 0.f;
  te.entry(r, tid0, id, z);
  if (id >= 0 && id < V) x = load1<DT>(row_at(r), id);
  u32x4 b[RES];
#pragma unroll
  for (int j = 0; j < RES; ++j) b[j] = load_mine<NT>(row_at(r), j, nfull0, tid0);
  float xt = tid0 < ntail ? load1<DT>(row_at(r), (long)N * nfull0 + tid0) : 0.f;
  for (; r < T; r += gridDim.x) {
    // opaque copies: what depends on them is not kept in registers from row to row
    int tid = tid0, nfull = nfull0;
    asm volatile("" : "+v"(tid), "+s"(nfull));
    const long rn = r + gridDim.x;
    const bool more = rn < T;
    const char* rown = row_at(more ? rn : r);
    char* orow = (char*)out + r * ldo * Elem<DT>::bytes;
    // the thread that holds an element: that of its piece, or of its place in the tail
    auto owner = [&](int c) { return c < N * nfull ? (c / N) % NT : c - N * nfull; };
    // ---- the teacher's row: thread k holds entry k
    head[tid] = 0;
    const bool mine = id >= 0 && id < V;
    const bool bad = block_reduce<NT>(id == BAD ? 1.f : 0.f, 0.f, red[0], OpMax{}, tid) != 0.f;
    float W = 1.f, rest = 0.f;
    bool some;
    {
      float lq, q;
      if constexpr (REST) {
        const double qd = te.mass(r, id, z, lq), Q = block_sum(qd, kwaves, redq, tid);
        q = (float)qd;
        some = !(Q == 0.0);
        rest = (float)fmax(1.0 - Q, 0.0);
        W = (float)Q + rest;
      } else {
        const float zm = block_reduce<NT>(z, -INFINITY, red[1], OpMax{}, tid);
        z -= stat_ref(zm);
        q = id >= 0 ? __builtin_amdgcn_exp2f(z * a) : 0.f;
        const float n = block_reduce<NT>(q, 0.f, red[2], OpAdd{}, tid);
        lq = z * inv_temp - LN2 * __log2f(n);
        q = n == 0.f ? 0.f : q / n;
        some = !(n == 0.f);
        if (n != n) W = n;                               // a NaN entry: the whole row
      }
      if (tid < K) { sid[tid] = mine ? id : -1; sq[tid] = q; slq[tid] = lq; sx[tid] = x; }
      if (mine) next[tid] = atomicExch(&head[owner(id)], tid + 1);
    }
    lds_barrier();
    bool first = mine;                                   // of the entries with this id
    if (mine) {
      // the same id twice: its entries add up.  They are in one list; its order is that of the
      // atomics, so the sum is formed in the order of the entries
      bool twice = false;
      for (int h = head[owner(id)]; h; h = next[h - 1]) {
        const bool same = h - 1 != tid && sid[h - 1] == id;
        twice = twice || same;
        first = first && !(same && h - 1 < tid);
      }
      float qs = sq[tid];
      if (twice) {
        qs = 0.f;
        for (int k = 0; k < K; ++k) qs += sid[k] == id ? sq[k] : 0.f;
      }
      sqs[tid] = qs;
    }
    if (!some || bad) {
      // nothing of the student's row counts, NaN least of all
#pragma unroll
      for (int j = 0; j < RES; ++j) b[j] = u32x4{0, 0, 0, 0};
      xt = 0.f;
      first = false;
    } else if constexpr (REST) {
      // the ids' elements read as -inf: what is summed then lies outside
      for (int h = head[tid]; h; h = next[h - 1]) {
        const int c = sid[h - 1];
        if (c >= N * nfull) {
          xt = -INFINITY;
        } else {
          const int at = (c / N / NT) * 4 + (c % N) * Elem<DT>::bytes / 4;     // which of the 4 RES words
          const u32 kept = DT == DT_FP32 ? 0u : (c & 1) ? 0xffffu : 0xffff0000u;
          const u32 fill = Elem<DT>::neg_inf & ~kept;
#pragma unroll
          for (int j = 0; j < RES; ++j) {
            if (__ballot(at >> 2 == j) == 0) continue;       // no thread of the wave has one in this piece
#pragma unroll
            for (int w = 0; w < 4; ++w) b[j][w] = at == 4 * j + w ? (b[j][w] & kept) | fill : b[j][w];
          }
        }
      }
    }
    if (more) te.entry(rn, tid, id, z);
    // ---- sums, each piece as it arrives
    RowStat st = stat_empty();
#pragma unroll
    for (int g = 0; g < RES; g += GRP) {
      if (g * NT >= nfull) continue;                     // behind the end for the whole block
      float f[GRP][N];
      float bm = st.m;
#pragma unroll
      for (int j = 0; j < GRP; ++j) {
        asm volatile("" : "+v"(b[g + j]), "+v"(st.m), "+v"(st.s));     // one group after the other
        unpack_piece<DT>(b[g + j], f[j]);
        if ((g + j + 1) * NT > nfull) {
#pragma unroll
          for (int i = 0; i < N; ++i) f[j][i] = (g + j) * NT + tid < nfull ? f[j][i] : -INFINITY;
        }
        bm = fmaxf(bm, max_piece<DT>(f[j]));
      }
      stat_move<PLAIN>(st, bm, a);
      const float ref = stat_ref(bm);
#pragma unroll
      for (int j = 0; j < GRP; ++j)
#pragma unroll
        for (int i = 0; i < N; ++i) stat_add<PLAIN>(st, ref, f[j][i], a);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (tid < ntail) {
      stat_move<PLAIN>(st, fmaxf(st.m, xt), a);
      stat_add<PLAIN>(st, stat_ref(st.m), xt, a);
    }
    RowStat so = st;                                     // what lies outside
    if constexpr (REST) {
      if (first) {
        const float v = sx[tid];
        stat_move<PLAIN>(st, fmaxf(st.m, v), a);
        stat_add<PLAIN>(st, stat_ref(st.m), v, a);
      }
    }
#pragma unroll
    for (int j = 0; j < RES; ++j) asm volatile("" : "+v"(b[j]));        // unpacked anew below, not kept
    asm volatile("" : "+s"(nfull));                      // nor are the comparisons with it
    if constexpr (REST) block_stat2<NT>(st, so, kwaves, a, red3, tid);
    else st = block_stat<PLAIN, NT>(st, a, red3[0], tid);
    const float m = st.m, L = __log2f(st.s);
    if (more && id >= 0 && id < V) x = load1<DT>(rown, id);
    // ---- gradient; each piece of the next row is read as this row's leaves.  ci: 0 without
    // entries, NaN for a bad row
    const bool live = some && !bad;
    const float ci = bad ? quiet_nan() : some ? sc : 0.f;
    const float kW = ci * W, k1 = REST ? ci * outside_factor(m, st.s, so.m, so.s, W, rest, a) : kW;
    const float ref = REST ? stat_ref(so.m) : m, shift = REST ? 0.f : -L;
    if (tid < ntail) {
      const float p = __builtin_amdgcn_exp2f(fmaf(xt - ref, a, shift));
      store1<DT>(orow, (long)N * nfull + tid, k1 * p);
      xt = load1<DT>(rown, (long)N * nfull + tid);
    }
#pragma unroll
    for (int j = 0; j < RES; ++j) {
      if (j * NT >= nfull) continue;
      float f[N];
      unpack_piece<DT>(b[j], f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = k1 * __builtin_amdgcn_exp2f(fmaf(f[i] - ref, a, shift));
      u32x4 piece = pack_piece<DT>(f);
      asm volatile("" : "+v"(piece));                      // done with b[j] before it is loaded again
      b[j] = load_mine<NT>(rown, j, nfull, tid);
      int oj = j * NT * 16;
      asm volatile("" : "+s"(oj));
      if (j * NT + tid < nfull) {
        u32x4_a2* at = (u32x4_a2*)(orow + oj + (size_t)(u32)(tid * 16));
        if (keep) {
          *at = piece;
        } else {
          asm volatile("; past the caches");             // what keeps the two stores from becoming one
          __builtin_nontemporal_store(piece, at);
          asm volatile("");
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // the ids' own elements, by the thread that stored the pieces around them, behind those stores
    asm volatile("" ::: "memory");
    for (int h = head[tid]; h; h = next[h - 1]) {
      const float p = __builtin_amdgcn_exp2f(fmaf(sx[h - 1] - m, a, -L));
      store1<DT>(orow, sid[h - 1], live ? fmaf(p, kW, -ci * sqs[h - 1]) : ci);
    }
    const float q = tid < K ? sq[tid] : 0.f;             // entries of q = 0 add nothing, whatever the student gives them
    float l = q != 0.f ? q * (slq[tid] - ((sx[tid] - m) * inv_temp - LN2 * L)) : 0.f;
    l = block_reduce<NT>(l, 0.f, red[4], OpAdd{}, tid);
    if (tid == 0) {
      if constexpr (REST) l += rest_loss(m, L, so.m, so.s, rest, inv_temp);
      loss[r] = bad ? quiet_nan() : some ? l : 0.f;
    }
  }
}

// ---------------------------------------------------------------- statistics: one block per row
// the sums of a thread's pieces; REST: of what lies outside, and the ids' elements go into `in`
template <int DT, int NT, bool REST>
__device__ __forceinline__ RowStat walk_sums(const char* row, int V, float a, const u32* bits, RowStat& in) {
  constexpr int N = Elem<DT>::N, UN = 4;
  const int nfull = V / N;
  RowStat st = stat_empty();
  in = stat_empty();
  float f[UN][N];
  auto eat = [&](int c0, int n) {
    if constexpr (REST) {
#pragma unroll
      for (int j = 0; j < UN; ++j) {
        if (j >= n) continue;
        const long e = (long)N * (c0 + j * NT);
        const u32 here = e < V ? bits[e >> 5] >> (e & 31) & ((1u << N) - 1) : 0u;
        if (here == 0) continue;                         // few pieces hold an id
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if ((here >> i & 1) == 0) continue;
          stat_move<PLAIN>(in, fmaxf(in.m, f[j][i]), a);
          stat_add<PLAIN>(in, stat_ref(in.m), f[j][i], a);
          f[j][i] = -INFINITY;
        }
      }
    }
    float bm = st.m;
#pragma unroll
    for (int j = 0; j < UN; ++j)
      if (j < n) bm = fmaxf(bm, max_piece<DT>(f[j]));
    if (bm != st.m) stat_move<PLAIN>(st, bm, a);
    const float ref = stat_ref(st.m);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (j >= n) continue;
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) part += __builtin_amdgcn_exp2f((f[j][i] - ref) * a);
      st.s += part;
    }
  };
  for (int c = threadIdx.x; c < nfull; c += UN * NT) {
    u32x4 v[UN];
    load_pieces<DT>(row, [&](int j) { return min(c + j * NT, nfull - 1); }, v);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      unpack_piece<DT>(v[j], f[j]);
      if (c + j * NT >= nfull)
#pragma unroll
        for (int i = 0; i < N; ++i) f[j][i] = -INFINITY;
    }
    eat(c, UN);
  }
  if (V % N && (int)threadIdx.x == nfull % NT) {
    load_any<DT>(row, nfull, V, -INFINITY, f[0]);
    eat(nfull, 1);
  }
  return st;
}

template <int DT, int NT, bool REST>
__global__ __launch_bounds__(NT, 8) void distill_stats_kernel(const void* __restrict__ logits, long ld, int V,
                                                              long vstart, Teacher te, float temp,
                                                              float* __restrict__ loss, float* __restrict__ stats) {
  __shared__ float red[6][NT / 64];
  __shared__ RowStat red3[NT / 64][2];
  __shared__ double redq[NT / 64];
  extern __shared__ u32 bits[];                          // REST: one bit per element
  const float inv_temp = 1.f / temp, a = LOG2E * inv_temp;
  const long r = blockIdx.x;
  const int tid = threadIdx.x;
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  int id;
  float z, lq, q, zm = 0.f, n, rest = 0.f;
  te.entry(r, tid, id, z);
  const bool mine = id >= vstart && id < vstart + V;     // inside this part of the vocabulary
  const float x = mine ? load1<DT>(row, id - vstart) : 0.f;
  if constexpr (REST)
    for (int i = tid; i < (V + 31) / 32; i += NT) bits[i] = 0;
  const bool bad = block_reduce<NT>(id == BAD ? 1.f : 0.f, 0.f, red[0], OpMax{}, tid) != 0.f;
  bool some;
  if constexpr (REST) {
    if (mine) atomicOr(&bits[(id - vstart) >> 5], 1u << ((id - vstart) & 31));
    const double qd = te.mass(r, id, z, lq), Q = block_sum(qd, (te.K + 63) / 64, redq, tid);
    q = (float)qd;
    n = (float)Q;
    some = !(Q == 0.0);
    rest = (float)fmax(1.0 - Q, 0.0);
  } else {
    zm = block_reduce<NT>(z, -INFINITY, red[1], OpMax{}, tid);
    z -= stat_ref(zm);
    q = id >= 0 ? __builtin_amdgcn_exp2f(z * a) : 0.f;
    n = block_reduce<NT>(q, 0.f, red[2], OpAdd{}, tid);
    lq = z * inv_temp - LN2 * __log2f(n);
    q = n == 0.f ? 0.f : q / n;
    some = !(n == 0.f);
  }
  float* st_row = stats + r * ST_COLS;
  if (!some || bad) {
    const float v = bad ? quiet_nan() : 0.f;
    if (tid == 0) loss[r] = v;
    if (tid < ST_COLS) st_row[tid] = v;
    return;
  }
  RowStat in, so = walk_sums<DT, NT, REST>(row, V, a, bits, in), st = so;
  if constexpr (REST) {
    // the ids' elements join the rest of the row
    const float mn = fmaxf(st.m, in.m);
    stat_move<PLAIN>(st, mn, a);
    stat_move<PLAIN>(in, mn, a);
    st.s += in.s;
    block_stat2<NT>(st, so, NT / 64, a, red3, tid);
  } else {
    st = block_stat<PLAIN, NT>(st, a, red3[0], tid);
    so = stat_empty();
  }
  const float L = __log2f(st.s);
  // entries of q = 0 add nothing, whatever the student gives them
  const bool use = mine && q != 0.f;
  // (a part of nothing but -inf: its ids' logits, against 0)
  const float xq = block_reduce<NT>(use ? q * (x - stat_ref(st.m)) : 0.f, 0.f, red[3], OpAdd{}, tid);
  const float ql = block_reduce<NT>(mine ? q : 0.f, 0.f, red[4], OpAdd{}, tid);
  float l = block_reduce<NT>(use ? q * (lq - ((x - st.m) * inv_temp - LN2 * L)) : 0.f, 0.f, red[5], OpAdd{}, tid);
  if (tid == 0) {
    if constexpr (REST) l += rest_loss(st.m, L, so.m, so.s, rest, inv_temp);
    loss[r] = l;
    const float row_stats[ST_COLS] = {st.m, st.s, so.m, so.s, xq, ql, REST ? rest : stat_ref(zm), n, 1.f};
#pragma unroll
    for (int i = 0; i < ST_COLS; ++i) st_row[i] = row_stats[i];
  }
}

// ---------------------------------------------------------------- gradient from statistics
//
// One block per 4 pieces a thread of a row, in the order of the addresses (4096 rows of 128256 bf16
// logits: 2048 blocks that walk longer parts are half as fast): streams, and forms q again from the
// statistics for the ids in its own columns.
constexpr int GRAD_NT = 256, GRAD_UN = 4;

template <int DT, bool REST>
__global__ __launch_bounds__(GRAD_NT) void distill_grad_kernel(const void* logits, long ld, void* out, long ldo, int V,
                                                               int parts, long vstart, Teacher te, float temp,
                                                               const float* scale_ptr, float scale_h,
                                                               const float* __restrict__ rows, float* __restrict__ loss,
                                                               const float* __restrict__ stats) {
  constexpr int N = Elem<DT>::N, W4 = GRAD_NT / 64;
  __shared__ float red[W4], sq[K_MAX], sx[K_MAX], sqs[K_MAX];
  __shared__ int cnt[W4], scol[K_MAX], head[GRAD_NT], next[K_MAX];
  const float inv_temp = 1.f / temp, a = LOG2E * inv_temp;
  const long r = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - r * parts), tid = threadIdx.x, wave = tid >> 6;
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  char* orow = (char*)out + r * ldo * Elem<DT>::bytes;
  const int nfull = V / N, p0 = part * (GRAD_NT * GRAD_UN), c0 = p0 + tid;
  u32x4 v[GRAD_UN];
#pragma unroll
  for (int j = 0; j < GRAD_UN; ++j)
    if (c0 + j * GRAD_NT < nfull) v[j] = load_piece<DT>(row, c0 + j * GRAD_NT);
  // the tail: one logit each of the first threads of the last block
  const int tail = nfull * N + tid;
  const bool has_tail = part == parts - 1 && tail < V;
  const float xt = has_tail ? load1<DT>(row, tail) : 0.f;
  const float* st = stats + r * ST_COLS;
  const float live = st[ST_LIVE], m = st[ST_M], s = st[ST_S], n = st[ST_ZN], zm = st[ST_ZM];
  const bool all = loss && part == 0;                    // every entry counts in the loss
  int id;
  float z;
  te.entry(r, tid, id, z);
  if (live != 1.f) {                                     // 0 without entries, NaN for a bad row
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = live;
#pragma unroll
    for (int j = 0; j < GRAD_UN; ++j)
      if (c0 + j * GRAD_NT < nfull) store_piece<DT>(orow, c0 + j * GRAD_NT, f);
    if (has_tail) store1<DT>(orow, tail, live);
    if (all && tid == 0) loss[r] = live;
    return;
  }
  // ---- the ids in this block's columns, in the order of the entries
  const long col = (long)id - vstart;
  const bool mine = id >= 0 && col >= (long)N * p0 && col < min((long)V, part == parts - 1 ? (long)V : (long)N * (p0 + GRAD_NT * GRAD_UN));
  const float x = mine ? load1<DT>(row, col) : 0.f;
  const float L = __log2f(s);
  float lq = 0.f, q, rest = 0.f, W = 1.f;
  if constexpr (REST) {
    q = mine || all ? (float)te.mass(r, id, z, lq) : 0.f;
    rest = st[ST_REST];
    W = n + rest;
  } else {
    z -= zm;
    q = id >= 0 ? __builtin_amdgcn_exp2f(z * a) / n : 0.f;
    lq = z * inv_temp - LN2 * __log2f(n);
    if (n != n) W = n;                                   // a NaN entry: the whole row
  }
  const u64 here = __ballot(mine);
  if ((tid & 63) == 0) cnt[wave] = __popcll(here);
  lds_barrier();
  int at = __popcll(here & ((1ull << (tid & 63)) - 1)), nin = 0;
#pragma unroll
  for (int w = 0; w < W4; ++w) {
    if (w < wave) at += cnt[w];
    nin += cnt[w];
  }
  head[tid] = 0;
  if (mine) {
    scol[at] = (int)col;
    sq[at] = q;
    sx[at] = x;
  }
  lds_barrier();
  // the thread that holds an element: that of its piece, or of its place in the tail
  auto owner = [&](int c) { return c < N * nfull ? (c / N - p0) % GRAD_NT : c - N * nfull; };
  if (tid < nin) next[tid] = atomicExch(&head[owner(scol[tid])], tid + 1);
  lds_barrier();
  if (tid < nin) {
    // the same id twice: as in the fused kernel
    const int c = scol[tid];
    bool twice = false;
    for (int h = head[owner(c)]; h; h = next[h - 1]) twice = twice || (h - 1 != tid && scol[h - 1] == c);
    float qs = sq[tid];
    if (twice) {
      qs = 0.f;
      for (int k = 0; k < nin; ++k) qs += scol[k] == c ? sq[k] : 0.f;
    }
    sqs[tid] = qs;
  }
  lds_barrier();
  const float sc = (rows ? rows[r] : 1.f) * (scale_ptr ? scale_ptr[0] : scale_h) * inv_temp;
  const float k1 = sc * (REST ? outside_factor(m, s, st[ST_MO], st[ST_U], W, rest, a) : W), ref = REST ? stat_ref(st[ST_MO]) : m, shift = REST ? 0.f : -L;
#pragma unroll
  for (int j = 0; j < GRAD_UN; ++j) {
    if (c0 + j * GRAD_NT >= nfull) continue;
    float f[N];
    unpack_piece<DT>(v[j], f);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = k1 * __builtin_amdgcn_exp2f(fmaf(f[i] - ref, a, shift));
    store_piece<DT>(orow, c0 + j * GRAD_NT, f);
  }
  if (has_tail) store1<DT>(orow, tail, k1 * __builtin_amdgcn_exp2f(fmaf(xt - ref, a, shift)));
  // each by the thread that stored around it, behind that store
  asm volatile("" ::: "memory");
  for (int h = head[tid]; h; h = next[h - 1])
    store1<DT>(orow, scol[h - 1], sc * fmaf(W, __builtin_amdgcn_exp2f(fmaf(sx[h - 1] - m, a, -L)), -sqs[h - 1]));
  if (all) {
    float l = block_reduce<GRAD_NT>(q != 0.f ? q * (lq + LN2 * L) : 0.f, 0.f, red, OpAdd{}, tid) - inv_temp * st[ST_XQ];
    if (tid == 0) {
      if constexpr (REST) l += rest_loss(m, L, st[ST_MO], st[ST_U], rest, inv_temp);
      loss[r] = l;
    }
  }
}

int cu_count() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    return 256;
  return n;
}

bool fits_registers(int dt, int V) {
  const int n = dt == DT_FP32 ? 4 : 8;
  return V >= n && V / n <= 1024 * RES_MAX;
}

// outputs of more than the last-level cache's 256 MB leave nothing in it for their reader: they are
// stored past the caches where every row starts on a multiple of 64 bytes (4096 rows of 128256 bf16
// logits 443 us against 450, of 128288 458 and 464; of 128272, where waves share such pieces, 472 and
// 468, of 128258 482 and 473)
constexpr long CACHE_BYTES = 256L << 20, LINE = 64;

}  // namespace

extern "C" {

int kf_distill_k_max() { return K_MAX; }
int kf_distill_stats_cols() { return ST_COLS; }
long kf_distill_rest_v_max() { return 8L * BITS_MAX; }

// whether mode 0 needs statistics [T, ST_COLS] as scratch
int kf_distill_needs_stats(int dt, int V) { return fits_registers(dt, V) ? 0 : 1; }

// mode 0: loss rows and gradient; 1: this part's statistics [T, ST_COLS], and the loss rows of an
// undivided vocabulary; 2: gradient (and loss rows) from joined statistics
int kf_distill_topk(const void* logits, int dt, long ld, void* out, long ldo, long rows, int V, long vstart, long vtotal,
                    const void* ids, int ids32, long ldi, const void* z, int zt, long ldz, const float* lse, int K,
                    double temperature, const float* scale_ptr, float scale_h, const float* row_scale, float* loss, float* stats,
                    int mode, hipStream_t s) {
  if (V < 1 || K < 0 || K > K_MAX || dt < DT_BF16 || dt > DT_FP32 || zt < DT_BF16 || zt > DT_FP32) return 1;
  const Teacher te{ids, z, lse, 1.0 / temperature, ldi, ldz, vtotal, ids32, zt, K};
  const float temp = (float)temperature;
  const size_t lds = lse ? ((size_t)V + 31) / 32 * 4 : 0;
  if (lds > BITS_MAX) return 2;
  if (rows == 0) return 0;
  Launcher launch;
  if (mode == KD_FUSED && fits_registers(dt, V)) {
    const long bytes = (long)V * (dt == DT_FP32 ? 4 : 2);
    const int keep = rows * bytes <= CACHE_BYTES || (((size_t)out | (size_t)(ldo * (dt == DT_FP32 ? 4 : 2))) & (LINE - 1));
    by_type(dt, [&](auto DTc) {
      auto go = [&](auto NTc, auto Sc, auto Rc) {
        constexpr int DT = decltype(DTc)::value, NT = decltype(NTc)::value, RES = decltype(Sc)::value;
        const unsigned grid = (unsigned)std::min<long>(rows, (long)cu_count() * (256 * fused_waves(RES) / NT));
        launch(distill_fused_kernel<DT, NT, RES, decltype(Rc)::value>, grid, NT, 0, s, logits, ld, out, ldo, rows, V, te,
               temp, scale_ptr, scale_h, loss, keep);
      };
      auto by_rest = [&](auto NTc, auto Sc) {
        if (lse) go(NTc, Sc, std::true_type{});
        else go(NTc, Sc, std::false_type{});
      };
      // the smallest block that holds a row: more of them share a CU
      const int np = V / Elem<decltype(DTc)::value>::N;
      using Short = std::integral_constant<int, RES_SHORT>;
      using Long = std::integral_constant<int, RES_MAX>;
      if (np <= 256 * RES_SHORT) by_rest(std::integral_constant<int, 256>{}, Short{});
      else if (np <= 256 * RES_MAX) by_rest(std::integral_constant<int, 256>{}, Long{});
      else if (np <= 512 * RES_MAX) by_rest(std::integral_constant<int, 512>{}, Long{});
      else by_rest(std::integral_constant<int, 1024>{}, Long{});
    });
    return launch.rc;
  }
  if (mode != KD_GRAD) {
    if (!stats) return 3;
    for (long r0 = 0; r0 < rows; r0 += ROWS_PER_LAUNCH) {
      const unsigned n = (unsigned)std::min(ROWS_PER_LAUNCH, rows - r0);
      Teacher t = te;
      t.ids = (const char*)ids + r0 * ldi * (ids32 ? 4 : 8);
      t.z = (const char*)z + r0 * ldz * (zt == DT_FP32 ? 4 : 2);
      if (lse) t.lse = lse + r0;
      by_type(dt, [&](auto DTc) {
        constexpr int DT = decltype(DTc)::value;
        auto go = [&](auto NTc, auto Rc) {
          constexpr int NT = decltype(NTc)::value;
          launch(distill_stats_kernel<DT, NT, decltype(Rc)::value>, n, NT, lds, s,
                 (const char*)logits + r0 * ld * Elem<DT>::bytes, ld, V, vstart, t, temp, loss + r0, stats + r0 * ST_COLS);
        };
        auto by_rest = [&](auto NTc) {
          if (lse) go(NTc, std::true_type{});
          else go(NTc, std::false_type{});
        };
        // eight to sixteen pieces a thread, as for the log-probabilities: 2000 rows of 32000 bf16 logits
        // take 27 us with 512 threads and 36 with 1024, 4096 of 128256 179 and 170
        const int np = V / Elem<DT>::N;
        if (np > 8192) by_rest(std::integral_constant<int, 1024>{});
        else if (np > 2048) by_rest(std::integral_constant<int, 512>{});
        else by_rest(std::integral_constant<int, 256>{});
      });
    }
  }
  if (mode != KD_STATS) {
    by_type(dt, [&](auto DTc) {
      constexpr int DT = decltype(DTc)::value;
      const int parts = std::max(1, cdiv(V / Elem<DT>::N, GRAD_NT * GRAD_UN));
      const long step = std::max<long>(1, (1L << 23) / parts);    // rows of a launch: less than 2^32 threads
      for (long r0 = 0; r0 < rows; r0 += step) {
        const long n = std::min(step, rows - r0);
        Teacher t = te;
        t.ids = (const char*)ids + r0 * ldi * (ids32 ? 4 : 8);
        t.z = (const char*)z + r0 * ldz * (zt == DT_FP32 ? 4 : 2);
        if (lse) t.lse = lse + r0;
        auto go = [&](auto Rc) {
          launch(distill_grad_kernel<DT, decltype(Rc)::value>, (unsigned)(n * parts), GRAD_NT, 0, s,
              (const char*)logits + r0 * ld * Elem<DT>::bytes, ld, (char*)out + r0 * ldo * Elem<DT>::bytes, ldo, V, parts,
              vstart, t, temp, scale_ptr, scale_h, row_scale ? row_scale + r0 : nullptr,
              // the statistics' launch wrote the loss of an undivided row already
              loss && mode == KD_GRAD ? loss + r0 : nullptr, stats + r0 * ST_COLS);
        };
        if (lse) go(std::true_type{});
        else go(std::false_type{});
      }
    });
  }
  return launch.rc;
}

}  // extern "C"
