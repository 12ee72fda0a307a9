// Log-probabilities of given tokens over rows of logits, with each row's entropy and its top
// alternatives, and the gradient of the first two.
//
//   ln p_t = (x_t - m) / temperature - ln2 log2 s        H = ln2 log2 s - (u / s) / temperature
//   dx_j   = [ g (1[j = t] - p_j) - h p_j (ln p_j + H) ] / temperature
//
// with the row statistics (m, s, u) of logits.h.  Forward: one pass over a row by one block, or by
// several where the rows are few.
#include "logits.h"

using namespace kf;

namespace {

typedef unsigned long long u64;

// ---- order of the alternatives: greater value first, NaN greatest, equal values by lower index.
// One 64-bit key per element, value above index, makes all elements different.
__device__ __forceinline__ u32 value_key(float f) {
  if (f != f) return 0xffffffffu;
  const u32 b = __float_as_uint(f + 0.f);      // -0 and +0 are one value
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(u32 k) {
  if (k == 0xffffffffu) return quiet_nan();
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ u64 elem_key(float f, u32 idx) { return ((u64)value_key(f) << 32) | (u32)~idx; }

constexpr int TOP_MAX = 128;
constexpr int CAND = 1024;     // candidate elements held at a time
constexpr int GROUPS = 256;    // thread groups whose maxima bound the k-th element from below

struct TopShared {
  u32 group[GROUPS];
  alignas(16) u64 cand[CAND + 4];
  int alone[1024];             // best pieces of threads where no second one reaches the bound
  unsigned short who[1024];    // threads with several that do
  int nalone, nwho, ncand;
  u64 bound;
};

// a value that at least k of 256 keys (4 a lane) reach, and where the keys differ few more than k;
// 0 where fewer than k are not 0.  Bit by bit below the first bit in which the keys differ.
__device__ __forceinline__ u32 wave_kth(const u32* key, int k) {
  u32 v[4], hi = 0, lo = ~0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = key[4 * __lane_id() + i];
    hi = max(hi, v[i]);
    lo = min(lo, v[i]);
  }
  hi = wave_max(hi);
  lo = ~wave_max(~lo);
  if (hi == lo) return lo;
  u32 bit = 0x80000000u >> __clz(hi ^ lo);
  u32 t = hi & ~(2 * bit - 1);                   // the bits that all keys share
#pragma unroll 1
  for (; bit; bit >>= 1) {
    const u32 w = t | bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += __popcll(__ballot(v[i] >= w));
    if (n >= k) {
      t = w;
      if (n <= k + 16) break;
    }
  }
  return t;
}

// out(rank, key) for the keys of rank < k among the n different keys at `key`, by all threads of a
// block of nt: `per` neighbouring threads (a power of two) count a share of the others each.  n^2
// comparisons: for some hundred keys.  The list is 16-byte aligned and filled up with zeros to a multiple of 4.
typedef __attribute__((ext_vector_type(2))) u64 u64x2;
template <typename Out>
__device__ __forceinline__ void block_rank(const u64* key, int n, int k, int tid, int nt, Out out) {
  int per = 1;
  while (per < 16 && 2 * per * n <= nt) per <<= 1;
  const int q = tid & (per - 1);
  for (int i0 = 0; i0 < n; i0 += nt / per) {
    const int i = i0 + tid / per;
    const u64 mine = i < n ? key[i] : ~0ull;
    int c = 0;
#pragma unroll 2
    for (int j = 4 * q; j < n; j += 4 * per) {
      const u64x2 x = *(const u64x2*)(key + j), y = *(const u64x2*)(key + j + 2);
      c += (x[0] > mine) + (x[1] > mine) + (y[0] > mine) + (y[1] > mine);
    }
    for (int s = 1; s < per; s <<= 1) c += __shfl_xor(c, s, 64);
    if (i < n && q == 0 && c < k) out(c, mine);
  }
}

// A thread's best piece and the greatest value of its other pieces.
struct Best {
  float v, second;
  int c;
};

// The k greatest elements of the pieces [p0, p1) of a row, in order: out(rank, key) is called once
// for each rank < min(k, number of elements).
//
// If k groups of threads have maxima of at least `bound`, the k greatest elements all have values of
// at least `bound`.  The k-th greatest of 256 group maxima is such a bound, and close: for values in
// no order about 1.1 k elements reach it (k = 64).  Only threads whose best piece reaches it can own
// one, and only those whose second piece does are read in full again.  Where more than CAND
// elements reach the bound (many equal values, or a row in an order that meets the threads'
// stride), the k-th greatest of CAND held ones is the next, strictly greater bound: at least
// CAND - k elements drop out each time.
template <int DT, int NT, typename Out>
__device__ __forceinline__ void block_top(const char* row, int V, int p0, int p1, int k, bool have, Best best, bool by_key,
                                          TopShared& sh, Out out) {
  constexpr int N = Elem<DT>::N, PER = NT / GROUPS;             // PER: threads of a group
  const int tid = threadIdx.x;
  u32 mine = have ? value_key(best.v) : 0u, second = have ? value_key(best.second) : 0u;
  if (by_key && have) {
    // NaN or +inf in the row (every log-probability is NaN): the walk's maxima pass over NaN, so the
    // pieces are gone over again by key
    mine = 0;
    for (int c = p0 + tid; c < p1; c += NT) {
      float f[N];
      load_any<DT>(row, c, V, -INFINITY, f);
#pragma unroll
      for (int j = 0; j < N; ++j) mine = max(mine, value_key(f[j]));
    }
    second = mine;
  }
  u32 g = mine;
#pragma unroll
  for (int o = 1; o < PER; o <<= 1) g = max(g, (u32)__shfl_xor((int)g, o, 64));
  if (tid % PER == 0) sh.group[tid / PER] = g;
  if (tid == 0) sh.nalone = sh.nwho = 0;
  __syncthreads();
  if (tid < 64) {
    const u32 b = wave_kth(sh.group, k);
    if (tid == 0) sh.bound = (u64)b << 32;
  }
  __syncthreads();
  u64 bound = sh.bound;                          // 0: fewer than k groups, every element is taken
  const u32 floor = (u32)(bound >> 32);
  if (have && second >= floor) sh.who[atomicAdd(&sh.nwho, 1)] = (unsigned short)tid;
  else if (have && mine >= floor) sh.alone[atomicAdd(&sh.nalone, 1)] = best.c;
  for (;;) {
    if (tid == 0) sh.ncand = 0;
    __syncthreads();
    const int nwho = sh.nwho, nall = nwho * ((p1 - p0 + NT - 1) / NT), nwork = nall + sh.nalone;
    for (int w = tid; w < nwork; w += NT) {
      const int c = w < nall ? p0 + (w / nwho) * NT + sh.who[w % nwho] : sh.alone[w - nall];
      // too many already: another round
      if (c >= p1 || *(volatile int*)&sh.ncand > CAND) continue;
      float f[N];
      load_any<DT>(row, c, V, 0.f, f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const u32 idx = (u32)N * c + j;
        const u64 key = elem_key(f[j], idx);
        if (idx < (u32)V && key >= bound) {
          const int at = atomicAdd(&sh.ncand, 1);
          if (at < CAND) sh.cand[at] = key;
        }
      }
    }
    __syncthreads();
    const int n = sh.ncand, held = n < CAND ? n : CAND;
    if (tid < 4) sh.cand[held + tid] = 0;
    __syncthreads();
    if (n <= CAND) {
      block_rank(sh.cand, n, k, tid, NT, out);
      break;
    }
    block_rank(sh.cand, held, k, tid, NT, [&](int rank, u64 key) {
      if (rank == k - 1) sh.bound = key;
    });
    __syncthreads();
    bound = sh.bound;
  }
}

// one pass over the pieces [p0, p1) of a row: the thread's statistics and, with TOP, its best piece
constexpr int UN = 4;          // pieces in flight per thread

template <int DT, int NT, bool TOP>
__device__ __forceinline__ RowStat walk_row(const char* row, int V, int p0, int p1, float a, Best& best) {
  constexpr int N = Elem<DT>::N;
  const int nfull = min(V / N, p1);
  RowStat st = stat_empty();
  best = {-INFINITY, -INFINITY, p0 + (int)threadIdx.x};     // all -inf: the first piece
  float f[UN][N];
  auto eat = [&](int c0, int n) {
    float bm = st.m;
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (j >= n) continue;
      const float vm = max_piece<DT>(f[j]);
      if constexpr (TOP) {
        best.second = fmaxf(best.second, fminf(vm, best.v));
        if (vm > best.v) { best.v = vm; best.c = c0 + j * NT; }
      }
      bm = fmaxf(bm, vm);
    }
    if (bm != st.m) stat_move<MOMENT>(st, bm, a);
    const float ref = stat_ref(st.m);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (j >= n) continue;
#pragma unroll
      for (int i = 0; i < N; ++i) stat_add<MOMENT>(st, ref, f[j][i], a);
    }
  };
  int c = p0 + threadIdx.x;
  for (; c + (UN - 1) * NT < nfull; c += UN * NT) {
    u32x4 r[UN];
    load_pieces<DT>(row, [&](int j) { return c + j * NT; }, r);
#pragma unroll
    for (int j = 0; j < UN; ++j) unpack_piece<DT>(r[j], f[j]);
    eat(c, UN);
  }
  if (c < nfull) {
    // the rest, loaded together: pieces behind the end are the last full one again, read as -inf
    u32x4 r[UN];
    load_pieces<DT>(row, [&](int j) { return min(c + j * NT, nfull - 1); }, r);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      unpack_piece<DT>(r[j], f[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) f[j][i] = c + j * NT < nfull ? f[j][i] : -INFINITY;
    }
    eat(c, UN);
  }
  if (p1 > nfull && (int)threadIdx.x == (nfull - p0) % NT) {
    load_any<DT>(row, nfull, V, -INFINITY, f[0]);
    eat(nfull, 1);
  }
  return st;
}

// written out, so that a token's log-probability is the same bits as the given one and as an alternative
__device__ __forceinline__ float ln_p(float x, float m, float L, float inv_temp) {
  return fmaf(x - m, inv_temp, -__fmul_rn(LN2, L));
}

struct Result {
  float *logp, *entropy, *stats, *top;
  long* ids;
};
__device__ __forceinline__ void write_ignored(const Result& o, long r, int k, int tid, int nt) {
  if (tid == 0) { o.logp[r] = 0.f; o.entropy[r] = 0.f; o.stats[2 * r] = 0.f; o.stats[2 * r + 1] = 0.f; }
  for (int i = tid; i < k; i += nt) { o.ids[r * k + i] = -1; o.top[r * k + i] = 0.f; }
}
__device__ __forceinline__ void write_row(const Result& o, long r, RowStat st, float L, bool in, float x, float inv_temp) {
  o.logp[r] = in ? ln_p(x, st.m, L, inv_temp) : quiet_nan();
  o.entropy[r] = LN2 * L - st.u / st.s * inv_temp;
  o.stats[2 * r] = st.m;
  o.stats[2 * r + 1] = L;
}
__device__ __forceinline__ void write_top(const Result& o, long r, int k, int rank, u64 key, float m, float L, float inv_temp) {
  o.ids[r * k + rank] = (long)(u32)~(u32)key;
  o.top[r * k + rank] = ln_p(key_value((u32)(key >> 32)), m, L, inv_temp);
}

// one block per row; 8 waves a SIMD (registers of both kinds: 100 scalar ones already halve that), so
// that blocks share a CU and some read while others rank: 2048 rows with 64 alternatives 103 us, 143
// with a block of 1024 alone on its CU
template <int DT, int NT, bool TOP>
__global__ __launch_bounds__(NT, 8) void logprobs_kernel(const void* __restrict__ logits, long ld, int V,
                                                      const long* __restrict__ tokens, long ignore, float a,
                                                      float inv_temp, int k, Result o) {
  __shared__ RowStat red[NT / 64];
  const long r = blockIdx.x;
  const int tid = threadIdx.x;
  const long t = tokens[r];
  if (t == ignore) return write_ignored(o, r, TOP ? k : 0, tid, NT);     // a padding row: not read
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  const int np = (V + Elem<DT>::N - 1) / Elem<DT>::N;
  Best best;
  const RowStat st = block_stat<MOMENT, NT>(walk_row<DT, NT, TOP>(row, V, 0, np, a, best), a, red, tid);
  const float L = __log2f(st.s);
  if (tid == 0) {
    const bool in = t >= 0 && t < V;
    write_row(o, r, st, L, in, in ? load1<DT>(row, t) : 0.f, inv_temp);
  }
  if constexpr (TOP) {
    __shared__ TopShared sh;
    block_top<DT, NT>(row, V, 0, np, k, tid < np, best, !(st.s < INFINITY), sh,
                      [&](int rank, u64 key) { write_top(o, r, k, rank, key, st.m, L, inv_temp); });
  }
}

// Few long rows: one CU alone takes 8 us to read 128256 bf16 logits and form their exponentials, so a
// row goes to `parts` blocks of PART_NT threads and a second launch joins their statistics and
// alternatives.
constexpr int PART_NT = 256;
struct Part {
  RowStat st;
  float pad;
};

template <int DT, bool TOP>
__global__ __launch_bounds__(PART_NT, 8) void logprobs_part_kernel(const void* __restrict__ logits, long ld, int V,
                                                                float a, int k, int parts, int per,
                                                                Part* __restrict__ part,
                                                                u64* __restrict__ keys) {
  __shared__ RowStat red[PART_NT / 64];
  const long r = blockIdx.x / parts;
  const int q = (int)(blockIdx.x - r * parts), tid = threadIdx.x;
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  const int np = (V + Elem<DT>::N - 1) / Elem<DT>::N, p0 = q * per, p1 = min(np, p0 + per);
  Best best;
  const RowStat st = block_stat<MOMENT, PART_NT>(walk_row<DT, PART_NT, TOP>(row, V, p0, p1, a, best), a, red, tid);
  if (tid == 0) part[blockIdx.x].st = st;
  if constexpr (TOP) {
    __shared__ TopShared sh;
    u64* mine = keys + (long)blockIdx.x * k;
    const int n = min(V, Elem<DT>::N * p1) - Elem<DT>::N * p0;
    for (int i = n + tid; i < k; i += PART_NT) mine[i] = 0;            // a part of fewer than k logits
    block_top<DT, PART_NT>(row, V, p0, p1, k, p0 + tid < p1, best, !(st.s < INFINITY), sh,
                           [&](int rank, u64 key) { mine[rank] = key; });
  }
}

// The parts' alternatives are `parts` lists of k keys in order.  The first ones of each list, 256
// together, give a bound as the groups' maxima above, and some k + 16 keys reach it: those are
// ranked.  Up to 192 keys are ranked as they are, which takes less than finding the bound (160 keys:
// 13.3 us a call against 13.6; 320: 12.2 against 9.6, 1024: 32 against 10.5).
constexpr int JOIN_NT = 512, PARTS_MAX = 16, JOIN_KEYS = PARTS_MAX * TOP_MAX, JOIN_DIRECT = 192;

template <int DT>
__global__ __launch_bounds__(JOIN_NT) void logprobs_join_kernel(const void* __restrict__ logits, long ld, int V,
                                                                const long* __restrict__ tokens, long ignore, float a,
                                                                float inv_temp, int k, int parts,
                                                                const Part* __restrict__ part,
                                                                const u64* __restrict__ keys, Result o) {
  constexpr int HELD = JOIN_KEYS / JOIN_NT;
  __shared__ alignas(16) u64 cand[JOIN_KEYS + 4];
  __shared__ u32 first[GROUPS], bound;
  __shared__ int ncand;
  const long r = blockIdx.x;
  const int tid = threadIdx.x, n = parts * k;
  const long t = tokens[r];
  const bool in = t >= 0 && t < V, direct = n <= JOIN_DIRECT;
  const float x = in ? load1<DT>((const char*)logits + r * ld * Elem<DT>::bytes, t) : 0.f;
  const int l = tid & 15;
  const RowStat mine = l < parts ? part[r * parts + l].st : stat_empty();
  u64 key[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) key[i] = tid + i * JOIN_NT < n ? keys[r * n + tid + i * JOIN_NT] : 0;
  if (!direct && tid < GROUPS) {
    // parts >= 2; `each` a power of two: with fewer than k keys in `first` the bound would be 0
    const int each = GROUPS >> (32 - __clz(parts - 1)), q = tid / each, at = tid & (each - 1);
    first[tid] = q < parts && at < k ? (u32)(keys[r * n + q * k + at] >> 32) : 0u;
  }
  if (t == ignore) return write_ignored(o, r, k, tid, blockDim.x);
  const RowStat st = lanes_stat<MOMENT, 16>(mine, a);
  const float L = __log2f(st.s);
  if (tid == 0) write_row(o, r, st, L, in, x, inv_temp);
  if (k == 0) return;
  for (int i = tid; i < n + 4; i += JOIN_NT) cand[i] = 0;
  if (tid == 0) {
    ncand = 0;
    bound = 1;                                   // key 0: a part of fewer than k logits
  }
  __syncthreads();
  if (!direct) {
    if (tid < 64) {
      const u32 b = wave_kth(first, k);
      if (tid == 0) bound = max(b, 1u);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if ((u32)(key[i] >> 32) >= bound) cand[atomicAdd(&ncand, 1)] = key[i];
  __syncthreads();
  block_rank(cand, ncand, k, tid, JOIN_NT, [&](int rank, u64 v) { write_top(o, r, k, rank, v, st.m, L, inv_temp); });
}

// gradient: one block per 4 pieces a thread of a row, nothing to reduce
constexpr int BWD_NT = 256, BWD_UN = 4;

template <int DT>
__global__ __launch_bounds__(BWD_NT) void logprobs_bwd_kernel(const void* logits, long ld, void* out, long ldo, int V,
                                                              int parts, const long* __restrict__ tokens, long ignore,
                                                              const float* __restrict__ stats,
                                                              const float* __restrict__ entropy,
                                                              const float* __restrict__ dlogp,
                                                              const float* __restrict__ dent, float a,
                                                              float inv_temp) {
  constexpr int N = Elem<DT>::N;
  const long r = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - r * parts);
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  char* orow = (char*)out + r * ldo * Elem<DT>::bytes;
  const long t = tokens[r];
  const int np = (V + N - 1) / N;
  const int c0 = part * (BWD_NT * BWD_UN) + threadIdx.x;
  if (t == ignore) {
    const float z[N] = {};
#pragma unroll
    for (int j = 0; j < BWD_UN; ++j)
      if (c0 + j * BWD_NT < np) store_any<DT>(orow, c0 + j * BWD_NT, V, z);
    return;
  }
  const float m = stats[2 * r], L = stats[2 * r + 1];
  const float g = dlogp ? dlogp[r] : 0.f, h = dent ? dent[r] : 0.f;
  const bool in = t >= 0 && t < V;
  // dx_j = p_j (A + B log2 p_j) + 1[j = t] g / temperature; a token outside the row: NaN
  const float A = in ? -(g + h * entropy[r]) * inv_temp : quiet_nan();
  const float B = -h * LN2 * inv_temp;
  float f[BWD_UN][N];
#pragma unroll
  for (int j = 0; j < BWD_UN; ++j)
    if (c0 + j * BWD_NT < np) load_any<DT>(row, c0 + j * BWD_NT, V, 0.f, f[j]);
#pragma unroll
  for (int j = 0; j < BWD_UN; ++j) {
    const int c = c0 + j * BWD_NT;
    if (c >= np) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float l = fmaf(f[j][i] - m, a, -L);
      const float p = __builtin_amdgcn_exp2f(l);
      f[j][i] = p * fmaf(B, fmaxf(l, FAR), A);
    }
    if (t / N == c) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((int)(t % N) == i) f[j][i] += g * inv_temp;
    }
    store_any<DT>(orow, c, V, f[j]);
  }
}

// Blocks of one row for `rows` rows of np pieces.  A row is split where one block would take longer
// than two launches: from 8192 pieces on with alternatives, whose ranking the parts do twice, and
// from 4096 without (24 rows of 50021 bf16 logits: 5.9 us split and 7.0 whole without alternatives,
// 12.0 and 11.1 with 20; of 32000 5.4 whole, 4.9 split and 8.9, 10.3; of 128256 5.6, 10.9 and 11.1,
// 15.5), and below 128 rows, where the two take the same (128256 logits: 11.9 and 12.1 us).  Then up to
// two blocks a CU, with at least two pieces a thread.
static int split_parts(long rows, int np, int k) {
  if (rows >= 128 || np <= (k > 0 ? 8192 : 4096)) return 1;
  return (int)std::min<long>(std::min<long>(512 / std::max<long>(rows, 1), cdiv(np, 2 * PART_NT)), PARTS_MAX);
}

}  // namespace

extern "C" {

int kf_token_logprobs_top_max() { return TOP_MAX; }

// bytes of scratch for kf_token_logprobs (0: none)
long kf_token_logprobs_scratch(int dt, long rows, int V, int k) {
  const int n = dt == DT_FP32 ? 4 : 8, parts = split_parts(rows, (V + n - 1) / n, k);
  return parts > 1 ? rows * parts * ((long)sizeof(Part) + 8L * k) : 0;
}

int kf_token_logprobs(const void* logits, int dt, long ld, long rows, int V, const long* tokens, long ignore, float temp,
                      float* logp, float* entropy, float* stats, int k, long* ids, float* top, void* scratch,
                      hipStream_t s) {
  if (V < 1 || k < 0 || k > V || k > TOP_MAX || dt < DT_BF16 || dt > DT_FP32) return 1;
  if (rows == 0) return 0;
  const float a = LOG2E / temp, inv = 1.f / temp;
  Launcher launch;
  by_type(dt, [&](auto DTc) {
    constexpr int DT = decltype(DTc)::value;
    const int np = (V + Elem<DT>::N - 1) / Elem<DT>::N, parts = split_parts(rows, np, k);
    if (parts > 1) {
      const int per = cdiv(cdiv(np, parts), 64) * 64;           // the lanes of a wave end together
      const Result o{logp, entropy, stats, top, ids};
      Part* part = (Part*)scratch;
      u64* keys = (u64*)(part + rows * parts);
      // the parts are of equal size, so the last ones may be empty: as many as hold a piece
      const int used = cdiv(np, per);
      if (k > 0)
        launch(logprobs_part_kernel<DT, true>, (unsigned)(rows * used), PART_NT, 0, s, logits, ld, V, a, k, used, per,
               part, keys);
      else
        launch(logprobs_part_kernel<DT, false>, (unsigned)(rows * used), PART_NT, 0, s, logits, ld, V, a, 0, used, per,
               part, keys);
      launch(logprobs_join_kernel<DT>, (unsigned)rows, k > 0 ? JOIN_NT : 64, 0, s, logits, ld, V, tokens, ignore, a, inv, k,
             used, part, keys, o);
      return;
    }
    for (long r0 = 0; r0 < rows; r0 += ROWS_PER_LAUNCH) {
      const unsigned n = (unsigned)std::min(ROWS_PER_LAUNCH, rows - r0);
      const void* x = (const char*)logits + r0 * ld * Elem<DT>::bytes;
      const Result o{logp + r0, entropy + r0, stats + 2 * r0, k > 0 ? top + r0 * k : nullptr, k > 0 ? ids + r0 * k : nullptr};
      auto go = [&](auto NTc, auto TOPc) {
        constexpr int NT = decltype(NTc)::value;
        launch(logprobs_kernel<DT, NT, decltype(TOPc)::value>, n, NT, 0, s, x, ld, V, tokens + r0, ignore, a, inv, k,
               o);
      };
      // eight to sixteen pieces a thread: 4000 rows of 128256 bf16 logits take 157 us with 1024
      // threads and 172 with 512, of 32000 logits 52 and 47.  With alternatives smaller blocks: more
      // of them share a CU, and some read while others rank (2500 rows of 128256: 131 us with 1024,
      // 124 with 512; 4000 rows of 32000: 95 with 1024, 66 with 512, 62 with 256).  Up to 512 rows
      // are held at once also as blocks of 1024 threads (256 rows of 50021, 20 alternatives: 12.8 us
      // with 1024, 15.2 with 256; 512 rows of 128256: 32.1 and 32.3 with 512; 700: 43.8 and 41.8)
      if (k > 0) {
        if (np > 4096 && rows <= 512) go(std::integral_constant<int, 1024>{}, std::true_type{});
        else if (np > 8192 || (np > 2048 && rows <= 512)) go(std::integral_constant<int, 512>{}, std::true_type{});
        else go(std::integral_constant<int, 256>{}, std::true_type{});
      } else {
        if (np > 8192) go(std::integral_constant<int, 1024>{}, std::false_type{});
        else if (np > 2048) go(std::integral_constant<int, 512>{}, std::false_type{});
        else go(std::integral_constant<int, 256>{}, std::false_type{});
      }
    }
  });
  return launch.rc;
}

int kf_token_logprobs_bwd(const void* logits, int dt, long ld, void* out, long ldo, long rows, int V, const long* tokens,
                          long ignore, const float* stats, const float* entropy, const float* dlogp, const float* dent,
                          float temp, hipStream_t s) {
  if (V < 1 || dt < DT_BF16 || dt > DT_FP32) return 1;
  const float a = LOG2E / temp, inv = 1.f / temp;
  Launcher launch;
  by_type(dt, [&](auto DTc) {
    constexpr int DT = decltype(DTc)::value;
    const int parts = cdiv((V + Elem<DT>::N - 1) / Elem<DT>::N, BWD_NT * BWD_UN);
    const long per = std::max<long>(1, (1L << 23) / parts);     // rows of a launch: less than 2^32 threads
    for (long r0 = 0; r0 < rows; r0 += per) {
      const long n = std::min(per, rows - r0);
      launch(logprobs_bwd_kernel<DT>, (unsigned)(n * parts), BWD_NT, 0, s,
          (const char*)logits + r0 * ld * Elem<DT>::bytes, ld, (char*)out + r0 * ldo * Elem<DT>::bytes, ldo, V, parts,
          tokens + r0, ignore, stats + 2 * r0, entropy + r0, dlogp ? dlogp + r0 : nullptr, dent ? dent + r0 : nullptr, a,
          inv);
    }
  });
  return launch.rc;
}

}  // extern "C"
