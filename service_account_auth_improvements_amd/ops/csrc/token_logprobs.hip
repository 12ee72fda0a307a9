// Log-probabilities of given tokens over rows of logits, with each row's entropy and its top
// alternatives, and the gradient of the first two.
//
//   ln p_t = (x_t - m) / temperature - ln2 log2 s        H = ln2 log2 s - (u / s) / temperature
//   dx_j   = [ g (1[j = t] - p_j) - h p_j (ln p_j + H) ] / temperature
//
// with the row statistics (m, s, u) of logits.h.  Forward: one block per row, one pass over it.
#include "logits.h"

#include <type_traits>

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
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ u64 elem_key(float f, u32 idx) { return ((u64)value_key(f) << 32) | (u32)~idx; }

constexpr int TOP_MAX = 128;
constexpr int CAND = 1024;     // candidate elements held at a time
constexpr int GROUPS = 256;    // thread groups whose best chunks bound the k-th element from below

struct TopShared {
  u64 group[GROUPS];
  u64 cand[CAND];
  unsigned short who[1024];    // threads whose best chunk reaches the bound
  int nwho, ncand;
  u64 bound;
};

__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int o) {
  const u32 lo = __shfl_xor((u32)v, o, 64), hi = __shfl_xor((u32)(v >> 32), o, 64);
  return ((u64)hi << 32) | lo;
}

// The k greatest elements of the row, in order: out(rank, key) is called once for each rank < k
// (k <= V).  `best` is the thread's greatest chunk key (chunk c: its greatest value over the index
// 8c + 7, so that an element of a chunk reaches a chunk's key only if it comes no later), 0 for a
// thread without chunks.
//
// If k chunks have keys of at least `bound`, the k greatest elements all have keys of at least
// `bound`: each of those chunks holds one element that does.  The k-th greatest of 256 group
// maxima is such a bound, and close: for values in no order about 1.1 k elements reach it (k =
// 64).  Only threads whose own best chunk reaches it can own one, so little of the row is read
// again.  Where more than CAND elements reach the bound (a row in an order that meets the
// threads' stride), the k-th greatest of the CAND held ones is the next, strictly greater bound:
// at least CAND - k elements drop out each time.
template <int DT, int NT, typename Out>
__device__ __forceinline__ void block_top(const void* row, int V, int k, u64 best, TopShared& sh, Out out) {
  const int tid = threadIdx.x;
  const int nchunk = (V + 7) >> 3;
  constexpr int PER = NT / GROUPS;               // threads of a group
  u64 g = best;
#pragma unroll
  for (int o = 1; o < PER; o <<= 1) {
    const u64 x = shfl_xor_u64(g, o);
    g = x > g ? x : g;
  }
  if (tid % PER == 0) sh.group[tid / PER] = g;
  if (tid == 0) { sh.bound = 0; sh.nwho = 0; }
  __syncthreads();
  {
    // rank of each group: PER threads count a share of the others each
    int n = 0;
    const int q = tid % PER;
#pragma unroll 8
    for (int i = 0; i < GROUPS / PER; ++i) n += sh.group[i * PER + q] > g;
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) n += __shfl_xor(n, o, 64);
    if (q == 0 && n == k - 1 && g != 0) sh.bound = g;   // one group at most: keys differ
  }
  __syncthreads();
  u64 bound = sh.bound;                          // 0: fewer than k chunks, every element is taken
  if (best != 0 && best >= bound) sh.who[atomicAdd(&sh.nwho, 1)] = (unsigned short)tid;
  for (;;) {
    if (tid == 0) sh.ncand = 0;
    __syncthreads();
    const int nwho = sh.nwho, niter = (nchunk + NT - 1) / NT;
    for (int w = tid; w < nwho * niter; w += NT) {
      const int c = (w / nwho) * NT + sh.who[w % nwho];
      if (c >= nchunk) continue;
      float f[8];
      load_chunk<DT>(row, c, V, 0.f, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u32 idx = 8u * c + j;
        const u64 key = elem_key(f[j], idx);
        if (idx < (u32)V && key >= bound) {
          const int at = atomicAdd(&sh.ncand, 1);
          if (at < CAND) sh.cand[at] = key;
        }
      }
    }
    __syncthreads();
    const int n = sh.ncand, held = n < CAND ? n : CAND;
    for (int i = tid; i < held; i += NT) {
      const u64 key = sh.cand[i];
      int r = 0;
      for (int j = 0; j < held; ++j) r += sh.cand[j] > key;
      if (n <= CAND) {
        if (r < k) out(r, key);
      } else if (r == k - 1) {
        sh.bound = key;
      }
    }
    if (n <= CAND) break;
    __syncthreads();
    bound = sh.bound;
  }
}

// one pass over a row part [c0, c1) of chunks, c0 multiple of NT: the thread's statistics and, with
// TOP, its greatest chunk (first of equals)
constexpr int UN = 4;          // chunks in flight per thread

template <int DT, int NT, bool TOP>
__device__ __forceinline__ void walk_row(const void* row, int V, float a, RowStat& st, float& bestv, int& bestc) {
  const int nfull = V >> 3;
  st = stat_empty();
  bestv = -INFINITY;
  bestc = (int)threadIdx.x;    // a thread whose logits are all -inf: its first chunk
  float f[UN][8];
  auto eat = [&](int c0, int n) {
    float bm = -INFINITY;
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (j >= n) continue;
      const float vm = max8(f[j]);
      if (TOP && vm > bestv) { bestv = vm; bestc = c0 + j * NT; }
      bm = fmaxf(bm, vm);
    }
    stat_move(st, fmaxf(st.m, bm), a);
    const float ref = stat_ref(st.m);
#pragma unroll
    for (int j = 0; j < UN; ++j) {
      if (j >= n) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) stat_add(st, ref, f[j][i], a);
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
    // the rest, loaded together: chunks behind the end are the last full one again, read as -inf
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
}

template <int DT, int NT, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_kernel(const void* __restrict__ logits, long ld, int V,
                                                      const long* __restrict__ tokens, long ignore, float a,
                                                      float inv_temp, float* __restrict__ logp,
                                                      float* __restrict__ entropy, float* __restrict__ stats, int k,
                                                      long* __restrict__ ids, float* __restrict__ top) {
  __shared__ RowStat red[NT / 64];
  const long r = blockIdx.x;
  const int tid = threadIdx.x;
  const long t = tokens[r];
  if (t == ignore) {            // a padding row: not read
    if (tid == 0) { logp[r] = 0.f; entropy[r] = 0.f; stats[2 * r] = 0.f; stats[2 * r + 1] = 0.f; }
    if (TOP)
      for (int i = tid; i < k; i += NT) { ids[r * k + i] = -1; top[r * k + i] = 0.f; }
    return;
  }
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  RowStat st;
  float bestv;
  int bestc;
  walk_row<DT, NT, TOP>(row, V, a, st, bestv, bestc);
  st = block_stat<NT>(st, a, red);
  const float L = __log2f(st.s);
  if (tid == 0) {
    const bool in = t >= 0 && t < V;
    logp[r] = in ? (load1<DT>(row, t) - st.m) * inv_temp - LN2 * L : __uint_as_float(0x7fc00000u);
    entropy[r] = LN2 * L - st.u / st.s * inv_temp;
    stats[2 * r] = st.m;
    stats[2 * r + 1] = L;
  }
  if constexpr (TOP) {
    __shared__ TopShared sh;
    const int nchunk = (V + 7) >> 3;
    u64 best = tid < nchunk ? elem_key(bestv, 8u * bestc + 7u) : 0;
    if (!(st.s < INFINITY)) {
      // NaN or +inf in the row (every log-probability is NaN): the walk's maxima ignore NaN, so
      // the chunks are gone over again by key
      best = 0;
      for (int c = tid; c < nchunk; c += NT) {
        float f[8];
        load_chunk<DT>(row, c, V, -INFINITY, f);
        u32 vk = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) vk = max(vk, value_key(f[j]));
        const u64 key = ((u64)vk << 32) | (u32)~(8u * c + 7u);
        best = key > best ? key : best;
      }
    }
    const float m = st.m;
    block_top<DT, NT>(row, V, k, best, sh, [&](int rank, u64 key) {
      ids[r * k + rank] = (long)(u32)~(u32)key;
      top[r * k + rank] = (key_value((u32)(key >> 32)) - m) * inv_temp - LN2 * L;
    });
  }
}

// gradient: one block per 8192 logits of a row, nothing to reduce
constexpr int BWD_NT = 256, BWD_UN = 4;

template <int DT>
__global__ __launch_bounds__(BWD_NT) void logprobs_bwd_kernel(const void* logits, long ld, void* out, long ldo, int V,
                                                              int parts, const long* __restrict__ tokens, long ignore,
                                                              const float* __restrict__ stats,
                                                              const float* __restrict__ entropy,
                                                              const float* __restrict__ dlogp,
                                                              const float* __restrict__ dent, float a,
                                                              float inv_temp) {
  const long r = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - r * parts);
  const char* row = (const char*)logits + r * ld * Elem<DT>::bytes;
  char* orow = (char*)out + r * ldo * Elem<DT>::bytes;
  const long t = tokens[r];
  const int nchunk = (V + 7) >> 3;
  const int c0 = part * (BWD_NT * BWD_UN) + threadIdx.x;
  if (t == ignore) {
    const float z[8] = {};
#pragma unroll
    for (int j = 0; j < BWD_UN; ++j)
      if (c0 + j * BWD_NT < nchunk) store_chunk<DT>(orow, c0 + j * BWD_NT, V, z);
    return;
  }
  const float m = stats[2 * r], L = stats[2 * r + 1];
  const float g = dlogp ? dlogp[r] : 0.f, h = dent ? dent[r] : 0.f;
  const bool in = t >= 0 && t < V;
  // dx_j = p_j (A + B log2 p_j) + 1[j = t] g / temperature; a token outside the row: NaN
  const float A = in ? -(g + h * entropy[r]) * inv_temp : __uint_as_float(0x7fc00000u);
  const float B = -h * LN2 * inv_temp;
  float f[BWD_UN][8];
#pragma unroll
  for (int j = 0; j < BWD_UN; ++j)
    if (c0 + j * BWD_NT < nchunk) load_chunk<DT>(row, c0 + j * BWD_NT, V, 0.f, f[j]);
#pragma unroll
  for (int j = 0; j < BWD_UN; ++j) {
    const int c = c0 + j * BWD_NT;
    if (c >= nchunk) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float l = fmaf(f[j][i] - m, a, -L);
      const float p = __builtin_amdgcn_exp2f(l);
      f[j][i] = p * fmaf(B, fmaxf(l, FAR), A);
    }
    if ((t >> 3) == c) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((int)(t & 7) == i) f[j][i] += g * inv_temp;
    }
    store_chunk<DT>(orow, c, V, f[j]);
  }
}

constexpr long ROWS_PER_LAUNCH = 1 << 20;   // a launch holds less than 2^32 threads

template <int DT, int NT>
void launch_fwd(const void* logits, long ld, long rows, int V, const long* tokens, long ignore, float a, float inv_temp,
                float* logp, float* entropy, float* stats, int k, long* ids, float* top, hipStream_t s) {
  for (long r0 = 0; r0 < rows; r0 += ROWS_PER_LAUNCH) {
    const int n = (int)std::min(ROWS_PER_LAUNCH, rows - r0);
    const void* x = (const char*)logits + r0 * ld * Elem<DT>::bytes;
    if (k > 0)
      logprobs_kernel<DT, NT, true><<<n, NT, 0, s>>>(x, ld, V, tokens + r0, ignore, a, inv_temp, logp + r0, entropy + r0,
                                                     stats + 2 * r0, k, ids + r0 * k, top + r0 * k);
    else
      logprobs_kernel<DT, NT, false><<<n, NT, 0, s>>>(x, ld, V, tokens + r0, ignore, a, inv_temp, logp + r0,
                                                      entropy + r0, stats + 2 * r0, 0, nullptr, nullptr);
  }
}

}  // namespace

extern "C" {

int kf_token_logprobs_top_max() { return TOP_MAX; }

int kf_token_logprobs(const void* logits, int dt, long ld, long rows, int V, const long* tokens, long ignore, float temp,
                      float* logp, float* entropy, float* stats, int k, long* ids, float* top, hipStream_t s) {
  if (V < 1 || k < 0 || k > V || k > TOP_MAX || dt < DT_BF16 || dt > DT_FP32) return 1;
  const float a = 1.4426950408889634f / temp, inv = 1.f / temp;
  auto go = [&](auto DTc, auto NTc) {
    launch_fwd<decltype(DTc)::value, decltype(NTc)::value>(logits, ld, rows, V, tokens, ignore, a, inv, logp, entropy,
                                                           stats, k, ids, top, s);
  };
  auto by_type = [&](auto NTc) {
    if (dt == DT_BF16) go(std::integral_constant<int, DT_BF16>{}, NTc);
    else if (dt == DT_FP16) go(std::integral_constant<int, DT_FP16>{}, NTc);
    else go(std::integral_constant<int, DT_FP32>{}, NTc);
  };
  if (V > 16384) by_type(std::integral_constant<int, 1024>{});
  else by_type(std::integral_constant<int, 256>{});
  return 0;
}

int kf_token_logprobs_bwd(const void* logits, int dt, long ld, void* out, long ldo, long rows, int V, const long* tokens,
                          long ignore, const float* stats, const float* entropy, const float* dlogp, const float* dent,
                          float temp, hipStream_t s) {
  if (V < 1 || dt < DT_BF16 || dt > DT_FP32) return 1;
  const float a = 1.4426950408889634f / temp, inv = 1.f / temp;
  const int parts = cdiv((V + 7) / 8, BWD_NT * BWD_UN);
  const long per = std::max<long>(1, (1L << 23) / parts);     // rows of a launch: less than 2^32 threads
  for (long r0 = 0; r0 < rows; r0 += per) {
    const long n = std::min(per, rows - r0);
    auto go = [&](auto DTc) {
      constexpr int DT = decltype(DTc)::value;
      logprobs_bwd_kernel<DT><<<(unsigned)(n * parts), BWD_NT, 0, s>>>(
          (const char*)logits + r0 * ld * Elem<DT>::bytes, ld, (char*)out + r0 * ldo * Elem<DT>::bytes, ldo, V, parts,
          tokens + r0, ignore, stats + 2 * r0, entropy + r0, dlogp ? dlogp + r0 : nullptr, dent ? dent + r0 : nullptr, a,
          inv);
    };
    if (dt == DT_BF16) go(std::integral_constant<int, DT_BF16>{});
    else if (dt == DT_FP16) go(std::integral_constant<int, DT_FP16>{});
    else go(std::integral_constant<int, DT_FP32>{});
  }
  return 0;
}

}  // extern "C"
