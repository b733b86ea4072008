// Log probability of a given token, entropy and the most probable alternatives of rows of logits x [rows, V], and the logits'
// gradient:
//   m = max x,  s = sum e^(x - m),   log p_j = (x_j - m) - log s,   H = log s + sum p_j (m - x_j)   (no cancellation: all terms
//   of the last sum are positive),   d x_j = g_lp (onehot_j - p_j) - g_H p_j (log p_j + H).
// Bound by one read of the logits (the backward: one read, one write).
//
// Forward: a row belongs to a cluster of 1 to 8 blocks, which split it where there are few rows (one row of 32000 in one block:
// its load and its 64 exponentials per thread would be a chain of their own) or where it is long.  A block's share stays in
// registers between its one read and the three uses (maximum, exponentials, alternatives); shares of more than NV vectors per
// thread are read again, from L2 for the most part.  Blocks combine (m, s, sum) through distributed shared memory.
//
// Alternatives: the maxima of 64 subsets of a block's share are ranked; the top-th largest is a bound that at least `top`
// elements reach, and for values in no particular order few more do.  Those are collected, and each counts how many come before
// it (value, then index: ties go to the lowest index).  Where ties make the bound useless (a row that is mostly masked: every
// masked element reaches it) the alternatives are drawn one by one instead, each a maximum over what comes after the last.
#include <algorithm>

#include "common.cuh"

namespace hawk {

constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32;
constexpr int kLpSubsets = 64;   // subsets whose maxima bound the alternatives
constexpr int kLpCand = 512;     // candidates a block keeps
constexpr int kLpMaxTop = 32, kLpMaxCluster = 8;
constexpr float kLn2 = 0.6931471805599453f;

// e^d for d <= 0 as (2^t, t); t is floored where the result is 0 in any case, so that no product 0 * infinity arises.  A NaN
// stays one.
__device__ __forceinline__ float lp_exp(float d, float& t) {
  t = d * kLog2e;
  t = t < -200.f ? -200.f : t;
  return ex2_approx(t);
}

struct Cand {
  float x;
  int j;
};
__device__ __forceinline__ bool comes_before(const Cand& a, const Cand& b) { return a.x > b.x || (a.x == b.x && a.j < b.j); }

struct LpShared {  // what the blocks of a cluster read of one another
  float m, s, sx;  // maximum, sum of e^(x - m) over the other elements, sum of e^(x - m) (x - m) log2 e
  float ties;      // elements at the maximum
  int found;
  Cand best[kLpMaxTop];
};

struct LpArgs {
  const void* x;
  int64_t ld;               // row pitch, elements
  const int64_t* tokens;
  float *logprob, *entropy, *stats, *top_lp;  // stats [rows, 2]: m, log s
  int64_t* top_id;
  int64_t rows;
  int V, top, per;          // per: vectors of a block's share
};

template <typename T>
struct RowVec;  // 16 bytes of a row as floats
template <>
struct RowVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(uint4 r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint32_t bits(float v) { return __float_as_uint(v); }
};
template <>
struct RowVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 r, float (&v)[8]) {
    const float2 a = unpack_bf16x2(r.x), b = unpack_bf16x2(r.y), c = unpack_bf16x2(r.z), d = unpack_bf16x2(r.w);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y; v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
  }
};

// A row in 16-byte vectors that start at aligned addresses: vector i holds elements [i * N - off, ...), where off is how far the
// row's start lies behind a boundary.  The first and last may be cut; what lies outside the row reads as -infinity.
template <typename T>
struct Row {
  static constexpr int N = RowVec<T>::N;
  const T* p;
  int off, V, vectors;
  __device__ __forceinline__ Row(const T* row, int V_) : p(row), V(V_) {
    off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    vectors = (off + V + N - 1) / N;
  }
  __device__ __forceinline__ int first(int i) const { return i * N - off; }
  __device__ __forceinline__ bool whole(int i) const { return first(i) >= 0 && first(i) + N <= V; }
  __device__ __forceinline__ uint4 load(int i) const {
    if (whole(i)) return __ldg(reinterpret_cast<const uint4*>(p + first(i)));
    return load_cut(i);
  }
  __device__ __noinline__ uint4 load_cut(int i) const {
    alignas(16) T t[N];
    for (int j = 0; j < N; ++j) {
      const int e = first(i) + j;
      t[j] = e >= 0 && e < V ? p[e] : from_float<T>(-INFINITY);
    }
    return *reinterpret_cast<const uint4*>(t);
  }
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ uint32_t lp_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void lp_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t lp_remote(const void* p, uint32_t rank) {  // `p` in the block of that rank
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t lp_ld_remote(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// f(vector's index, its 16 bytes) for the vectors of this thread: the NV in registers, then (LONG) the rest of the share
template <typename T, int NV, bool LONG, typename F>
__device__ __forceinline__ void each_vector(const Row<T>& row, const uint4 (&v)[NV], int i0, int i1, F f) {
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int i = i0 + threadIdx.x + q * kLpThreads;
    if (i < i1) f(i, v[q]);
  }
  if (LONG)
    for (int i = i0 + threadIdx.x + NV * kLpThreads; i < i1; i += kLpThreads) f(i, row.load(i));
}

template <typename T, int NV, bool LONG>
__global__ void __launch_bounds__(kLpThreads, 2) lp_rows_kernel(LpArgs a) {
  constexpr int N = RowVec<T>::N;
  __shared__ LpShared sh;
  __shared__ float red[4][kLpWarps], subset[kLpSubsets];
  __shared__ Cand cand[kLpCand], draw[kLpWarps];
  __shared__ int ncand;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t blocks, rank = lp_cluster_rank();
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  const int64_t r = blockIdx.x / blocks;
  const int64_t token = a.tokens[r];
  if (token < 0) {  // left out: the same for all blocks of the cluster
    if (rank == 0) {
      if (tid == 0) {
        a.logprob[r] = 0.f;
        a.entropy[r] = 0.f;
        a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
      }
      if (tid < a.top) {
        a.top_lp[r * a.top + tid] = -INFINITY;
        a.top_id[r * a.top + tid] = -1;
      }
    }
    return;
  }
  const Row<T> row(static_cast<const T*>(a.x) + r * a.ld, a.V);
  const int i0 = min((int)rank * a.per, row.vectors), i1 = min(i0 + a.per, row.vectors);
  uint4 v[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    const int i = i0 + tid + q * kLpThreads;
    if (i < i1) v[q] = row.load(i);
  }
  const auto each = [&](auto f) { each_vector<T, NV, LONG>(row, v, i0, i1, f); };

  // 1. the maximum
  float tmax = -INFINITY;
  each([&](int, uint4 raw) {
    float x[N];
    RowVec<T>::unpack(raw, x);
#pragma unroll
    for (int j = 0; j < N; ++j) tmax = fmaxf(tmax, x[j]);
  });
  {
    float w = tmax;  // subsets: 8 lanes each
#pragma unroll
    for (int o = 1; o < 32 * kLpWarps / kLpSubsets; o <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
    constexpr int kPerWarp = kLpSubsets / kLpWarps;
    if (lane % (32 / kPerWarp) == 0) subset[warp * kPerWarp + lane / (32 / kPerWarp)] = w;
    w = warp_max(w);
    if (lane == 0) red[0][warp] = w;
  }
  if (tid == 0) ncand = 0;
  __syncthreads();
  const float m = warp_max(lane < kLpWarps ? red[0][lane] : -INFINITY);

  // 2. the sums, of the terms below 1 alone: log s = log1p of them is then as exact for a token that is all but certain (s = 1.001)
  // as for any other.  Only threads that hold a maximum have to look for it.  Where m is -infinity no number is here: there is nothing to add, but a NaN (which no maximum shows) is to be seen
  float s = 0.f, sx = 0.f, ties = 0.f;
  if (m == -INFINITY)
    each([&](int, uint4 raw) {
      float x[N];
      RowVec<T>::unpack(raw, x);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (x[j] != x[j]) s = x[j];
    });
  else if (tmax == m)
    each([&](int, uint4 raw) {
      float x[N];
      RowVec<T>::unpack(raw, x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float t;
        const float e = lp_exp(x[j] - m, t);
        ties += x[j] == m ? 1.f : 0.f;
        s += x[j] == m ? (t - t) : e;  // 0; NaN where m is infinite
        sx = fmaf(e, t, sx);
      }
    });
  else
    each([&](int, uint4 raw) {
      float x[N];
      RowVec<T>::unpack(raw, x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float t;
        const float e = lp_exp(x[j] - m, t);
        s += e;
        sx = fmaf(e, t, sx);
      }
    });
  s = warp_sum(s);
  sx = warp_sum(sx);
  ties = warp_sum(ties);
  if (lane == 0) {
    red[1][warp] = s;
    red[2][warp] = sx;
    red[3][warp] = ties;
  }

  // 3. the alternatives among this block's elements, in order, to sh.best
  if (a.top > 0) {
    // the top-th largest of the subsets' maxima: each lane ranks two of them
    float bound = -INFINITY;
#pragma unroll
    for (int h = 0; h < kLpSubsets / 32; ++h) {
      const int i = lane + 32 * h;
      const float mine = subset[i];
      int before = 0;
      for (int j = 0; j < kLpSubsets; ++j) {
        const float o = subset[j];
        before += o > mine || (o == mine && j < i);
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, before == a.top - 1);
      if (hit) bound = __shfl_sync(0xffffffffu, mine, __ffs(hit) - 1);
    }
    each([&](int i, uint4 raw) {
      float x[N], vm = -INFINITY;
      RowVec<T>::unpack(raw, x);
#pragma unroll
      for (int j = 0; j < N; ++j) vm = fmaxf(vm, x[j]);
      if (vm >= bound) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int e = row.first(i) + j;
          if (x[j] >= bound && e >= 0 && e < a.V) {
            const int at = atomicAdd(&ncand, 1);
            if (at < kLpCand) cand[at] = Cand{x[j], e};
          }
        }
      }
    });
    __syncthreads();
    const int n = ncand;
    if (n <= kLpCand) {
      for (int i = tid; i < n; i += kLpThreads) {
        const Cand c = cand[i];
        int before = 0;
        for (int j = 0; j < n; ++j) before += comes_before(cand[j], c);
        if (before < a.top) sh.best[before] = c;
      }
      if (tid == 0) sh.found = min(n, a.top);
    } else {
      Cand last{INFINITY, -1};
      int k = 0;
      for (; k < a.top; ++k) {
        Cand mine{-INFINITY, 0x7fffffff};
        each([&](int i, uint4 raw) {
          float x[N];
          RowVec<T>::unpack(raw, x);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const Cand c{x[j], row.first(i) + j};
            if (c.j >= 0 && c.j < a.V && comes_before(last, c) && comes_before(c, mine)) mine = c;
          }
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const Cand c{__shfl_xor_sync(0xffffffffu, mine.x, o), __shfl_xor_sync(0xffffffffu, mine.j, o)};
          if (comes_before(c, mine)) mine = c;
        }
        if (lane == 0) draw[warp] = mine;
        __syncthreads();
        mine = draw[0];
        for (int w = 1; w < kLpWarps; ++w)
          if (comes_before(draw[w], mine)) mine = draw[w];
        __syncthreads();
        if (mine.j == 0x7fffffff) break;
        if (tid == 0) sh.best[k] = mine;
        last = mine;
      }
      if (tid == 0) sh.found = k;
    }
  }
  __syncthreads();
  if (warp == 0) {
    const float bs = warp_sum(lane < kLpWarps ? red[1][lane] : 0.f), bx = warp_sum(lane < kLpWarps ? red[2][lane] : 0.f),
                bt = warp_sum(lane < kLpWarps ? red[3][lane] : 0.f);
    if (lane == 0) {
      sh.m = m;
      sh.s = bs;
      sh.sx = bx;
      sh.ties = bt;
    }
  }

  // 4. the cluster's blocks together, in the first of them
  if (blocks > 1) lp_cluster_sync(); else __syncthreads();
  if (rank == 0) {
    float M = -INFINITY, S = 0.f, SX = 0.f, ties = 0.f;  // S without the elements at the maximum
    for (uint32_t b = 0; b < blocks; ++b) M = fmaxf(M, __uint_as_float(lp_ld_remote(lp_remote(&sh.m, b))));
    for (uint32_t b = 0; b < blocks; ++b) {
      const float bm = __uint_as_float(lp_ld_remote(lp_remote(&sh.m, b))), bs = __uint_as_float(lp_ld_remote(lp_remote(&sh.s, b)));
      if (bm == -INFINITY) {
        S += bs;  // 0 or NaN
        continue;
      }
      float t;
      const float k = lp_exp(bm - M, t), bt = __uint_as_float(lp_ld_remote(lp_remote(&sh.ties, b))), ball = bs + bt;
      if (bm == M) ties += bt;
      S = fmaf(bm == M ? bs : ball, k, S);
      SX = fmaf(fmaf(ball, t, __uint_as_float(lp_ld_remote(lp_remote(&sh.sx, b)))), k, SX);  // terms move by (m_b - M) log2 e
    }
    const float logs = log1pf((ties - 1.f) + S);  // no element at a maximum: -infinity of 0, or NaN
    if (tid == 0) {
      const float x = token < a.V ? to_float(row.p[token]) : __int_as_float(0x7fc00000);
      if (M == -INFINITY && S == 0.f) {  // nothing but -infinity: no distribution
        a.logprob[r] = token < a.V ? -INFINITY : x;
        a.entropy[r] = 0.f;
      } else {
        a.logprob[r] = (x - M) - logs;
        a.entropy[r] = logs - kLn2 * SX / (S + ties);
      }
      a.stats[2 * r] = M;
      a.stats[2 * r + 1] = logs;
    }
    if (a.top > 0) {
      // all blocks' alternatives side by side; each again counts those before it
      int n = 0;
      for (uint32_t b = 0; b < blocks; ++b) {
        const int k = (int)lp_ld_remote(lp_remote(&sh.found, b));
        if (tid < k) {
          cand[n + tid].x = __uint_as_float(lp_ld_remote(lp_remote(&sh.best[tid].x, b)));
          cand[n + tid].j = (int)lp_ld_remote(lp_remote(&sh.best[tid].j, b));
        }
        n += k;
      }
      __syncthreads();
      if (tid < n) {
        const Cand c = cand[tid];
        int before = 0;
        for (int j = 0; j < n; ++j) before += comes_before(cand[j], c);
        if (before < a.top) {
          a.top_lp[r * a.top + before] = c.x == -INFINITY ? -INFINITY : (c.x - M) - logs;
          a.top_id[r * a.top + before] = c.j;
        }
      }
      if (tid >= n && tid < a.top) {  // fewer numbers than alternatives: the others are NaN
        a.top_lp[r * a.top + tid] = -INFINITY;
        a.top_id[r * a.top + tid] = -1;
      }
    }
  }
  if (blocks > 1) lp_cluster_sync();  // no block leaves while its shared memory is read
}

// ---- backward: a block per row and share of it ---------------------------------------------------------------
struct LpBwdArgs {
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  const float *stats, *logprob, *entropy, *g_lp, *g_ent;  // upstream gradients; null: none
  void* dx;                                               // [rows, V] contiguous
  int V, shares;
};
constexpr int kLpBwdVectors = 4, kLpBwdThreads = 256, kLpBwdShare = kLpBwdVectors * kLpBwdThreads;

template <typename T>
__global__ void __launch_bounds__(kLpBwdThreads) lp_bwd_kernel(LpBwdArgs a) {
  constexpr int N = RowVec<T>::N;
  const int64_t r = blockIdx.x / a.shares;
  const int i0 = (int)(blockIdx.x % a.shares) * kLpBwdShare + threadIdx.x;
  const int64_t token = a.tokens[r];
  const Row<T> row(static_cast<const T*>(a.x) + r * a.ld, a.V);
  T* dx = static_cast<T*>(a.dx) + r * a.V;
  const bool same = ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(row.p)) & 15) == 0;
  uint4 v[kLpBwdVectors];
  if (token >= 0)
#pragma unroll
    for (int q = 0; q < kLpBwdVectors; ++q)
      if (i0 + q * kLpBwdThreads < row.vectors) v[q] = row.load(i0 + q * kLpBwdThreads);
  const float m = a.stats[2 * r], logs = a.stats[2 * r + 1], H = a.entropy[r];
  const float gl = a.g_lp ? a.g_lp[r] : 0.f, gh = a.g_ent ? a.g_ent[r] : 0.f;
#pragma unroll
  for (int q = 0; q < kLpBwdVectors; ++q) {
    const int i = i0 + q * kLpBwdThreads;
    if (i >= row.vectors) break;
    float d[N];
    if (token < 0 || (m == -INFINITY && logs == -INFINITY)) {  // left out, or nothing but -infinity
#pragma unroll
      for (int j = 0; j < N; ++j) d[j] = 0.f;
    } else {
      float x[N];
      RowVec<T>::unpack(v[q], x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float t;
        const float p = lp_exp((x[j] - m) - logs, t);  // t: log2 p
        d[j] = -p * fmaf(gh, fmaf(t, kLn2, H), gl);
      }
      const int64_t at = token - row.first(i);
      if (at >= 0 && at < N) {
        // 1 - p as -expm1(log p): the token is often all but certain
        const float lp = a.logprob[r], own = fmaf(-gl, expm1f(lp), -gh * expf(lp) * (lp == -INFINITY ? 0.f : lp + H));
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j == (int)at) d[j] = own;
      }
      if (token >= a.V)
#pragma unroll
        for (int j = 0; j < N; ++j) d[j] = __int_as_float(0x7fc00000);
    }
    const int e = row.first(i);
    if (same && row.whole(i)) {
      VecIO<T, N>::store(dx + e, d);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (e + j >= 0 && e + j < a.V) dx[e + j] = from_float<T>(d[j]);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------
static int check_lp(int64_t rows, int64_t V, int64_t ld, int dtype) {
  HAWK_REQUIRE(valid_dtype(dtype), HAWK_ERR_DTYPE);
  HAWK_REQUIRE(rows >= 1 && rows < (1LL << 28) && V >= 1 && V < (1LL << 28) && ld >= V, HAWK_ERR_SHAPE);
  return HAWK_OK;
}

template <typename T, int NV, bool LONG>
static int launch_rows(const LpArgs& a, int cluster, cudaStream_t st) {
  return launch_kernel(lp_rows_kernel<T, NV, LONG>, dim3((unsigned)(a.rows * cluster)), dim3(kLpThreads), 0, st, false, (unsigned)cluster, a);
}

template <typename T>
static int lp_rows(LpArgs a, cudaStream_t st) {
  const int64_t vectors = ((int64_t)a.V + RowVec<T>::N - 1) / RowVec<T>::N + 1;
  // as few blocks to a row as hold it in registers; more where that leaves SMs idle, down to a vector per thread
  int cluster = 1;
  while (cluster < kLpMaxCluster && (vectors > (int64_t)cluster * kLpThreads * 8 ||
                                     (a.rows * cluster * 2 <= 148 && vectors > (int64_t)cluster * kLpThreads)))
    cluster *= 2;
  a.per = (int)((vectors + cluster - 1) / cluster);
  if (a.per <= kLpThreads) return launch_rows<T, 1, false>(a, cluster, st);
  if (a.per <= 2 * kLpThreads) return launch_rows<T, 2, false>(a, cluster, st);
  if (a.per <= 4 * kLpThreads) return launch_rows<T, 4, false>(a, cluster, st);
  if (a.per <= 8 * kLpThreads) return launch_rows<T, 8, false>(a, cluster, st);
  return launch_rows<T, 8, true>(a, cluster, st);
}

}  // namespace hawk

using namespace hawk;

extern "C" int hawk_token_logprobs(const void* logits, int64_t ld, const int64_t* tokens, float* logprob, float* entropy, float* stats,
                                   float* top_logprob, int64_t* top_id, int64_t rows, int64_t V, int top, int dtype, void* stream) {
  HAWK_REQUIRE(logits && tokens && logprob && entropy && stats && (top == 0 || (top_logprob && top_id)), HAWK_ERR_NULL);
  const int ok = check_lp(rows, V, ld, dtype);
  if (ok != HAWK_OK) return ok;
  HAWK_REQUIRE(top >= 0 && top <= kLpMaxTop && top <= V, HAWK_ERR_SHAPE);
  HAWK_REQUIRE(aligned(logits, dtype_size(dtype)) && aligned(tokens, 8) && aligned(logprob, 4) && aligned(entropy, 4) &&
                   aligned(stats, 4) && aligned(top_logprob, 4) && aligned(top_id, 8),
               HAWK_ERR_ALIGN);
  LpArgs a{logits, ld, tokens, logprob, entropy, stats, top_logprob, top_id, rows, (int)V, top, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == HAWK_F32 ? lp_rows<float>(a, st) : lp_rows<__nv_bfloat16>(a, st);
}

extern "C" int hawk_token_logprobs_bwd(const void* logits, int64_t ld, const int64_t* tokens, const float* stats, const float* logprob,
                                       const float* entropy, const float* g_logprob, const float* g_entropy, void* dlogits, int64_t rows,
                                       int64_t V, int dtype, void* stream) {
  HAWK_REQUIRE(logits && tokens && stats && logprob && entropy && dlogits, HAWK_ERR_NULL);
  const int ok = check_lp(rows, V, ld, dtype);
  if (ok != HAWK_OK) return ok;
  HAWK_REQUIRE(aligned(logits, dtype_size(dtype)) && aligned(dlogits, dtype_size(dtype)) && aligned(tokens, 8) && aligned(stats, 4) &&
                   aligned(logprob, 4) && aligned(entropy, 4) && aligned(g_logprob, 4) && aligned(g_entropy, 4),
               HAWK_ERR_ALIGN);
  const int n = dtype == HAWK_F32 ? 4 : 8;
  const int64_t vectors = (V + n - 1) / n + 1, shares = (vectors + kLpBwdShare - 1) / kLpBwdShare;
  HAWK_REQUIRE(rows * shares < (1LL << 31), HAWK_ERR_SHAPE);
  const LpBwdArgs a{logits, ld, tokens, stats, logprob, entropy, g_logprob, g_entropy, dlogits, (int)V, (int)shares};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == HAWK_F32) lp_bwd_kernel<float><<<(unsigned)(rows * shares), kLpBwdThreads, 0, st>>>(a);
  else lp_bwd_kernel<__nv_bfloat16><<<(unsigned)(rows * shares), kLpBwdThreads, 0, st>>>(a);
  return launch_status();
}
