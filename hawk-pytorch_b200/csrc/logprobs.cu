// Log probability of a given token, entropy and the most probable alternatives of rows of logits x [rows, V], and the logits'
// gradient:
//   m = max x,  s = sum e^(x - m),   log p_j = (x_j - m) - log s,   H = log s + sum p_j (m - x_j)   (no cancellation: all terms
//   of the last sum are positive),   d x_j = g_lp (onehot_j - p_j) - g_H p_j (log p_j + H).
// Bound by one read of the logits (the backward: one read, one write).  Measured at 3108 rows of 32000 in bf16: forward 50 us
// (4.0 TB/s; 72 % of the issue slots and 56 % of the MUFU rate, one exponential per logit), with 20 alternatives 88, backward 64
// (6.2 TB/s; a torch copy of the same bytes 71); 1551 rows of 31999 in fp32: 51 and 62 us; one row 6 to 8.
// Rows left out are not read by the forward (a fifth of the latter: 46 us); the backward requests a row before it knows of its token, and takes
// as long whatever is left out.
//
// Forward: a row belongs to a cluster of 1 to 8 blocks, which split it where there are few rows (one row of 32000 in one block is a
// chain of 16 16-byte loads per thread).  One pass: every thread keeps its running maximum and the sums relative to it; threads, warps
// and blocks (through distributed shared memory) are combined in the same form.  A token that is all but certain leaves s = 1.001,
// whose logarithm an fp32 s gives to 1e-4: where a block's s is under 2, the threads that hold its maximum add up the rest of their
// elements once more without it, and log s is log1p of that.
//
// Alternatives: the maxima of 64 subsets of a block's share (4 threads each) are ranked; the top-th largest is a bound that at
// least `top` elements reach, and for values in no particular order few more do.  Threads whose maximum reaches it read their
// vectors again (from L2) and collect what does; each candidate counts how many come before it (value, then index).  Where ties
// make that too many (a row that is mostly masked: every masked element reaches the bound) those above the bound are collected, and
// the first ones at it in the order of their indices; where even the former are too many (values in rising order) the alternatives
// are drawn one by one, each a maximum over what comes after the last.
#include <algorithm>

#include "common.cuh"

namespace hawk {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpAhead = 4;      // 16-byte vectors per thread in flight, twice; 2 or 3 with more blocks, 6 or 8 with fewer: 4 to 20 % slower
constexpr int kLpSubsets = 64;   // subsets whose maxima bound the alternatives
constexpr int kLpCand = 512;     // candidates a block keeps
constexpr int kLpMaxTop = 32, kLpMaxCluster = 8;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// e^d for d <= 0 as (2^t, t); t is floored where the result is 0 in any case, so that no product 0 * infinity arises
__device__ __forceinline__ float lp_exp(float d, float& t) {
  t = max_nan(d * kLog2e, -200.f);
  return ex2_approx(t);
}

// Sums over some of a row's elements, relative to their maximum m: of e = e^(x - m), apart from `ties` elements at the maximum that
// are counted instead (where it matters), and of e (x - m) log2 e.  NaN among the elements makes s NaN (m does not show it).
struct LpSums {
  float m, s, sx, ties;
  static __device__ __forceinline__ LpSums none() { return LpSums{-INFINITY, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ void raise(float to) {  // the same relative to `to` >= m
    if (to > m) {
      float t;
      const float k = lp_exp(m - to, t), all = s + ties;  // m = -infinity: k = 0
      sx = fmaf(all, t, sx) * k;
      s = all * k;
      ties = 0.f;
      m = to;
    }
  }
};

// An alternative as one number that orders as they do: by logit, then by falling index.  0: none.
typedef unsigned long long Cand;
__device__ __forceinline__ Cand make_cand(float x, int j) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 is 0
  return (Cand)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~j;
}
__device__ __forceinline__ int cand_id(Cand c) { return (int)~(uint32_t)c; }
__device__ __forceinline__ float cand_logit(Cand c) {
  const uint32_t u = (uint32_t)(c >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// how many of list[0..n) come before c
__device__ __forceinline__ int cands_before(const Cand* list, int n, Cand c) {
  int before = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) before += list[j] > c;
  return before;
}

struct LpShared {  // what the blocks of a cluster read of one another
  LpSums sums;
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
  __device__ __forceinline__ uint4 load_whole(int i) const { return __ldg(reinterpret_cast<const uint4*>(p + first(i))); }
  __device__ __forceinline__ uint4 load(int i) const { return whole(i) ? load_whole(i) : load_cut(i); }
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
// the lanes' sums together, in all of them
__device__ __forceinline__ LpSums warp_sums(LpSums v) {
  v.raise(warp_max(v.m));
  v.s = warp_sum(v.s);
  v.sx = warp_sum(v.sx);
  v.ties = warp_sum(v.ties);
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

// the largest of a thread's vectors
template <typename T, int K>
__device__ __forceinline__ float max_of(const uint4 (&v)[K]) {
  if (sizeof(T) == 2) {
    const auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    __nv_bfloat162 top = pair(v[0].x);
#pragma unroll
    for (int q = 0; q < K; ++q) top = __hmax2(__hmax2(top, __hmax2(pair(v[q].x), pair(v[q].y))), __hmax2(pair(v[q].z), pair(v[q].w)));
    const float2 f = __bfloat1622float2(top);
    return fmaxf(-INFINITY, fmaxf(f.x, f.y));
  }
  float top = -INFINITY;
#pragma unroll
  for (int q = 0; q < K; ++q)
    top = fmaxf(top, fmaxf(fmaxf(__uint_as_float(v[q].x), __uint_as_float(v[q].y)), fmaxf(__uint_as_float(v[q].z), __uint_as_float(v[q].w))));
  return top;
}

// a thread's vectors added to its sums
template <typename T, int K>
__device__ __forceinline__ void add_vectors(LpSums& a, const uint4 (&v)[K]) {
  constexpr int N = RowVec<T>::N;
  a.raise(max_of<T, K>(v));
  const float m = a.m == -INFINITY ? 0.f : a.m;  // only -infinity so far (or NaN): any number serves
  float2 sx = f2(0.f), s = f2(0.f);
#pragma unroll
  for (int q = 0; q < K; ++q) {
    float x[N];
    RowVec<T>::unpack(v[q], x);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      float2 t = mul2(add2(make_float2(x[j], x[j + 1]), f2(-m)), f2(kLog2e));
      t = make_float2(max_nan(t.x, -200.f), max_nan(t.y, -200.f));
      const float2 e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
      s = add2(s, e);
      sx = fma2(e, t, sx);
    }
  }
  a.s += s.x + s.y;
  a.sx += sx.x + sx.y;
}

// f(vector's index) for the vectors, from i0 on, of the warp's threads whose bit is set: the warp reads a thread's vectors together,
// one per lane, and four threads' at once
template <typename T, typename F>
__device__ __forceinline__ void vectors_of(const Row<T>& row, int i0, int i1, uint32_t threads, F f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  while (threads) {
    int first[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      first[q] = threads ? i0 + warp * 32 + __ffs(threads) - 1 + lane * kLpThreads : i1;
      threads &= threads - 1;
    }
    for (int ahead = 0; i0 + ahead < i1; ahead += 32 * kLpThreads) {
      uint4 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (first[q] + ahead < i1) v[q] = row.load(first[q] + ahead);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (first[q] + ahead < i1) f(first[q] + ahead, v[q]);
    }
  }
}

// the alternatives among a block's share, in order, to sh.best; `mine`: this thread's maximum
template <typename T>
__device__ __forceinline__ void block_alternatives(const Row<T>& row, int i0, int i1, float mine, int top, LpShared& sh, Cand* cand,
                                                   Cand* draw, float* subset, int* counters) {
  constexpr int N = RowVec<T>::N;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  {
    float w = mine;
    constexpr int kLanes = kLpThreads / kLpSubsets;
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
    if (lane % kLanes == 0) subset[tid / kLanes] = w;
  }
  if (tid < 2) counters[tid] = 0;
  __syncthreads();
  // the top-th largest of the subsets' maxima: each lane ranks two of them
  float bound = -INFINITY;
#pragma unroll
  for (int h = 0; h < kLpSubsets / 32; ++h) {
    const int i = lane + 32 * h;
    const float own = subset[i];
    int before = 0;
#pragma unroll
    for (int j = 0; j < kLpSubsets; j += 4) {
      const float4 o = *reinterpret_cast<const float4*>(subset + j);
      before += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own) + ((o.x == own) & (j < i)) + ((o.y == own) & (j + 1 < i)) +
                ((o.z == own) & (j + 2 < i)) + ((o.w == own) & (j + 3 < i));
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before == top - 1);
    if (hit) bound = __shfl_sync(0xffffffffu, own, __ffs(hit) - 1);
  }
  // f(element) for this thread's elements that lie in the row
  const auto each = [&](auto f) {
    for (int i = i0 + tid; i < i1; i += kLpThreads) {
      float x[N];
      RowVec<T>::unpack(row.load(i), x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int e = row.first(i) + j;
        if (e >= 0 && e < row.V && x[j] == x[j]) f(make_cand(x[j], e));
      }
    }
  };
  const auto rank_all = [&](int n) {  // cand[0..n) counted against one another
    for (int i = tid; i < n; i += kLpThreads) {
      const Cand c = cand[i];
      const int before = cands_before(cand, n, c);
      if (before < top) sh.best[before] = c;
    }
    if (tid == 0) sh.found = min(n, top);
  };
  // collects the elements that reach `least` of the warp's threads whose bit is set
  const auto collect = [&](uint32_t threads, float least, int* counter, int most) {
    vectors_of<T>(row, i0, i1, threads, [&](int i, uint4 raw) {
      float x[N];
      RowVec<T>::unpack(raw, x);
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) hits |= (x[j] >= least) << j;
      for (; hits; hits &= hits - 1) {
        const int e = row.first(i) + __ffs(hits) - 1;
        if (e < 0 || e >= row.V) continue;
        const int at = atomicAdd(counter, 1);
        if (at < most) cand[at] = make_cand(to_float(row.p[e]), e);
      }
    });
  };
  collect(__ballot_sync(0xffffffffu, mine >= bound), bound, &counters[0], kLpCand);
  __syncthreads();
  if (counters[0] <= kLpCand) {
    rank_all(counters[0]);
    return;
  }
  // the next float above the bound (0 of either sign is one value)
  const uint32_t bits = __float_as_uint(bound);
  const float above = bound == 0.f ? __uint_as_float(1u) : __uint_as_float(bits & 0x80000000u ? bits - 1 : bits + 1);
  collect(__ballot_sync(0xffffffffu, mine > bound), above, &counters[1], kLpCand - kLpMaxTop);
  __syncthreads();
  int n = counters[1];
  if (n <= kLpCand - kLpMaxTop) {
    // at least `top` elements reach the bound, so there are enough at it
    const int want = n + max(0, top - n);
    __shared__ int warp_counts[2][kLpWarps];
    for (int base = i0, step = 0; base < i1 && n < want; base += kLpThreads, step ^= 1) {
      const int i = base + tid;
      float x[N];
      uint32_t at_bound = 0;
      if (i < i1) {
        RowVec<T>::unpack(row.load(i), x);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int e = row.first(i) + j;
          if (x[j] == bound && e >= 0 && e < row.V) at_bound |= 1u << j;
        }
      }
      int before = __popc(at_bound);
      const int own = before;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += t;
      }
      if (lane == 31) warp_counts[step][warp] = before;
      __syncthreads();
      before -= own;
      int all = 0;
#pragma unroll
      for (int w = 0; w < kLpWarps; ++w) {
        const int c = warp_counts[step][w];
        if (w < warp) before += c;
        all += c;
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (at_bound >> j & 1) {
          if (n + before < want) cand[n + before] = make_cand(bound, row.first(i) + j);
          ++before;
        }
      n = min(want, n + all);
    }
    __syncthreads();
    rank_all(n);
    return;
  }
  Cand last = ~0ull;
  int k = 0;
  for (; k < top; ++k) {
    Cand next = 0;
    each([&](Cand c) {
      if (c < last && c > next) next = c;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) next = max(next, __shfl_xor_sync(0xffffffffu, next, o));
    if (lane == 0) draw[warp] = next;
    __syncthreads();
    next = draw[0];
    for (int w = 1; w < kLpWarps; ++w) next = max(next, draw[w]);
    __syncthreads();
    if (next == 0) break;
    if (tid == 0) sh.best[k] = next;
    last = next;
  }
  if (tid == 0) sh.found = k;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) lp_rows_kernel(LpArgs a) {
  __shared__ LpShared sh;
  __shared__ LpSums parts[kLpWarps];
  __shared__ __align__(16) float subset[kLpSubsets];
  __shared__ Cand cand[kLpCand], draw[kLpWarps];
  __shared__ int counters[2];
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
  LpSums sums = LpSums::none();
  const uint32_t minus = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -infinity
  {
    constexpr int kStep = kLpAhead * kLpThreads;
    const int w0 = row.whole(0) ? 0 : 1, w1 = min(i1, row.whole(row.vectors - 1) ? row.vectors : row.vectors - 1);  // whole vectors
    uint4 v[kLpAhead], next[kLpAhead];
    const auto load = [&](uint4 (&to)[kLpAhead], int base) {
      if (base >= w0 && base + kStep <= w1) {
#pragma unroll
        for (int q = 0; q < kLpAhead; ++q) to[q] = row.load_whole(base + tid + q * kLpThreads);
      } else {
#pragma unroll
        for (int q = 0; q < kLpAhead; ++q) {
          const int i = base + tid + q * kLpThreads;
          to[q] = i >= w0 && i < w1 ? row.load_whole(i) : make_uint4(minus, minus, minus, minus);
        }
      }
    };
    load(v, i0);
    for (int base = i0; base < w1; base += kStep) {
      load(next, base + kStep);
      if (base + warp * 32 < w1) add_vectors<T>(sums, v);
#pragma unroll
      for (int q = 0; q < kLpAhead; ++q) v[q] = next[q];
    }
    // the row's first and last vectors, where they are cut, by the threads whose they are
    for (int i = 0;; i = row.vectors - 1) {
      if (!row.whole(i) && i >= i0 && i < i1 && (i - i0) % kLpThreads / 32 == warp) {
        uint4 cut[1] = {make_uint4(minus, minus, minus, minus)};
        if ((i - i0) % 32 == lane) cut[0] = row.load_cut(i);
        add_vectors<T>(sums, cut);
      }
      if (i == row.vectors - 1) break;
    }
  }
  const float mine = sums.m;
  const LpSums all = warp_sums(sums);
  if (lane == 0) parts[warp] = all;
  __syncthreads();
  LpSums block = warp_sums(lane < kLpWarps ? parts[lane] : LpSums::none());
  if (block.s < 2.f) {  // see above; not for NaN
    const uint32_t holders = __ballot_sync(0xffffffffu, mine == block.m && block.m != -INFINITY);
    sums.raise(block.m);
    float s = mine == block.m ? 0.f : sums.s, ties = 0.f;
    vectors_of<T>(row, i0, i1, holders, [&](int, uint4 raw) {
      float x[RowVec<T>::N];
      RowVec<T>::unpack(raw, x);
#pragma unroll
      for (int j = 0; j < RowVec<T>::N; ++j) {
        float t;
        const float e = lp_exp(x[j] - block.m, t);
        if (x[j] == block.m) ties += 1.f; else s += e;
      }
    });
    s = warp_sum(s);
    ties = warp_sum(ties);
    __syncthreads();
    if (lane == 0) parts[warp] = LpSums{block.m, s, 0.f, ties};
    __syncthreads();
    const LpSums again = warp_sums(lane < kLpWarps ? parts[lane] : LpSums::none());
    block.s = again.s;
    block.ties = again.ties;
  }
  if (tid == 0) sh.sums = block;
  if (a.top > 0) block_alternatives<T>(row, i0, i1, mine, a.top, sh, cand, draw, subset, counters);

  // the cluster's blocks together, in the first of them
  if (blocks > 1) lp_cluster_sync(); else __syncthreads();
  if (rank == 0) {
    LpSums all = LpSums::none();  // lane b: block b's
    if (lane < (int)blocks) {
      all.m = __uint_as_float(lp_ld_remote(lp_remote(&sh.sums.m, lane)));
      all.s = __uint_as_float(lp_ld_remote(lp_remote(&sh.sums.s, lane)));
      all.sx = __uint_as_float(lp_ld_remote(lp_remote(&sh.sums.sx, lane)));
      all.ties = __uint_as_float(lp_ld_remote(lp_remote(&sh.sums.ties, lane)));
    }
    all = warp_sums(all);
    const float M = all.m;
    const bool nan = all.s != all.s;
    const float logs = log1pf((all.ties - 1.f) + all.s);  // -infinity where nothing is at a maximum
    if (tid == 0) {
      const float x = token < a.V ? to_float(row.p[token]) : __int_as_float(0x7fc00000);
      if (M == -INFINITY && !nan) {  // nothing but -infinity: no distribution
        a.logprob[r] = token < a.V ? -INFINITY : x;
        a.entropy[r] = 0.f;
      } else {
        a.logprob[r] = (x - M) - logs;
        a.entropy[r] = logs - kLn2 * all.sx / (all.s + all.ties);
      }
      a.stats[2 * r] = M;
      a.stats[2 * r + 1] = logs;
    }
    if (a.top > 0) {
      // all blocks' alternatives side by side; each again counts those before it.  What a block has too few of comes last: where
      // there are fewer numbers than alternatives, the others are NaN
      const int n = (int)blocks * a.top;
      Cand c = 0;
      if (tid < n) {
        const int b = tid / a.top, i = tid % a.top;
        if (i < (int)lp_ld_remote(lp_remote(&sh.found, b))) {
          const uint32_t at = lp_remote(&sh.best[i], b);
          c = (Cand)lp_ld_remote(at + 4) << 32 | lp_ld_remote(at);
        }
        cand[tid] = c;
      }
      __syncthreads();
      if (tid < n) {
        int before = cands_before(cand, n, c);
        if (c == 0)  // these are alike: in the order of their threads
          for (int j = 0; j < tid; ++j) before += cand[j] == 0;
        if (before < a.top) {
          const float x = c == 0 ? -INFINITY : cand_logit(c);
          a.top_lp[r * a.top + before] = x == -INFINITY ? -INFINITY : (x - M) - logs;
          a.top_id[r * a.top + before] = c == 0 ? -1 : cand_id(c);
        }
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
  const int share = (int)(blockIdx.x % a.shares), i0 = share * kLpBwdShare + threadIdx.x;
  const Row<T> row(static_cast<const T*>(a.x) + r * a.ld, a.V);
  const int w0 = row.whole(0) ? 0 : 1, w1 = row.whole(row.vectors - 1) ? row.vectors : row.vectors - 1;  // whole vectors
  uint4 v[kLpBwdVectors];
#pragma unroll
  for (int q = 0; q < kLpBwdVectors; ++q) {  // requested before anything is known of the row
    const int i = i0 + q * kLpBwdThreads;
    if (i >= w0 && i < w1) v[q] = row.load_whole(i);
  }
  const int64_t token = a.tokens[r];
  const float m = a.stats[2 * r], logs = a.stats[2 * r + 1], H = a.entropy[r], lp = a.logprob[r];
  const float gl = a.g_lp ? a.g_lp[r] : 0.f, gh = a.g_ent ? a.g_ent[r] : 0.f;
  T* dx = static_cast<T*>(a.dx) + r * a.V;
  const bool same = ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(row.p)) & 15) == 0;
  const bool none = token < 0 || (m == -INFINITY && logs == -INFINITY);  // left out, or nothing but -infinity
  const float nan = __int_as_float(0x7fc00000), scale = token >= a.V ? nan : -1.f;
  const float k0 = fmaf(gh, H, gl), k1 = gh * kLn2;
  // t = log2 p, floored where p is 0 (so that p t is): d = -p (gl + gh (log p + H))
  const auto gradient = [&](float2 x) {
    float2 t = mul2(add2(add2(x, f2(-m)), f2(-logs)), f2(kLog2e));
    t = make_float2(max_nan(t.x, -200.f), max_nan(t.y, -200.f));
    const float2 p = mul2(make_float2(ex2_approx(t.x), ex2_approx(t.y)), f2(scale)), g = mul2(p, fma2(t, f2(k1), f2(k0)));
    return none ? f2(0.f) : g;
  };
#pragma unroll
  for (int q = 0; q < kLpBwdVectors; ++q) {
    const int i = i0 + q * kLpBwdThreads, e = row.first(i);
    if (i < w0 || i >= w1) continue;
    float d[N], x[N];
    RowVec<T>::unpack(v[q], x);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const float2 g = gradient(make_float2(x[j], x[j + 1]));
      d[j] = g.x;
      d[j + 1] = g.y;
    }
    if (same) {
      VecIO<T, N>::store(dx + e, d);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) dx[e + j] = from_float<T>(d[j]);
    }
  }
  // elements of the row's cut vectors, by one warp of the first and last share
  if (threadIdx.x < 32) {
    for (int side = 0; side < 2; ++side) {
      const int i = side == 0 ? 0 : row.vectors - 1;
      if (row.whole(i) || i / kLpBwdShare != share || (side == 1 && i == 0)) continue;
      const int e = row.first(i) + (int)threadIdx.x;
      if ((int)threadIdx.x < N && e >= 0 && e < a.V) dx[e] = from_float<T>(gradient(f2(to_float(row.p[e]))).x);
    }
  }
  // the token's own element anew, by the thread that wrote it: 1 - p as -expm1(log p), as the token is often all but certain
  if (token >= 0 && token < a.V && !none) {
    const int i = ((int)token + row.off) / N, in = i - share * kLpBwdShare;
    const bool whole = i >= w0 && i < w1;
    if (in >= 0 && in < kLpBwdShare && (int)threadIdx.x == (whole ? in % kLpBwdThreads : (int)token - row.first(i)))
      dx[token] = from_float<T>(fmaf(-gl, expm1f(lp), -gh * expf(lp) * (lp == -INFINITY ? 0.f : lp + H)));
  }
}

// ---- host --------------------------------------------------------------------------------------------------
static int check_lp(int64_t rows, int64_t V, int64_t ld, int dtype) {
  HAWK_REQUIRE(valid_dtype(dtype), HAWK_ERR_DTYPE);
  HAWK_REQUIRE(rows >= 1 && rows < (1LL << 28) && V >= 1 && V < (1LL << 28) && ld >= V, HAWK_ERR_SHAPE);
  return HAWK_OK;
}

template <typename T>
static int lp_rows(LpArgs a, cudaStream_t st) {
  const int64_t vectors = ((int64_t)a.V + RowVec<T>::N - 1) / RowVec<T>::N + 1;
  // More blocks to a row while SMs are left without one and each block still has two vectors for a thread.  Blocks to a row against
  // us, 32000 in bf16: one row without alternatives 14 (1), 10 (2), 8 (4, 8); 64 rows with 20 alternatives 19 (1), 18 (2, 4), 25 (8);
  // 256 rows with 20: 23 (1), 27 (2), 37 (4): every block ranks alternatives of its own.  64 rows of 256000 with 5: 37, 27, 23, 25.
  int cluster = 1;
  while (cluster < kLpMaxCluster && a.rows * cluster < 148 && vectors > (int64_t)cluster * kLpThreads * 2) cluster *= 2;
  a.per = (int)((vectors + cluster - 1) / cluster);
  return launch_kernel(lp_rows_kernel<T>, dim3((unsigned)(a.rows * cluster)), dim3(kLpThreads), 0, st, false, (unsigned)cluster, a);
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
