// Embedding of token ids, out[i] = scale * W[ids[i]], and the table's gradient
//   dW[v] = scale * sum over { i : ids[i] = v } of dout[i],
// summed in fp32 in the order of the positions and rounded once: the same bits on every run (adding rows with atomics is
// neither ordered nor, in bf16, exact).  Both are bound by memory: the forward by N rows read and written, the backward by
// N rows read and V rows written, the rows that no token names among them.
//
// Measured (32768 tokens as frequent as in text, V32000 H2048): forward 55 us fp32 (6.2 TB/s), 29 bf16; backward 135 us fp32 of
// 81 for its 530 MB alone, 103 bf16: group 23, windows 30, rows 83.
//
// Backward, three launches (up to 2048 tokens one, embed_small_kernel):
//   1. group   the positions of each id side by side, in their order (a stable counting sort).  A block owns one id in 128 (EmbedOrder)
//              and reads all ids (from L2: 128 blocks x 8 B, against rows of kilobytes): it counts those of the blocks before it,
//              which gives its place in the result without a word from them, and queues its own in shared memory in their order.
//              The queue's warps rank equal ids among their 32 (match.any) and take turns at the counters.  (Blocks that own a range
//              of ids each: the frequent tokens of a vocabulary have low ids, the first block had half of a text's tokens and took
//              143 us.)
//   2. windows sums of 8 consecutive places that lie in a run of more than 16 positions of one id (the most frequent token of a text
//              is 5 to 10 % of it, and one warp would walk its rows alone).  Windows of 16 in runs of more than 32: 144 and 116 us
//              backward, 42 instead of 34 for 1551 tokens at H512.
//   3. rows    a warp per 8 table rows and 512 columns walks the places of its rows as one stream, three rows of dout ahead whichever
//              table rows they belong to (most have no position or one: a loop per row would wait for each); zeros where there is
//              nothing.  Long runs it passes over: the first blocks add them up from their windows' sums and ragged ends.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace hawk {

template <>
struct VecIO<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[1]) { v[0] = __ldg(p); }
  static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};
template <>
struct VecIO<__nv_bfloat16, 1> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[1]) { v[0] = __bfloat162float(__ldg(p)); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
};

// VEC elements as they are stored
template <typename T, int VEC>
struct Raw {
  static constexpr int B = VEC * sizeof(T);
  using type = std::conditional_t<B == 16, uint4, std::conditional_t<B == 8, uint2, std::conditional_t<B == 4, uint32_t, uint16_t>>>;
  static __device__ __forceinline__ type load(const T* p) { return __ldg(reinterpret_cast<const type*>(p)); }
  static __device__ __forceinline__ void unpack(const type& r, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = reinterpret_cast<const float*>(&r)[j];
    } else if constexpr (VEC == 1) {
      v[0] = __uint_as_float((uint32_t)r << 16);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float2 f = unpack_bf16x2(reinterpret_cast<const uint32_t*>(&r)[j / 2]);
        v[j] = f.x;
        v[j + 1] = f.y;
      }
    }
  }
};

// ---- forward: 2^log_tpr threads to a row, four vectors of each in flight -----------------------------------
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const int64_t* __restrict__ ids, const T* __restrict__ w, T* __restrict__ out,
                                                        int64_t N, int64_t V, int H, float scale, int log_tpr) {
  const int tpr = 1 << log_tpr;
  const int64_t row = (int64_t)blockIdx.x * (256 >> log_tpr) + (threadIdx.x >> log_tpr);
  if (row >= N) return;
  const int64_t id = ids[row];
  const bool known = id >= 0 && id < V;
  const T* src = w + (known ? id : 0) * H;
  T* dst = out + row * H;
  for (int c0 = (threadIdx.x & (tpr - 1)) * VEC; c0 < H; c0 += 4 * tpr * VEC) {
    typename Raw<T, VEC>::type r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + u * tpr * VEC < H) r[u] = Raw<T, VEC>::load(src + c0 + u * tpr * VEC);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + u * tpr * VEC < H) {
        float v[VEC];
        Raw<T, VEC>::unpack(r[u], v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = known ? v[j] * scale : __int_as_float(0x7fc00000);
        VecIO<T, VEC>::store(dst + c0 + u * tpr * VEC, v);
      }
  }
}

// ---- backward 1: positions grouped by id ---------------------------------------------------------------------
// Where the positions of id v come in the order of the groups: with those of its block, and there the ids whose quotients lie
// slots / 8 apart next to one another, so that the 8 table rows of a warp are one that may be frequent and 7 rarer ones (8
// neighbouring quotients: the first warp had 8 rows of 60 positions each to add, 158 us where 60 were left to do).  Low ids go to
// all blocks alike (the frequent tokens of a vocabulary have them), and so do ids any power of two apart.
constexpr int kRowGroup = 8;
struct EmbedOrder {
  int log_blocks, slots;  // slots: ids of a block, a multiple of kRowGroup
  __host__ __device__ int64_t groups() const { return (int64_t)slots << log_blocks; }
  __device__ int block(int64_t v) const { return (int)(v + (v >> log_blocks) * 37) & ((1 << log_blocks) - 1); }
  __device__ int slot(int64_t v) const {  // within its block
    const int x = (int)(v >> log_blocks), q = slots / kRowGroup;
    return x % q * kRowGroup + x / q;
  }
  __device__ int64_t id(int64_t place) const {  // of the slot at place block * slots + slot
    const int64_t b = place / slots, s = place % slots, x = s % kRowGroup * (slots / kRowGroup) + s / kRowGroup;
    return x << log_blocks | ((b - x * 37) & ((1 << log_blocks) - 1));
  }
};
constexpr int kGroupThreads = 1024, kIdsPerThread = 8, kGroupStep = kGroupThreads * kIdsPerThread;
constexpr int kMinQueue = kGroupStep, kMaxQueue = 3 * kGroupStep;  // one step's ids always fit; 192 KB at most
constexpr int kMaxSlots = 4096, kMinLogBlocks = 7;
constexpr int kWindow = 8, kLong = 2 * kWindow;  // a run of more than kLong positions holds a whole window

// exclusive sum over the block's threads; `all`: of all of them.  The shared words may be reused after the next barrier.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += t;
  }
  all = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return inc - v + (warp > 0 ? before : 0);
}

// One step's ids of this thread: its 8 positions are consecutive, so the threads are in the order of the positions.
struct StepIds {
  int64_t id[kIdsPerThread];
  __device__ __forceinline__ void load(const int64_t* ids, int64_t i0, int64_t N) {
    if (i0 + kIdsPerThread <= N && aligned16(ids)) {  // i0 is a multiple of 8
#pragma unroll
      for (int q = 0; q < kIdsPerThread / 2; ++q) {
        const longlong2 t = __ldg(reinterpret_cast<const longlong2*>(ids + i0) + q);
        id[2 * q] = t.x;
        id[2 * q + 1] = t.y;
      }
    } else {
#pragma unroll
      for (int q = 0; q < kIdsPerThread; ++q) id[q] = i0 + q < N ? __ldg(ids + i0 + q) : -1;
    }
  }
  // which of them are this block's; `below` counts those of the blocks before it
  __device__ __forceinline__ uint32_t mine(int64_t V, int64_t padding, EmbedOrder order, int block, int& below) const {
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < kIdsPerThread; ++q) {
      if (id[q] < 0 || id[q] >= V || id[q] == padding) continue;
      const int b = order.block(id[q]);
      below += b < block;
      if (b == block) m |= 1u << q;
    }
    return m;
  }
};

// hands out the places of n queued (slot, position) pairs; the whole block
__device__ __forceinline__ void place(const uint2* queue, int n, int* cursor, int* perm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int k = 0; k < n; k += kGroupThreads) {
    const int i = k + threadIdx.x, warps = min(kGroupThreads / 32, (n - k + 31) / 32);
    const bool have = i < n;
    const uint32_t active = __ballot_sync(0xffffffffu, have);
    uint2 q = make_uint2(0u, 0u);
    uint32_t peers = 0;
    if (have) {
      q = queue[i];
      peers = __match_any_sync(active, q.x);
    }
    const int rank = __popc(peers & ((1u << lane) - 1));
    int at = 0;
    for (int w = 0; w < warps; ++w) {  // in the order of the positions
      if (w == warp && have) {
        at = cursor[q.x];
        __syncwarp(active);
        if (rank == 0) cursor[q.x] = at + __popc(peers);
      }
      __syncthreads();
    }
    if (have) perm[at + rank] = (int)q.y;
  }
}

__global__ void __launch_bounds__(kGroupThreads) embed_group_kernel(const int64_t* __restrict__ ids, int64_t N, int64_t V, int64_t padding,
                                                                    EmbedOrder order, int* __restrict__ perm, int* __restrict__ start,
                                                                    int* __restrict__ owner, int4* __restrict__ runs, int windows,
                                                                    int queue_size) {
  extern __shared__ uint2 queue[];                           // [queue_size]
  int* count = reinterpret_cast<int*>(queue + queue_size);   // [slots], the cursors later
  __shared__ int warp_sums[2][32];
  __shared__ int nruns;
  const int tid = threadIdx.x, slots = order.slots;
  for (int j = tid; j < slots; j += kGroupThreads) count[j] = 0;
  if (tid == 0) nruns = 0;
  int below = 0, total = 0, all, step = 0;
  StepIds s, next;
  s.load(ids, tid * kIdsPerThread, N);
  __syncthreads();
  for (int64_t base = 0; base < N; base += kGroupStep, step ^= 1) {  // the scans take turns with their shared words
    const int64_t i0 = base + tid * kIdsPerThread;
    if (base + kGroupStep < N) next.load(ids, i0 + kGroupStep, N);
    const uint32_t mine = s.mine(V, padding, order, blockIdx.x, below);
    int at = total + block_scan(__popc(mine), warp_sums[step], all);
#pragma unroll
    for (int q = 0; q < kIdsPerThread; ++q)
      if (mine >> q & 1) {
        const int j = order.slot(s.id[q]);
        atomicAdd(&count[j], 1);
        if (at < queue_size) queue[at] = make_uint2((uint32_t)j, (uint32_t)(i0 + q));
        ++at;
      }
    total += all;
    s = next;
  }
  __syncthreads();
  int ahead;
  block_scan(below, warp_sums[0], ahead);
  __syncthreads();
  // counts -> first places
  constexpr int kPer = kMaxSlots / kGroupThreads;
  int c[kPer], sum = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int j = tid * kPer + q;
    c[q] = j < slots ? count[j] : 0;
    sum += c[q];
  }
  int at = ahead + block_scan(sum, warp_sums[1], all);
  int* mystart = start + (int64_t)blockIdx.x * slots;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int j = tid * kPer + q;
    if (j < slots) count[j] = mystart[j] = at;
    at += c[q];
    if (windows > 0 && c[q] > kLong)  // in any order
      runs[(int64_t)blockIdx.x * (slots + 1) + 1 + atomicAdd(&nruns, 1)] = make_int4(at - c[q], at, (int)blockIdx.x * slots + j, 0);
  }
  const int behind = ahead + total;
  __syncthreads();
  if (windows > 0 && tid == 0) runs[(int64_t)blockIdx.x * (slots + 1)] = make_int4(nruns, 0, 0, 0);
  if (blockIdx.x == gridDim.x - 1 && tid == 0) mystart[slots] = behind;
  // whose long run each window lies in (-1: none): the windows that start in this block's share, and those behind the last share
  const int w_end = blockIdx.x == gridDim.x - 1 ? windows : min(windows, (behind + kWindow - 1) / kWindow);
  for (int w = (ahead + kWindow - 1) / kWindow + tid; w < w_end; w += kGroupThreads) {
    int lo = 0, hi = slots;  // the last slot that starts at or before the window
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (count[mid] <= w * kWindow) lo = mid; else hi = mid;
    }
    const int end = lo + 1 < slots ? count[lo + 1] : behind;
    owner[w] = end - count[lo] > kLong && (w + 1) * kWindow <= end ? (int)(blockIdx.x * slots + lo) : -1;
  }
  __syncthreads();
  if (total <= queue_size) {
    place(queue, total, count, perm);
    return;
  }
  for (int64_t base = 0; base < N; base += kGroupStep, step ^= 1) {  // more than the queue holds: read the ids again
    const int64_t i0 = base + tid * kIdsPerThread;
    s.load(ids, i0, N);
    const uint32_t mine = s.mine(V, padding, order, blockIdx.x, below);
    int to = block_scan(__popc(mine), warp_sums[step], all);
#pragma unroll
    for (int q = 0; q < kIdsPerThread; ++q)
      if (mine >> q & 1) queue[to++] = make_uint2((uint32_t)order.slot(s.id[q]), (uint32_t)(i0 + q));
    __syncthreads();
    place(queue, all, count, perm);
    __syncthreads();
  }
}

// ---- backward 2 and 3: sums --------------------------------------------------------------------------------

template <typename T>
__host__ __device__ constexpr int unit_vectors(int vec) { return vec == 1 ? 8 : 512 / (32 * vec); }  // vectors per lane: 512 columns (256 in the scalar form)

// a warp per window and 32 * VEC columns, all of its rows in flight
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_window_kernel(const T* __restrict__ dout, const int* perm, const int* owner, float* partial, int H,
                                                           int narrow, int64_t units) {
  pdl_wait();
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int lane = threadIdx.x & 31, win = (int)(unit / narrow), c0 = ((int)(unit % narrow) * 32 + lane) * VEC;
  if (owner[win] < 0) return;
  const int mine = perm[win * kWindow + lane % kWindow];
  typename Raw<T, VEC>::type v[kWindow];
#pragma unroll
  for (int r = 0; r < kWindow; ++r) {
    const int64_t p = __shfl_sync(0xffffffffu, mine, r);
    if (c0 < H) v[r] = Raw<T, VEC>::load(dout + p * H + c0);
  }
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
#pragma unroll
  for (int r = 0; r < kWindow; ++r) {
    float x[VEC];
    Raw<T, VEC>::unpack(v[r], x);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] += x[j];
  }
  if (c0 < H) VecIO<float, VEC>::store(partial + (int64_t)win * H + c0, acc);
}

// acc += n rows of `src`, the k-th of them row(k), one after the other; 16 values per lane in flight, 2 rows at least
template <typename T, int VEC, typename Row>
__device__ __forceinline__ void add_rows(float (&acc)[VEC], const T* src, int H, int c0, int n, Row row) {
  constexpr int D = 16 / VEC;
#pragma unroll 1
  for (int k = 0; k < n; k += D) {
    float v[D][VEC];
#pragma unroll
    for (int r = 0; r < D; ++r)
      if (k + r < n) VecIO<T, VEC>::load(src + (int64_t)row(k + r) * H + c0, v[r]);
#pragma unroll
    for (int r = 0; r < D; ++r)
      if (k + r < n) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] += v[r][j];
      }
  }
}

// The rows of the ids with long runs of one block of the order, 32 * VEC columns: a warp to a run, and all eight to a run of more than
// kWarpWindows windows (each some of them, added up in their order).  `runs`: per block their number, then {first place, end, place of
// the id} of each.
constexpr int kWarpWindows = 16;
template <typename T, int VEC>
__device__ __forceinline__ void add_runs(const T* dout, const int* perm, const float* partial, const int4* runs, T* dw, EmbedOrder order, int H,
                                         float scale, int narrow) {
  __shared__ __align__(16) float sums[8][32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x / narrow, c0 = (blockIdx.x % narrow * 32 + lane) * VEC;
  const int4* list = runs + (int64_t)b * (order.slots + 1);
  const int n = list[0].x;
  float acc[VEC];
  const auto add_part = [&](int s, int e, int parts, int part) {  // of the windows, with the ragged ends in the first and last part
    const int w0 = (s + kWindow - 1) / kWindow, w1 = e / kWindow, per = (w1 - w0 + parts - 1) / parts;
    const int u0 = min(w0 + part * per, w1), u1 = min(u0 + per, w1);
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    if (c0 >= H) return;
    if (part == 0) add_rows<T, VEC>(acc, dout, H, c0, w0 * kWindow - s, [&](int r) { return perm[s + r]; });
    add_rows<float, VEC>(acc, partial, H, c0, u1 - u0, [&](int w) { return u0 + w; });
    if (part == parts - 1) add_rows<T, VEC>(acc, dout, H, c0, e - w1 * kWindow, [&](int r) { return perm[w1 * kWindow + r]; });
  };
  const auto write = [&](int place) {
    if (c0 >= H) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] *= scale;
    VecIO<T, VEC>::store(dw + order.id(place) * H + c0, acc);
  };
  for (int base = 0; base < n; base += 32) {
    int4 mine = base + lane < n ? list[1 + base + lane] : make_int4(0, 0, 0, 0);
    const uint32_t big = __ballot_sync(0xffffffffu, mine.y - mine.x > kWarpWindows * kWindow);
#pragma unroll 1
    for (int i = 0; i < min(32, n - base); ++i) {
      const int s = __shfl_sync(0xffffffffu, mine.x, i), e = __shfl_sync(0xffffffffu, mine.y, i), place = __shfl_sync(0xffffffffu, mine.z, i);
      const bool all = big >> i & 1;
      if (!all && i % 8 != warp) continue;
      add_part(s, e, all ? 8 : 1, all ? warp : 0);
      if (all) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[warp][lane * VEC + j] = acc[j];
        __syncthreads();
        if (warp == 0)
#pragma unroll
          for (int w = 1; w < 8; ++w)
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += sums[w][lane * VEC + j];
        __syncthreads();
      }
      if (!all || warp == 0) write(place);
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256, 3) embed_rows_kernel(const T* __restrict__ dout, const int* perm, const int* start, const int4* runs,
                                                            const float* partial, T* __restrict__ dw, EmbedOrder order, int64_t V, int H,
                                                            float scale, int chunks, int64_t units, int narrow, int run_blocks) {
  constexpr int U = unit_vectors<T>(VEC);
  pdl_wait();
  if ((int)blockIdx.x < run_blocks) {  // first: they take longest
    add_runs<T, VEC>(dout, perm, partial, runs, dw, order, H, scale, narrow);
    return;
  }
  const int64_t unit = (int64_t)(blockIdx.x - run_blocks) * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int lane = threadIdx.x & 31;
  const int64_t k0 = unit / chunks * kRowGroup;
  const int c0 = ((int)(unit % chunks) * 32 * U + lane) * VEC;
  const int st = start[k0 + min(lane, kRowGroup)];
  const int first = __shfl_sync(0xffffffffu, st, 0), last = __shfl_sync(0xffffffffu, st, kRowGroup);
  float acc[U][VEC];
  const auto clear = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
  };
  const auto write = [&](int row) {
    const int64_t v = order.id(k0 + row);
    if (v >= V) return;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * 32 * VEC < H) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = acc[u][j] * scale;
        VecIO<T, VEC>::store(dw + v * H + c0 + u * 32 * VEC, o);
      }
  };
  // the places of all rows as one stream, three rows of dout ahead; long runs are passed over
  typename Raw<T, VEC>::type v0[U], v1[U], v2[U];
  int pbase = first, places = first + lane < last ? perm[first + lane] : 0;  // 32 places, one per lane
  int i = first, ahead = first, bound = first, row = -1;  // v2, v1, v0 hold places ahead - 1, - 2, - 3
  uint32_t long_rows = 0;
  clear();
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    while (i == bound) {  // the row ends here (and any empty ones behind it)
      if (row >= 0 && !(long_rows >> row & 1)) {
        write(row);
        clear();
      }
      if (++row == kRowGroup) break;
      bound = __shfl_sync(0xffffffffu, st, row + 1);
      if (bound - i > kLong) {
        long_rows |= 1u << row;
        i = ahead = bound;
      }
    }
    if (row == kRowGroup) break;
#pragma unroll 1
    do {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v0[u] = v1[u];
        v1[u] = v2[u];
      }
      if (ahead < last) {
        if (ahead - pbase >= 32) {
          pbase = ahead;
          places = ahead + lane < last ? perm[ahead + lane] : 0;
        }
        const T* p = dout + (int64_t)__shfl_sync(0xffffffffu, places, ahead - pbase) * H + c0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + u * 32 * VEC < H) v2[u] = Raw<T, VEC>::load(p + u * 32 * VEC);
      }
      ++ahead;
    } while (ahead - 3 < i);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VEC];
      Raw<T, VEC>::unpack(v0[u], x);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] += x[j];
    }
    ++i;
  }
}

// ---- backward of few tokens: one launch, no workspace --------------------------------------------------------
// Up to 2048 positions (us, this against the three launches, text-like ids and in brackets one id for all; V32000): N64 H512 fp32 12
// against 20 (14, 22), N1551 16 against 23 (57, 26: one SM reads all rows), N2048 H2048 bf16 30 against 42 (82, 42); N4096 37 against
// 48 (150, 48) is left to the three.  Two launches and a workspace less are 15 us of the host's time.
// A block owns the ids b, b + blocks, .. and 512 columns of their rows (256 in the scalar form).  Its warps go through an eighth of the
// positions each and list their block's in order; then a warp to a table row adds up its positions, or writes its zeros.  Ids with more
// than kSmallLong positions are added up by all warps, each its eighth of them, and the eight sums in order.
constexpr int kSmallIds = 2048, kSmallSlots = 1024, kSmallLogBlocks = 9, kSmallLong = 16;
__host__ __device__ constexpr bool few_ids(int64_t N, int64_t V) { return N <= kSmallIds && V <= (int64_t)kSmallSlots << kSmallLogBlocks; }

template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_small_kernel(const int64_t* __restrict__ ids, const T* __restrict__ dout, T* __restrict__ dw, int N,
                                                          int V, int H, int64_t padding, float scale, int log_blocks, int share) {
  constexpr int U = unit_vectors<T>(VEC), kRows = 32 / (U * (Raw<T, VEC>::B > 4 ? Raw<T, VEC>::B / 4 : 1));  // rows in flight
  __shared__ uint32_t list[kSmallIds];                // slot << 16 | position, `share` words to a warp
  __shared__ int count[kSmallSlots], found[8], longs[kSmallIds / kSmallLong], nlongs;
  __shared__ __align__(16) float sums[8][32 * VEC * U];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y;
  const int slots = (V - b + (1 << log_blocks) - 1) >> log_blocks, c0 = (blockIdx.x * U * 32 + lane) * VEC;
  for (int k = tid; k < slots; k += 256) count[k] = 0;
  if (tid == 0) nlongs = 0;
  __syncthreads();
  int n = 0;
  uint32_t* mine = list + warp * share;
  for (int i0 = warp * share, end = min(N, i0 + share); i0 < end; i0 += 128) {
    int64_t id[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) id[q] = i0 + q * 32 + lane < end ? __ldg(ids + i0 + q * 32 + lane) : -1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool own = id[q] >= 0 && id[q] < V && id[q] != padding && ((int)id[q] & ((1 << log_blocks) - 1)) == b;
      const uint32_t m = __ballot_sync(0xffffffffu, own);
      if (own) {
        const int k = (int)id[q] >> log_blocks;
        mine[n + __popc(m & ((1u << lane) - 1))] = (uint32_t)k << 16 | (uint32_t)(i0 + q * 32 + lane);
        atomicAdd(&count[k], 1);
      }
      n += __popc(m);
    }
  }
  if (lane == 0) found[warp] = n;
  __syncthreads();

  float acc[U][VEC];
  const auto clear = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
  };
  // adds the rows of the positions that lanes of `m` hold, in the lanes' order
  const auto add = [&](uint32_t m, int position) {
    while (m) {
      typename Raw<T, VEC>::type v[kRows][U];
      int have = 0;
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (m) {
          const T* row = dout + (int64_t)__shfl_sync(0xffffffffu, position, __ffs((int)m) - 1) * H;
          m &= m - 1;
          have = r + 1;
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + u * 32 * VEC < H) v[r][u] = Raw<T, VEC>::load(row + c0 + u * 32 * VEC);
        }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (r < have) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + u * 32 * VEC < H) {
              float x[VEC];
              Raw<T, VEC>::unpack(v[r][u], x);
#pragma unroll
              for (int j = 0; j < VEC; ++j) acc[u][j] += x[j];
            }
        }
    }
  };
  // the positions of slot k in warp w's list
  const auto add_list = [&](int w, int k) {
    for (int i = 0; i < found[w]; i += 32) {
      const uint32_t e = i + lane < found[w] ? list[w * share + i + lane] : 0xffffffffu;
      add(__ballot_sync(0xffffffffu, e >> 16 == (uint32_t)k), (int)(e & 0xffffu));
    }
  };
  for (int k = warp; k < slots; k += 8) {
    const int c = count[k];
    if (c > kSmallLong) {
      if (lane == 0) longs[atomicAdd(&nlongs, 1)] = k;
      continue;
    }
    clear();
    if (c)
      for (int w = 0; w < 8; ++w) add_list(w, k);
    T* out = dw + ((int64_t)k << log_blocks | b) * H;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * 32 * VEC < H) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[u][j] *= scale;
        VecIO<T, VEC>::store(out + c0 + u * 32 * VEC, acc[u]);
      }
  }
  __syncthreads();
  for (int l = 0; l < nlongs; ++l) {
    const int k = longs[l];
    clear();
    add_list(warp, k);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sums[warp][(u * 32 + lane) * VEC + j] = acc[u][j];
    __syncthreads();
    T* out = dw + ((int64_t)k << log_blocks | b) * H;
    for (int i = tid; i < 32 * U * VEC; i += 256) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sums[w][i];
      const int col = blockIdx.x * U * 32 * VEC + i;
      if (col < H) out[col] = from_float<T>(s * scale);
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------------------------------
static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

struct EmbedWs {
  size_t perm, start, partial, owner, runs, total;
};
// as many blocks as nearly fill the GPU, more where a block's counters would not fit its shared memory
static EmbedOrder embed_order(int64_t V) {
  EmbedOrder o{kMinLogBlocks, 0};
  while ((V >> o.log_blocks) >= kMaxSlots) ++o.log_blocks;
  const int64_t slots = (V + (1LL << o.log_blocks) - 1) >> o.log_blocks;
  o.slots = (int)((slots + kRowGroup - 1) / kRowGroup * kRowGroup);
  return o;
}

static EmbedWs embed_ws(int64_t N, int64_t V, int64_t H) {
  EmbedWs L;
  size_t o = 0;
  L.perm = o;    o += up256((size_t)N * 4);
  L.start = o;   o += up256((size_t)(embed_order(V).groups() + 1) * 4);
  L.partial = o; o += N > kLong ? up256((size_t)(N / kWindow) * H * 4) : 0;
  L.owner = o;   o += N > kLong ? up256((size_t)(N / kWindow) * 4) : 0;
  const EmbedOrder order = embed_order(V);
  L.runs = o;    o += N > kLong ? up256((size_t)(order.groups() + (1LL << order.log_blocks)) * sizeof(int4)) : 0;
  L.total = o;
  return L;
}

template <typename T, int VEC>
static int embed_small(const int64_t* ids, const void* dout, void* dw, int64_t N, int64_t V, int H, int64_t padding, float scale,
                       cudaStream_t st) {
  int log_blocks = kSmallLogBlocks;
  while (log_blocks > 0 && (1LL << log_blocks) > V) --log_blocks;
  const int cols = 32 * VEC * unit_vectors<T>(VEC), chunks = (H + cols - 1) / cols, share = (int)((N + 255) / 256) * 32;
  embed_small_kernel<T, VEC><<<dim3((unsigned)chunks, 1u << log_blocks), 256, 0, st>>>(
      ids, static_cast<const T*>(dout), static_cast<T*>(dw), (int)N, (int)V, H, padding, scale, log_blocks, share);
  return launch_status();
}

static int check_embed(int64_t N, int64_t V, int64_t H, int dtype) {
  HAWK_REQUIRE(valid_dtype(dtype), HAWK_ERR_DTYPE);
  HAWK_REQUIRE(N >= 1 && N < (1LL << 31) - kGroupStep && V >= 1 && V < (1LL << 30) && H >= 1 && H < (1 << 24), HAWK_ERR_SHAPE);
  return HAWK_OK;
}

// the widest vectors (in elements) that every row of width H at these addresses starts and ends with
static int common_vec(int H, int es, const void* a, const void* b) {
  for (int bytes = 16; bytes > es; bytes /= 2)
    if ((int64_t)H * es % bytes == 0 && aligned(a, bytes) && aligned(b, bytes)) return bytes / es;
  return 1;
}

template <typename T, int VEC>
static int embed_fwd(const int64_t* ids, const void* w, void* out, int64_t N, int64_t V, int H, float scale, cudaStream_t st) {
  int log_tpr = 0;
  while (log_tpr < 8 && (4 * VEC << log_tpr) < H) ++log_tpr;
  const int rows = 256 >> log_tpr;
  embed_fwd_kernel<T, VEC><<<(unsigned)((N + rows - 1) / rows), 256, 0, st>>>(ids, static_cast<const T*>(w), static_cast<T*>(out), N, V, H,
                                                                              scale, log_tpr);
  return launch_status();
}

template <typename T, int VEC>
static int embed_sums(const void* dout, void* dw, const int* perm, const int* start, float* partial, const int* owner, const int4* runs, EmbedOrder order,
                      int64_t N, int64_t V, int H, float scale, cudaStream_t st) {
  const int cols = 32 * VEC * unit_vectors<T>(VEC), chunks = (H + cols - 1) / cols, narrow = (H + 32 * VEC - 1) / (32 * VEC);
  const int64_t windows = N > kLong ? N / kWindow * narrow : 0, rows = order.groups() / kRowGroup * chunks;
  const int64_t run_blocks = windows ? (int64_t)narrow << order.log_blocks : 0;
  HAWK_REQUIRE((rows + 7) / 8 + run_blocks < (1LL << 31) && (windows + 7) / 8 < (1LL << 31), HAWK_ERR_SHAPE);
  const auto* g = static_cast<const T*>(dout);
  if (windows) {
    const int rc = launch_kernel(embed_window_kernel<T, VEC>, dim3((unsigned)((windows + 7) / 8)), dim3(256), 0, st, true, 1, g, perm, owner,
                                 partial, H, narrow, windows);
    if (rc != HAWK_OK) return rc;
  }
  return launch_kernel(embed_rows_kernel<T, VEC>, dim3((unsigned)((rows + 7) / 8 + run_blocks)), dim3(256), 0, st, true, 1, g, perm, start, runs,
                       partial, static_cast<T*>(dw), order, V, H, scale, chunks, rows, narrow, (int)run_blocks);
}

#define HAWK_BY_VEC(f, dtype, vec, ...)                                                                      \
  ((dtype) == HAWK_F32 ? ((vec) == 4 ? f<float, 4>(__VA_ARGS__) : (vec) == 2 ? f<float, 2>(__VA_ARGS__) : f<float, 1>(__VA_ARGS__))     \
                       : ((vec) == 8 ? f<__nv_bfloat16, 8>(__VA_ARGS__) : (vec) == 4 ? f<__nv_bfloat16, 4>(__VA_ARGS__)               \
                          : (vec) == 2 ? f<__nv_bfloat16, 2>(__VA_ARGS__) : f<__nv_bfloat16, 1>(__VA_ARGS__)))

}  // namespace hawk

using namespace hawk;

extern "C" int hawk_embedding_fwd(const int64_t* ids, const void* weight, void* out, int64_t N, int64_t V, int64_t H, float scale,
                                  int dtype, void* stream) {
  HAWK_REQUIRE(ids && weight && out, HAWK_ERR_NULL);
  const int ok = check_embed(N, V, H, dtype);
  if (ok != HAWK_OK) return ok;
  const int es = (int)dtype_size(dtype);
  HAWK_REQUIRE(aligned(ids, 8) && aligned(weight, es) && aligned(out, es), HAWK_ERR_ALIGN);
  const int vec = common_vec((int)H, es, weight, out);
  return HAWK_BY_VEC(embed_fwd, dtype, vec, ids, weight, out, N, V, (int)H, scale, static_cast<cudaStream_t>(stream));
}

extern "C" size_t hawk_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t H) {
  return N < 1 || V < 1 || H < 1 || few_ids(N, V) ? 0 : embed_ws(N, V, H).total;
}

extern "C" int hawk_embedding_bwd_kernels(int64_t N, int64_t V, int64_t H) {
  return N < 1 || V < 1 || H < 1 ? 0 : few_ids(N, V) ? 1 : N > kLong ? 3 : 2;
}

extern "C" int hawk_embedding_bwd(const int64_t* ids, const void* dout, void* dweight, void* workspace, size_t workspace_bytes, int64_t N,
                                  int64_t V, int64_t H, int64_t padding_idx, float scale, int dtype, void* stream) {
  HAWK_REQUIRE(ids && dout && dweight, HAWK_ERR_NULL);
  const int ok = check_embed(N, V, H, dtype);
  if (ok != HAWK_OK) return ok;
  const int es = (int)dtype_size(dtype);
  HAWK_REQUIRE(aligned(ids, 8) && aligned(dout, es) && aligned(dweight, es) && aligned(workspace, 16), HAWK_ERR_ALIGN);
  const int vec = common_vec((int)H, es, dout, dweight);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few_ids(N, V)) return HAWK_BY_VEC(embed_small, dtype, vec, ids, dout, dweight, N, V, (int)H, padding_idx, scale, st);
  const EmbedWs L = embed_ws(N, V, H);
  HAWK_REQUIRE(workspace && workspace_bytes >= L.total, HAWK_ERR_WORKSPACE);
  auto* ws = static_cast<unsigned char*>(workspace);
  auto* perm = reinterpret_cast<int*>(ws + L.perm);
  auto* start = reinterpret_cast<int*>(ws + L.start);
  auto* owner = reinterpret_cast<int*>(ws + L.owner);
  const int windows = N > kLong ? (int)(N / kWindow) : 0;
  const EmbedOrder order = embed_order(V);
  auto* runs = reinterpret_cast<int4*>(ws + L.runs);
  const int queue = (int)std::min<int64_t>(kMaxQueue, std::max<int64_t>(kMinQueue, N));
  const size_t smem = queue * sizeof(uint2) + (size_t)order.slots * sizeof(int);
  // always the most that any call takes: calls of two threads share this setting
  constexpr int kMostSmem = kMaxQueue * (int)sizeof(uint2) + kMaxSlots * (int)sizeof(int);
  if (cudaFuncSetAttribute(embed_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem) != cudaSuccess) {
    (void)cudaGetLastError();
    return HAWK_ERR_LAUNCH;
  }
  embed_group_kernel<<<1u << order.log_blocks, kGroupThreads, smem, st>>>(ids, N, V, padding_idx, order, perm, start, owner, runs, windows, queue);
  const int rc = launch_status();
  if (rc != HAWK_OK) return rc;
  return HAWK_BY_VEC(embed_sums, dtype, vec, dout, dweight, perm, start, reinterpret_cast<float*>(ws + L.partial),
                     owner, runs, order, N, V, (int)H, scale, st);
}
