// Embedding of token ids, out[i] = scale * W[ids[i]], and the table's gradient
//   dW[v] = scale * sum over { i : ids[i] = v } of dout[i],
// summed in fp32 in the order of the positions and rounded once: the same bits on every run (adding rows with atomics is
// neither ordered nor, in bf16, exact).  Both are bound by memory: the forward by N rows read and written, the backward by
// N rows read and V rows written, the rows that no token names among them.
//
// Backward, three launches:
//   1. group   positions in the order of their ids (a stable counting sort).  A block owns a slice of the vocabulary and
//              reads all ids (they come from L2: 148 blocks x 8 B, against rows of kilobytes): it counts those below its slice,
//              which gives its place in the result without a word from the other blocks, and queues its own in shared memory
//              in their order; one warp then hands out the places, 32 at a time (match.any ranks equal ids).
//   2. windows sums of 32 consecutive sorted positions, only for windows that lie inside the run of an id with more than 64
//              of them: the most frequent token of a text is 5 to 10 % of it, and one warp would walk its rows alone.
//   3. rows    a warp per table row and 512 columns (fp32: 4 16-byte loads in flight per position, 4 positions at a time): its
//              few positions, or for the long runs the ragged ends and the windows' sums; zeros where there are none.
#include <algorithm>

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
    float v[4][VEC];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + u * tpr * VEC < H) VecIO<T, VEC>::load(src + c0 + u * tpr * VEC, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (c0 + u * tpr * VEC < H) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[u][j] = known ? v[u][j] * scale : __int_as_float(0x7fc00000);
        VecIO<T, VEC>::store(dst + c0 + u * tpr * VEC, v[u]);
      }
  }
}

// ---- backward 1: positions grouped by id ---------------------------------------------------------------------
constexpr int kGroupThreads = 1024, kIdsPerThread = 8, kGroupStep = kGroupThreads * kIdsPerThread;
constexpr int kQueue = kGroupStep;  // one step's ids always fit
constexpr int kMaxSlice = 4096;

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

// One step's ids of this thread (its 8 positions are consecutive, so the threads are in the order of the positions): which of
// them are in [lo, hi), and how many valid ones lie below.
struct StepIds {
  int64_t id[kIdsPerThread];
  uint32_t mine;
};
__device__ __forceinline__ void load_step(const int64_t* ids, int64_t i0, int64_t N, int64_t lo, int64_t hi, int64_t padding, StepIds& s,
                                          int& below) {
  if (i0 + kIdsPerThread <= N && aligned16(ids)) {  // i0 is a multiple of 8
#pragma unroll
    for (int q = 0; q < kIdsPerThread / 2; ++q) {
      const longlong2 t = __ldg(reinterpret_cast<const longlong2*>(ids + i0) + q);
      s.id[2 * q] = t.x;
      s.id[2 * q + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int q = 0; q < kIdsPerThread; ++q) s.id[q] = i0 + q < N ? __ldg(ids + i0 + q) : -1;
  }
  s.mine = 0;
#pragma unroll
  for (int q = 0; q < kIdsPerThread; ++q) {
    const int64_t id = s.id[q];
    if (id < 0 || id == padding) continue;
    below += id < lo;
    if (id >= lo && id < hi) s.mine |= 1u << q;
  }
}

__device__ __forceinline__ void place(const uint2* queue, int n, int* cursor, int* perm) {  // one warp
  const int lane = threadIdx.x & 31;
  for (int k = 0; k < n; k += 32) {
    const bool have = k + lane < n;
    const uint32_t active = __ballot_sync(0xffffffffu, have);
    if (have) {
      const uint2 q = queue[k + lane];
      const uint32_t peers = __match_any_sync(active, q.x);
      const int rank = __popc(peers & ((1u << lane) - 1)), at = cursor[q.x];
      perm[at + rank] = (int)q.y;
      __syncwarp(active);
      if (rank == 0) cursor[q.x] = at + __popc(peers);
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kGroupThreads) embed_group_kernel(const int64_t* __restrict__ ids, int64_t N, int64_t V, int64_t padding,
                                                                    int slice, int* __restrict__ perm, int* __restrict__ start) {
  extern __shared__ uint2 queue[];                       // [kQueue]
  int* count = reinterpret_cast<int*>(queue + kQueue);   // [slice], the cursors later
  __shared__ int warp_sums[2][32];
  const int tid = threadIdx.x;
  const int64_t lo = (int64_t)blockIdx.x * slice, hi = lo + slice < V ? lo + slice : V;
  for (int j = tid; j < slice; j += kGroupThreads) count[j] = 0;
  __syncthreads();
  int below = 0, total = 0, all;
  StepIds s;
  int step = 0;
  for (int64_t base = 0; base < N; base += kGroupStep, step ^= 1) {  // the scans take turns with their shared words
    const int64_t i0 = base + tid * kIdsPerThread;
    load_step(ids, i0, N, lo, hi, padding, s, below);
    int at = total + block_scan(__popc(s.mine), warp_sums[step], all);
#pragma unroll
    for (int q = 0; q < kIdsPerThread; ++q)
      if (s.mine >> q & 1) {
        const int j = (int)(s.id[q] - lo);
        atomicAdd(&count[j], 1);
        if (at < kQueue) queue[at] = make_uint2((uint32_t)j, (uint32_t)(i0 + q));
        ++at;
      }
    total += all;
  }
  __syncthreads();
  int ahead;
  block_scan(below, warp_sums[0], ahead);
  __syncthreads();
  // counts -> first places
  constexpr int kPer = kMaxSlice / kGroupThreads;
  int c[kPer], sum = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int j = tid * kPer + q;
    c[q] = j < slice ? count[j] : 0;
    sum += c[q];
  }
  int at = ahead + block_scan(sum, warp_sums[1], all);
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int j = tid * kPer + q;
    if (j < slice) {
      count[j] = at;
      if (lo + j < V) start[lo + j] = at;
    }
    at += c[q];
  }
  if (hi == V && tid == 0) start[V] = ahead + total;
  __syncthreads();
  if (total <= kQueue) {
    if (tid < 32) place(queue, total, count, perm);
    return;
  }
  for (int64_t base = 0; base < N; base += kGroupStep, step ^= 1) {  // more than the queue holds: read the ids again
    const int64_t i0 = base + tid * kIdsPerThread;
    load_step(ids, i0, N, lo, hi, padding, s, below);
    int to = block_scan(__popc(s.mine), warp_sums[step], all);
#pragma unroll
    for (int q = 0; q < kIdsPerThread; ++q)
      if (s.mine >> q & 1) queue[to++] = make_uint2((uint32_t)(s.id[q] - lo), (uint32_t)(i0 + q));
    __syncthreads();
    if (tid < 32) place(queue, all, count, perm);
    __syncthreads();
  }
}

// ---- backward 2 and 3: sums --------------------------------------------------------------------------------
constexpr int kWindow = 32, kLong = 2 * kWindow;  // a run of more than kLong positions holds a whole window

template <typename T>
__host__ __device__ constexpr int unit_vectors(int vec) { return vec == 1 ? 8 : 512 / (32 * vec); }  // vectors per lane: 512 columns (256 in the scalar form)

// acc += the rows of `src` at the given places, one after the other; four rows in flight
template <typename T, int VEC, int U, typename Row>
__device__ __forceinline__ void add_rows(float (&acc)[U][VEC], const T* src, int H, int c0, int s, int e, Row row) {
  int i = s;
  for (; i + 4 <= e; i += 4) {
    float v[4][U][VEC];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const T* p = src + (int64_t)row(i + r) * H + c0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * 32 * VEC < H) VecIO<T, VEC>::load(p + u * 32 * VEC, v[r][u]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * 32 * VEC < H)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[u][j] += v[r][u][j];
  }
  for (; i < e; ++i) {
    const T* p = src + (int64_t)row(i) * H + c0;
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * 32 * VEC < H) VecIO<T, VEC>::load(p + u * 32 * VEC, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * 32 * VEC < H)
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[u][j] += v[u][j];
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_window_kernel(const int64_t* __restrict__ ids, const T* __restrict__ dout,
                                                           const int* __restrict__ perm, const int* __restrict__ start,
                                                           float* __restrict__ partial, int64_t V, int H, int chunks, int64_t units) {
  constexpr int U = unit_vectors<T>(VEC);
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int win = (int)(unit / chunks), c0 = ((int)(unit % chunks) * 32 * U + (threadIdx.x & 31)) * VEC;
  const int s = win * kWindow;
  if (s + kWindow > start[V]) return;
  const int64_t id = ids[perm[s]];
  if (ids[perm[s + kWindow - 1]] != id || start[id + 1] - start[id] <= kLong) return;
  float acc[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
  add_rows<T, VEC, U>(acc, dout, H, c0, s, s + kWindow, [&](int i) { return perm[i]; });
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + u * 32 * VEC < H)
#pragma unroll
      for (int j = 0; j < VEC; ++j) partial[(int64_t)win * H + c0 + u * 32 * VEC + j] = acc[u][j];
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_rows_kernel(const T* __restrict__ dout, const int* __restrict__ perm,
                                                         const int* __restrict__ start, const float* __restrict__ partial,
                                                         T* __restrict__ dw, int H, float scale, int chunks, int64_t units) {
  constexpr int U = unit_vectors<T>(VEC);
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int64_t v = unit / chunks;
  const int c0 = ((int)(unit % chunks) * 32 * U + (threadIdx.x & 31)) * VEC;
  const int s = start[v], e = start[v + 1];
  float acc[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[u][j] = 0.f;
  const auto at = [&](int i) { return perm[i]; };
  if (e - s <= kLong) {
    add_rows<T, VEC, U>(acc, dout, H, c0, s, e, at);
  } else {
    const int w0 = (s + kWindow - 1) / kWindow, w1 = e / kWindow;
    add_rows<T, VEC, U>(acc, dout, H, c0, s, w0 * kWindow, at);
    for (int w = w0; w < w1; ++w)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * 32 * VEC < H)
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[u][j] += partial[(int64_t)w * H + c0 + u * 32 * VEC + j];
    add_rows<T, VEC, U>(acc, dout, H, c0, w1 * kWindow, e, at);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (c0 + u * 32 * VEC < H) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[u][j] *= scale;
      VecIO<T, VEC>::store(dw + v * H + c0 + u * 32 * VEC, acc[u]);
    }
}

// ---- host --------------------------------------------------------------------------------------------------
static size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

struct EmbedWs {
  size_t perm, start, partial, total;
};
static EmbedWs embed_ws(int64_t N, int64_t V, int64_t H) {
  EmbedWs L;
  size_t o = 0;
  L.perm = o;    o += up256((size_t)N * 4);
  L.start = o;   o += up256((size_t)(V + 1) * 4);
  L.partial = o; o += N > kLong ? up256((size_t)(N / kWindow) * H * 4) : 0;
  L.total = o;
  return L;
}

static int check_embed(int64_t N, int64_t V, int64_t H, int dtype) {
  HAWK_REQUIRE(valid_dtype(dtype), HAWK_ERR_DTYPE);
  HAWK_REQUIRE(N >= 1 && N < (1LL << 31) - kGroupStep && V >= 1 && V < (1LL << 31) - kMaxSlice && H >= 1 && H < (1 << 24), HAWK_ERR_SHAPE);
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
static int embed_sums(const int64_t* ids, const void* dout, void* dw, const int* perm, const int* start, float* partial, int64_t N,
                      int64_t V, int H, float scale, cudaStream_t st) {
  const int cols = 32 * VEC * unit_vectors<T>(VEC), chunks = (H + cols - 1) / cols;
  const int64_t windows = N > kLong ? N / kWindow * chunks : 0, rows = V * chunks;
  HAWK_REQUIRE((rows + 7) / 8 < (1LL << 31) && (windows + 7) / 8 < (1LL << 31), HAWK_ERR_SHAPE);
  if (windows) {
    embed_window_kernel<T, VEC><<<(unsigned)((windows + 7) / 8), 256, 0, st>>>(ids, static_cast<const T*>(dout), perm, start, partial, V, H,
                                                                               chunks, windows);
    const int rc = launch_status();
    if (rc != HAWK_OK) return rc;
  }
  embed_rows_kernel<T, VEC><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(static_cast<const T*>(dout), perm, start, partial,
                                                                        static_cast<T*>(dw), H, scale, chunks, rows);
  return launch_status();
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
  return N < 1 || V < 1 || H < 1 ? 0 : embed_ws(N, V, H).total;
}

extern "C" int hawk_embedding_bwd(const int64_t* ids, const void* dout, void* dweight, void* workspace, size_t workspace_bytes, int64_t N,
                                  int64_t V, int64_t H, int64_t padding_idx, float scale, int dtype, void* stream) {
  HAWK_REQUIRE(ids && dout && dweight, HAWK_ERR_NULL);
  const int ok = check_embed(N, V, H, dtype);
  if (ok != HAWK_OK) return ok;
  const EmbedWs L = embed_ws(N, V, H);
  HAWK_REQUIRE(workspace && workspace_bytes >= L.total, HAWK_ERR_WORKSPACE);
  const int es = (int)dtype_size(dtype);
  HAWK_REQUIRE(aligned(ids, 8) && aligned(dout, es) && aligned(dweight, es) && aligned(workspace, 16), HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  auto* perm = reinterpret_cast<int*>(ws + L.perm);
  auto* start = reinterpret_cast<int*>(ws + L.start);
  // a slice of the vocabulary for every SM; no narrower than a warp's worth
  const int slice = (int)std::min<int64_t>(kMaxSlice, std::max<int64_t>(32, (V + 147) / 148));
  const size_t smem = kQueue * sizeof(uint2) + (size_t)slice * sizeof(int);
  if (cudaFuncSetAttribute(embed_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    (void)cudaGetLastError();
    return HAWK_ERR_LAUNCH;
  }
  embed_group_kernel<<<(unsigned)((V + slice - 1) / slice), kGroupThreads, smem, st>>>(ids, N, V, padding_idx, slice, perm, start);
  const int rc = launch_status();
  if (rc != HAWK_OK) return rc;
  const int vec = common_vec((int)H, es, dout, dweight);
  return HAWK_BY_VEC(embed_sums, dtype, vec, ids, dout, dweight, perm, start, reinterpret_cast<float*>(ws + L.partial), N, V, (int)H, scale,
                     st);
}
