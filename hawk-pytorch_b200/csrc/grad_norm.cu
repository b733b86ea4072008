// The 2-norm over all elements of a list of tensors (the gradients of a model) and clipping to it:
//   norm = sqrt(sum x^2),   coef = min(1, max_norm / (norm + 1e-6)),   x <- x * coef.
// Bound by one read of the tensors.  A launch takes up to 1024 of them from a table in its parameters (torch's
// one-launch-per-tensor norms of a 315-tensor model are mostly launches); its blocks walk over the 32 KB chunks of all
// tensors and leave one double each, which a second launch of one block adds up in a fixed order: the result does not
// depend on timing.  The clip itself rides on the optimiser's read of the gradients (hawk_adamw_multi_scaled) or is a pass
// of its own (hawk_scale_multi) that touches nothing where coef is 1.  A clipped AdamW step of 182 M parameters: norm 0.12 ms,
// update 0.75 ms.
//
// Squares: 16 (fp32) or 32 (bf16) of them are added in fp32, as two sums, and these go to a double.  Where that sum is not well inside
// fp32's range (over- or underflow of the squares, infinities, NaN) the same elements are squared in double instead, so the
// norm is right for every list whose norm fp32 can hold.  Zeros go that way, too, as underflow does (the rows of an embedding's gradient
// that no token names): 400 M of them in fp32 253 us, as dense ones take, in bf16 146 of 140.
#include "common.cuh"

namespace hawk {

constexpr int kNormThreads = 256, kNormBlocks = 148 * 8, kNormChunkBytes = 32768, kNormCap = 1024, kNormCapSmall = 128;

template <int CAP>
struct NormTable {
  const void* x[CAP];
  int64_t n[CAP];
  uint32_t first[CAP + 1];  // first chunk of each tensor
  uint8_t bf16[CAP];
  int count;
};

template <int CAP>
__device__ __forceinline__ int norm_find(const NormTable<CAP>& tab, uint32_t chunk) {  // the tensor that holds a chunk
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (chunk >= tab.first[mid]) lo = mid; else hi = mid;
  }
  return lo;
}

// 16 bytes of a tensor as pairs of floats
template <typename T>
struct Vec16;
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float2 pair(uint4 r, int k) {
    return k == 0 ? make_float2(__uint_as_float(r.x), __uint_as_float(r.y)) : make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
  }
};
template <>
struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float2 pair(uint4 r, int k) { return unpack_bf16x2(k == 0 ? r.x : k == 1 ? r.y : k == 2 ? r.z : r.w); }
};

// 16-byte loads per thread in flight, a chunk in one go: 2.7 GB of bf16 in 412 us (6.57 TB/s, the rate of a copy); with 4 loads and 8
// blocks of 256 per SM 451; loads and their squares one after the other 500
constexpr int kNormAhead = 8;

// the sum of the squares of a thread's vectors
template <typename T>
__device__ __forceinline__ double sum_squares(const uint4 (&r)[kNormAhead]) {
  double total = 0.0;
#pragma unroll
  for (int h = 0; h < kNormAhead; h += kNormAhead / 2) {
    float2 s2 = f2(0.f);
#pragma unroll
    for (int q = h; q < h + kNormAhead / 2; ++q)
#pragma unroll
      for (int k = 0; k < Vec16<T>::N / 2; ++k) s2 = fma2(Vec16<T>::pair(r[q], k), Vec16<T>::pair(r[q], k), s2);
    const float s = s2.x + s2.y;
    if (s > 1e-28f && s < 1e37f) {
      total += (double)s;
    } else {
#pragma unroll
      for (int q = h; q < h + kNormAhead / 2; ++q)
#pragma unroll
        for (int k = 0; k < Vec16<T>::N / 2; ++k) {
          const float2 v = Vec16<T>::pair(r[q], k);
          total = fma((double)v.x, (double)v.x, fma((double)v.y, (double)v.y, total));
        }
    }
  }
  return total;
}

// elements before the first 16-byte boundary of a chunk (all of a tensor's chunks start as far from one): gradients that are views
// of one flat buffer lie anywhere.  Norm / product of 200 M bf16 at an odd address 63 / 152 us (element by element 90 / 398), at an
// even one 62 / 136
template <typename T>
__device__ __forceinline__ int head_elements(const T* x, int n) {
  return min(n, (int)((0u - (uint32_t)reinterpret_cast<uintptr_t>(x)) & 15u) / (int)sizeof(T));
}

// the squares of up to kNormChunkBytes of one tensor, this thread's share
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* x, int n) {
  constexpr int N = Vec16<T>::N;
  static_assert(kNormChunkBytes == 16 * kNormThreads * kNormAhead, "a chunk is one batch of loads");
  const int head = head_elements(x, n), nvec = (n - head) / N, tail = head + nvec * N;
  const uint4* p = reinterpret_cast<const uint4*>(x + head);
  uint4 r[kNormAhead];
#pragma unroll
  for (int q = 0; q < kNormAhead; ++q) {
    const int i = threadIdx.x + q * kNormThreads;
    r[q] = i < nvec ? __ldg(p + i) : make_uint4(0u, 0u, 0u, 0u);
  }
  // fewer elements outside the vectors than threads
  const int i = threadIdx.x;
  const double v = i < head + n - tail ? (double)to_float(x[i < head ? i : tail + i - head]) : 0.0;
  return fma(v, v, sum_squares<T>(r));
}

__device__ __forceinline__ double block_sum(double v, double* red) {  // the sum in thread 0
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < kNormThreads / 32; ++w) s += red[w];
  return s;
}

template <int CAP>
__global__ void __launch_bounds__(kNormThreads, 4) norm_partial_kernel(const __grid_constant__ NormTable<CAP> tab, double* partial) {
  __shared__ double red[kNormThreads / 32];
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < tab.first[tab.count]; c += gridDim.x) {
    const int t = norm_find(tab, c);
    const bool bf16 = tab.bf16[t];
    const int per = kNormChunkBytes / (bf16 ? 2 : 4);
    const int64_t at = (int64_t)(c - tab.first[t]) * per;
    const int n = (int)min((int64_t)per, tab.n[t] - at);
    acc += bf16 ? chunk_squares(static_cast<const __nv_bfloat16*>(tab.x[t]) + at, n)
                : chunk_squares(static_cast<const float*>(tab.x[t]) + at, n);
  }
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(kNormThreads) norm_final_kernel(const double* partial, int n, float max_norm, float* out) {
  __shared__ double red[kNormThreads / 32];
  pdl_wait();
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kNormThreads) s += *reinterpret_cast<const volatile double*>(partial + i);
  s = block_sum(s, red);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s), coef = (double)max_norm / (norm + 1e-6);
    out[0] = (float)norm;
    out[1] = coef >= 1.0 ? 1.f : (float)coef;  // NaN stays NaN
  }
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* x, int n, float k) {
  constexpr int VPT = 16 / sizeof(T);
  const int head = head_elements(x, n), nvec = (n - head) / VPT, tail = head + nvec * VPT;
#pragma unroll 4
  for (int i = threadIdx.x; i < nvec; i += kNormThreads) {
    float v[VPT];
    VecIO<T, VPT>::load(x + head + (int64_t)i * VPT, v);
#pragma unroll
    for (int j = 0; j < VPT; ++j) v[j] *= k;
    VecIO<T, VPT>::store(x + head + (int64_t)i * VPT, v);
  }
  const int i = threadIdx.x, e = i < head ? i : tail + i - head;  // the elements outside the vectors, fewer than threads
  if (i < head + n - tail) x[e] = from_float<T>(to_float(x[e]) * k);
}

template <int CAP>
__global__ void __launch_bounds__(kNormThreads) scale_multi_kernel(const __grid_constant__ NormTable<CAP> tab, const float* scale) {
  const float k = *scale;
  if (k == 1.f) return;
  for (uint32_t c = blockIdx.x; c < tab.first[tab.count]; c += gridDim.x) {
    const int t = norm_find(tab, c);
    const bool bf16 = tab.bf16[t];
    const int per = kNormChunkBytes / (bf16 ? 2 : 4);
    const int64_t at = (int64_t)(c - tab.first[t]) * per;
    const int n = (int)min((int64_t)per, tab.n[t] - at);
    if (bf16) chunk_scale(static_cast<__nv_bfloat16*>(const_cast<void*>(tab.x[t])) + at, n, k);
    else chunk_scale(static_cast<float*>(const_cast<void*>(tab.x[t])) + at, n, k);
  }
}

static int check_norm(const hawk_norm_tensor* tensors, int count) {
  HAWK_REQUIRE(tensors, HAWK_ERR_NULL);
  HAWK_REQUIRE(count >= 1 && count <= (1 << 24), HAWK_ERR_SHAPE);
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    HAWK_REQUIRE(valid_dtype((int)tensors[i].dtype), HAWK_ERR_DTYPE);
    HAWK_REQUIRE(tensors[i].x, HAWK_ERR_NULL);
    HAWK_REQUIRE(tensors[i].n >= 1 && tensors[i].n <= (1LL << 40), HAWK_ERR_SHAPE);
    HAWK_REQUIRE(aligned(tensors[i].x, dtype_size((int)tensors[i].dtype)), HAWK_ERR_ALIGN);
    chunks += tensors[i].n * (int64_t)dtype_size((int)tensors[i].dtype) / kNormChunkBytes + 1;
    HAWK_REQUIRE(chunks < (1LL << 31), HAWK_ERR_SHAPE);  // 64 TB: a launch's chunks fit 32 bits
  }
  return HAWK_OK;
}

// fills a table from tensors[i0..]; the number of tensors taken, and of chunks
template <int CAP>
static int fill_table(NormTable<CAP>& tab, const hawk_norm_tensor* tensors, int count, int i0, uint32_t& chunks) {
  int k = 0;
  chunks = 0;
  for (; k < CAP && i0 + k < count; ++k) {
    const hawk_norm_tensor& t = tensors[i0 + k];
    const int64_t per = kNormChunkBytes / (int64_t)dtype_size((int)t.dtype);
    tab.x[k] = t.x;
    tab.n[k] = t.n;
    tab.bf16[k] = t.dtype == HAWK_BF16;
    tab.first[k] = chunks;
    chunks += (uint32_t)((t.n + per - 1) / per);
  }
  tab.first[k] = chunks;
  tab.count = k;
  return k;
}

// f(table, blocks) for as many launches as the list takes
template <typename F>
static int for_tables(const hawk_norm_tensor* tensors, int count, F f) {
  for (int i0 = 0; i0 < count;) {
    uint32_t chunks;
    int k;
    if (count - i0 <= kNormCapSmall) {  // 2.7 KB of parameters instead of 21
      NormTable<kNormCapSmall> tab;
      k = fill_table(tab, tensors, count, i0, chunks);
      f(tab, (int)(chunks < (uint32_t)kNormBlocks ? chunks : kNormBlocks));
    } else {
      NormTable<kNormCap> tab;
      k = fill_table(tab, tensors, count, i0, chunks);
      f(tab, (int)(chunks < (uint32_t)kNormBlocks ? chunks : kNormBlocks));
    }
    const int rc = launch_status();
    if (rc != HAWK_OK) return rc;
    i0 += k;
  }
  return HAWK_OK;
}

static int table_launches(int count) { return (count + kNormCap - 1) / kNormCap; }

}  // namespace hawk

using namespace hawk;

extern "C" size_t hawk_grad_norm_workspace_bytes(int count) {
  return count < 1 ? 0 : (size_t)table_launches(count) * kNormBlocks * sizeof(double);
}

extern "C" int hawk_grad_norm(const hawk_norm_tensor* tensors, int count, float max_norm, float* out, void* workspace,
                              size_t workspace_bytes, void* stream) {
  HAWK_REQUIRE(out, HAWK_ERR_NULL);
  const int ok = check_norm(tensors, count);
  if (ok != HAWK_OK) return ok;
  HAWK_REQUIRE(max_norm >= 0.f, HAWK_ERR_SHAPE);
  HAWK_REQUIRE(workspace && workspace_bytes >= hawk_grad_norm_workspace_bytes(count), HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(workspace, 8) && aligned(out, 4), HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* partial = static_cast<double*>(workspace);
  int blocks = 0;
  const int rc = for_tables(tensors, count, [&](const auto& tab, int grid) {
    norm_partial_kernel<<<grid, kNormThreads, 0, st>>>(tab, partial + blocks);
    blocks += grid;
  });
  if (rc != HAWK_OK) return rc;
  return launch_kernel(norm_final_kernel, dim3(1), dim3(kNormThreads), 0, st, true, 1, partial, blocks, max_norm, out);
}

extern "C" int hawk_scale_multi(const hawk_norm_tensor* tensors, int count, const float* scale, void* stream) {
  HAWK_REQUIRE(scale, HAWK_ERR_NULL);
  const int ok = check_norm(tensors, count);
  if (ok != HAWK_OK) return ok;
  HAWK_REQUIRE(aligned(scale, 4), HAWK_ERR_ALIGN);
  return for_tables(tensors, count, [&](const auto& tab, int grid) {
    scale_multi_kernel<<<grid, kNormThreads, 0, static_cast<cudaStream_t>(stream)>>>(tab, scale);
  });
}
