// Fused linear + cross-entropy: the loss in one call, d act and d weight in a second, replacing
// hawk/fused_cross_entropy.py:11-73 (2048-row chunks, three cuBLAS GEMMs and ~8 passes over
// [chunk, V] fp32 temporaries per chunk).
//
// Loss, all on the caller's stream:
//   1. cast           : fp32 weight [V,H] and act [N,H] -> bf16 copies (bf16 inputs are used in place).
//   2. GEMM + softmax epilogue (tcgen05): logits tile = act @ weight^T accumulated in TMEM; the
//      epilogue rounds it to bf16 (as F.linear does under autocast, fused_cross_entropy.py:28),
//      stores it once, and reduces each row's tile to (max, sum exp) online, 32 columns at a time;
//      it also picks out the label's logit.  No fp32 [N,V] tensor is ever written.
//   3. row reduce     : tile statistics -> log-sum-exp per row, loss = mean(lse - correct) (:37-44,59-64).
//   4. dprobs         : logits -> (softmax - onehot) / N in bf16, in place (:47-52); skipped when no gradient
//                       is wanted.
// Gradients: two GEMMs with a plain epilogue that can multiply by a gradient of the loss,
//      d act = dprobs @ weight (:56), d weight = dprobs^T @ act (:55).  Neither needs a transposed copy: an operand
//      whose contraction index is the row index of its tensor (weight in d act; dprobs and act in d weight) is read
//      as an MN-major tile straight from the row-major tensor.  The first call leaves dprobs and the bf16 operands
//      behind for it.
// The GEMM itself is head_gemm.cuh.
#include <algorithm>

#include "head_gemm.cuh"

namespace hawk {

// ---------------------------------------------------------------------------------------------
// small kernels around the GEMMs
// ---------------------------------------------------------------------------------------------
// stats [groups, N] -> lse [N]; per-block partial sums of (lse - correct) -> partial [gridDim.x].  A block is 32 rows
// x 8 slices of the column groups (a thread per row walked 125 groups alone: 31 us at N = 32760, 16 warps in flight
// per SM at most; 28 us with 8 slices, 32 MB of statistics).
__global__ void __launch_bounds__(256)
ce_row_reduce_kernel(const float2* __restrict__ stats, const float* __restrict__ correct, float* __restrict__ lse,
                     float* __restrict__ partial, int N, int groups) {
  __shared__ float2 sl[8][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  if (row < N)
    for (int t = slice; t < groups; t += 8) {
      const float2 st = stats[(long long)t * N + row];
      const float nm = fmaxf(m, st.x);
      s = s * expf(m - nm) + st.y * expf(st.x - nm);
      m = nm;
    }
  sl[slice][lane] = make_float2(m, s);
  __syncthreads();
  if (slice == 0) {
    float contrib = 0.f;
    if (row < N) {
      float mm = -INFINITY;
#pragma unroll
      for (int k = 0; k < 8; ++k) mm = fmaxf(mm, sl[k][lane].x);
      float ss = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) ss += sl[k][lane].y * expf(sl[k][lane].x - mm);  // an unused slice: 0 * exp(-inf)
      const float l = mm + logf(ss);
      lse[row] = l;
      contrib = l - correct[row];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) contrib += __shfl_xor_sync(0xffffffffu, contrib, o);
    if (lane == 0) partial[blockIdx.x] = contrib;
  }
}

__global__ void __launch_bounds__(256)
ce_loss_final_kernel(const float* __restrict__ partial, int n, float inv_n, float* __restrict__ loss,
                     const int* __restrict__ status) {
  __shared__ float red[256];
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) s += partial[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
    __syncthreads();
  }
  // a GEMM that abandoned a wait (this call or an earlier one nobody has looked at) shows in the loss itself
  if (threadIdx.x == 0) *loss = *status != 0 ? __int_as_float(0x7fc00000) : red[0] * inv_n;
}

// logits [N, ldl] bf16 -> dprobs = (exp(logit - lse) - onehot) / N, in place.  One CTA per row, 16 bytes
// per thread per step.
__global__ void __launch_bounds__(256)
ce_dprobs_kernel(__nv_bfloat16* __restrict__ logits, long long ldl, const float* __restrict__ lse,
                 const long long* __restrict__ labels, int N, int V, float inv_n) {
  const int r = blockIdx.x;
  if (r >= N) return;
  __nv_bfloat16* row = logits + (long long)r * ldl;
  const float l = lse[r];
  const long long label = labels[r];
  const int nvec = (ldl % 8 == 0) ? V / 8 : 0;
  for (int jv = threadIdx.x; jv < nvec; jv += blockDim.x) {
    const uint4 raw = *reinterpret_cast<const uint4*>(row + jv * 8);
    const int lab = (int)(label - (long long)jv * 8);  // 0..7 when the label is in this vector
    const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t out[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 f = unpack_bf16x2(in[q]);
      float p0 = __expf(f.x - l), p1 = __expf(f.y - l);
      if (lab == 2 * q) p0 -= 1.f;
      if (lab == 2 * q + 1) p1 -= 1.f;
      out[q] = pack_bf16x2(p0 * inv_n, p1 * inv_n);
    }
    *reinterpret_cast<uint4*>(row + jv * 8) = make_uint4(out[0], out[1], out[2], out[3]);
  }
  for (int c = nvec * 8 + threadIdx.x; c < V; c += blockDim.x) {
    float p = __expf(__bfloat162float(row[c]) - l);
    if ((long long)c == label) p -= 1.f;
    row[c] = __float2bfloat16(p * inv_n);
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// What the forward leaves for the backward: dprobs and the bf16 copies of fp32 operands (offsets 256-byte aligned)
struct CeSaved {
  size_t wb, ab, logits, total;
  long long ldV;
};
static CeSaved ce_saved(long long N, long long H, long long V, int w_dtype, int a_dtype) {
  CeSaved L;
  L.ldV = (V + 7) & ~7LL;
  size_t o = 0;
  L.wb = o;      o += w_dtype == HAWK_F32 ? up256((size_t)V * H * 2) : 0;
  L.ab = o;      o += a_dtype == HAWK_F32 ? up256((size_t)N * H * 2) : 0;
  L.logits = o;  o += up256((size_t)N * L.ldV * 2);
  L.total = o;
  return L;
}
// Scratch of one call
struct CeScratch {
  size_t stats, correct, lse, partial, total;
  int groups, n_blocks;
};
static CeScratch ce_fwd_scratch(long long N, long long V) {
  CeScratch L;
  L.groups = (int)((V + EPI_COLS - 1) / EPI_COLS);
  L.n_blocks = (int)((N + 31) / 32);
  size_t o = 0;
  L.stats = o;   o += up256((size_t)L.groups * N * sizeof(float2));
  L.correct = o; o += up256((size_t)N * 4);
  L.lse = o;     o += up256((size_t)N * 4);
  L.partial = o; o += up256((size_t)L.n_blocks * 4);
  L.total = o;
  return L;
}
static size_t ce_bwd_scratch(long long N, long long H, long long V) {  // the two GEMMs run one after the other
  const int sa = plan_grad(N, H, V).splits, sw = plan_grad(V, H, N).splits;
  return std::max(sa > 1 ? up256((size_t)sa * N * H * 4) : 0, sw > 1 ? up256((size_t)sw * V * H * 4) : 0);
}

static int check_ce(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype) {
  HAWK_REQUIRE(valid_dtype(w_dtype) && valid_dtype(a_dtype), HAWK_ERR_DTYPE);
  HAWK_REQUIRE(N >= 1 && V >= 2 && H >= 8 && H % 8 == 0, HAWK_ERR_SHAPE);
  HAWK_REQUIRE(N < (1LL << 31) - 512 && V < (1LL << 31) - 512 && H < (1LL << 31) - 512, HAWK_ERR_SHAPE);
  return HAWK_OK;
}

}  // namespace hawk

using namespace hawk;

extern "C" size_t hawk_linear_ce_saved_bytes(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype) {
  if (N < 1 || H < 1 || V < 1) return 0;
  return ce_saved(N, H, V, w_dtype, a_dtype).total;
}

extern "C" size_t hawk_linear_ce_scratch_bytes(int64_t N, int64_t H, int64_t V) {
  if (N < 1 || H < 1 || V < 1) return 0;
  return std::max(ce_fwd_scratch(N, V).total, ce_bwd_scratch(N, H, V));
}

extern "C" size_t hawk_linear_ce_workspace_bytes(int64_t N, int64_t H, int64_t V) {
  if (N < 1 || H < 1 || V < 1) return 0;
  return ce_saved(N, H, V, HAWK_F32, HAWK_F32).total + hawk_linear_ce_scratch_bytes(N, H, V);
}

// one cast per fp32 operand, the logits GEMM and the two reductions, the pass that makes dprobs; then a GEMM and, where K is
// split, a sum for each gradient, and the look at the status word
extern "C" int hawk_linear_ce_kernels(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int want_dw, int want_da) {
  if (N < 1 || H < 1 || V < 1) return 0;
  int n = (w_dtype == HAWK_F32) + (a_dtype == HAWK_F32) + 3;
  if (want_dw || want_da) n += 2;
  if (want_dw) n += plan_grad(V, H, N).splits > 1 ? 2 : 1;
  if (want_da) n += plan_grad(N, H, V).splits > 1 ? 2 : 1;
  return n;
}

extern "C" int hawk_linear_ce_fwd(const void* weight, const void* act, const int64_t* labels, float* loss, void* saved,
                                  size_t saved_bytes, void* scratch, size_t scratch_bytes, int64_t N, int64_t H, int64_t V,
                                  int w_dtype, int a_dtype, int want_grad, int* status, void* stream) {
  HAWK_REQUIRE(weight && act && labels && loss && status, HAWK_ERR_NULL);
  int rc = check_ce(N, H, V, w_dtype, a_dtype);
  if (rc != HAWK_OK) return rc;
  const CeSaved S = ce_saved(N, H, V, w_dtype, a_dtype);
  const CeScratch L = ce_fwd_scratch(N, V);
  HAWK_REQUIRE(saved && saved_bytes >= S.total && scratch && scratch_bytes >= L.total, HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(saved, 256) && aligned(scratch, 256) && aligned(weight, 16) && aligned(act, 16), HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* sv = static_cast<unsigned char*>(saved);
  auto* sc = static_cast<unsigned char*>(scratch);
  auto* logits = reinterpret_cast<__nv_bfloat16*>(sv + S.logits);
  auto* stats = reinterpret_cast<float2*>(sc + L.stats);
  auto* correct = reinterpret_cast<float*>(sc + L.correct);
  auto* lse = reinterpret_cast<float*>(sc + L.lse);
  auto* partial = reinterpret_cast<float*>(sc + L.partial);

  // 1. operands in bf16 (row-major, as given: no transposes)
  const __nv_bfloat16* wb = static_cast<const __nv_bfloat16*>(weight);
  const __nv_bfloat16* ab = static_cast<const __nv_bfloat16*>(act);
  if (w_dtype == HAWK_F32) {
    auto* wcast = reinterpret_cast<__nv_bfloat16*>(sv + S.wb);
    rc = hawk_cast_f32_bf16(static_cast<const float*>(weight), wcast, V * H, stream);
    if (rc != HAWK_OK) return rc;
    wb = wcast;
  }
  if (a_dtype == HAWK_F32) {
    auto* acast = reinterpret_cast<__nv_bfloat16*>(sv + S.ab);
    rc = hawk_cast_f32_bf16(static_cast<const float*>(act), acast, N * H, stream);
    if (rc != HAWK_OK) return rc;
    ab = acast;
  }
  // 2. logits + online softmax statistics.  The label's logit is written by the tile that holds the label;
  // a label outside [0, V) matches no tile, so its slot keeps this NaN pattern and the loss comes out NaN
  // (a label in the padding of the last chunk picks -inf: the loss comes out +inf).
  if (cudaMemsetAsync(correct, 0xFF, (size_t)N * sizeof(float), st) != cudaSuccess) {
    (void)cudaGetLastError();
    return HAWK_ERR_LAUNCH;
  }
  EpiParams ep{};
  ep.stats = stats;
  ep.correct = correct;
  ep.labels = reinterpret_cast<const long long*>(labels);
  rc = launch_gemm<EPI_LOGITS, 1, false, false>(ab, H, wb, H, logits, false, S.ldV, (int)N, (int)V, (int)H, 1, ep, status, st);
  if (rc != HAWK_OK) return rc;
  // 3. log-sum-exp per row and the mean loss
  ce_row_reduce_kernel<<<L.n_blocks, 256, 0, st>>>(stats, correct, lse, partial, (int)N, L.groups);
  ce_loss_final_kernel<<<1, 256, 0, st>>>(partial, L.n_blocks, 1.0f / (float)N, loss, status);
  // 4. dprobs in place
  if (want_grad)
    ce_dprobs_kernel<<<(unsigned)N, 256, 0, st>>>(logits, S.ldV, lse, reinterpret_cast<const long long*>(labels), (int)N,
                                                  (int)V, 1.0f / (float)N);
  return launch_status();
}

extern "C" int hawk_linear_ce_bwd(const void* weight, const void* act, const void* saved, size_t saved_bytes,
                                  const float* grad_loss, void* dweight, int dw_dtype, void* dact, int da_dtype,
                                  void* scratch, size_t scratch_bytes, int64_t N, int64_t H, int64_t V, int w_dtype,
                                  int a_dtype, int* status, void* stream) {
  HAWK_REQUIRE(weight && act && status && (dweight || dact), HAWK_ERR_NULL);
  HAWK_REQUIRE(valid_dtype(dw_dtype) && valid_dtype(da_dtype), HAWK_ERR_DTYPE);
  int rc = check_ce(N, H, V, w_dtype, a_dtype);
  if (rc != HAWK_OK) return rc;
  const CeSaved S = ce_saved(N, H, V, w_dtype, a_dtype);
  HAWK_REQUIRE(saved && saved_bytes >= S.total, HAWK_ERR_WORKSPACE);
  const size_t need = ce_bwd_scratch(N, H, V);
  HAWK_REQUIRE(need == 0 || (scratch && scratch_bytes >= need), HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(saved, 256) && aligned(scratch, 16) && aligned(dweight, 16) && aligned(dact, 16) &&
                   aligned(weight, 16) && aligned(act, 16) && aligned(grad_loss, 4),
               HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto* sv = static_cast<const unsigned char*>(saved);
  const auto* dprobs = reinterpret_cast<const __nv_bfloat16*>(sv + S.logits);
  const auto* wb = static_cast<const __nv_bfloat16*>(w_dtype == HAWK_F32 ? static_cast<const void*>(sv + S.wb) : weight);
  const auto* ab = static_cast<const __nv_bfloat16*>(a_dtype == HAWK_F32 ? static_cast<const void*>(sv + S.ab) : act);
  auto* part = static_cast<float*>(scratch);
  if (dact) {    // d act [N,H] = dprobs [N,V] . W [V,H]   : A K-major (dprobs rows), B MN-major (W's rows are the K index)
    rc = grad_gemm<false, true>(dprobs, S.ldV, wb, H, dact, da_dtype, grad_loss, (int)N, (int)H, (int)V, nullptr, part, status, st);
    if (rc != HAWK_OK) return rc;
  }
  if (dweight) {  // d weight [V,H] = dprobs^T . act [N,H] : A and B MN-major (the rows of dprobs and act are the K index)
    rc = grad_gemm<true, true>(dprobs, S.ldV, ab, H, dweight, dw_dtype, grad_loss, (int)V, (int)H, (int)N, nullptr, part, status, st);
    if (rc != HAWK_OK) return rc;
  }
  ce_poison_on_abort_kernel<<<1, 1, 0, st>>>(status, dweight, dw_dtype == HAWK_BF16, dact, da_dtype == HAWK_BF16);
  return launch_status();
}

extern "C" int hawk_linear_ce_fwd_bwd(const void* weight, const void* act, const int64_t* labels, float* loss,
                                      float* dweight, float* dact, void* workspace, size_t workspace_bytes,
                                      int64_t N, int64_t H, int64_t V, int dtype, int* status, void* stream) {
  HAWK_REQUIRE(weight && act && labels && loss && dweight && dact && status, HAWK_ERR_NULL);
  int rc = check_ce(N, H, V, dtype, dtype);
  if (rc != HAWK_OK) return rc;
  const size_t saved = ce_saved(N, H, V, dtype, dtype).total, scratch = hawk_linear_ce_scratch_bytes(N, H, V);
  HAWK_REQUIRE(workspace && workspace_bytes >= hawk_linear_ce_workspace_bytes(N, H, V), HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(workspace, 256) && aligned(dweight, 16) && aligned(dact, 16) && aligned(weight, 16) &&
                   aligned(act, 16),
               HAWK_ERR_ALIGN);
  auto* sc = static_cast<unsigned char*>(workspace) + saved;
  rc = hawk_linear_ce_fwd(weight, act, labels, loss, workspace, saved, sc, scratch, N, H, V, dtype, dtype, 1, status, stream);
  if (rc != HAWK_OK) return rc;
  rc = hawk_linear_ce_bwd(weight, act, workspace, saved, nullptr, dweight, HAWK_F32, dact, HAWK_F32, sc, scratch, N, H, V,
                          dtype, dtype, status, stream);
  if (rc != HAWK_OK) return rc;
  ce_poison_on_abort_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(status, loss, 0, nullptr, 0);
  return launch_status();
}
