// Log probability and entropy of tokens from activations and the head's weight, x = act W^T, and both gradients.  The logits
// are never rounded and never in memory:
//   1. GEMM (head_gemm.cuh) whose epilogue reduces every row's 128 columns, from the fp32 accumulators, to their maximum m_g,
//      the sum of e = e^(x - m_g) and the sum of e (x - m_g) log2 e; the token's logit is picked out on the way.  Where a
//      gradient is wanted it stores e, in fp16: at most 1, so its rounding is 2^-12 of a probability (2^-25 of the group's largest
//      below 2^-14 of it) whatever the logits' size (a bf16 logit of 20 is off by 0.06, 6 % of its probability), and exactly 1 at
//      each group's maximum, so that the probability of a token that is all but certain is as exact as the sums.
//   2. reduce  a warp per row over its groups: m, log s, log probability and entropy.  The token's own logit is formed once more,
//      as a plain fp32 dot product: the tensor core truncates its running sum at every step of 16 products, which leaves a large
//      logit a little too small (2e-5 of 16 after 2048 products), and a log probability near 0 would be nothing but that.  The
//      sums get its term anew as well.  N rows of act and weight read: 50 us of 11 ms at N32760 H2048 V32000.
// Backward, from e and the groups' maxima (2 N V bytes kept instead of a third GEMM: forming the logits again takes 2 N H V
// flops, 3.1 ms at N32760 H2048 V32000 where writing and reading e takes 1):
//   3. d x     d x_j = -p_j (g_lp + g_H (log p_j + H)) with p_j = e_j e^(m_g - m - log s), and at the token from its exact log
//      probability, g_lp (1 - p) as -expm1; bf16 for the products, out of place: a second backward finds e as it was.
//   4. two GEMMs, d act = dx W and d W = dx^T act.
// Bound by the tensor pipe: 2 N H V flops forward, 4 N H V backward.  Measured at N32760 H2048 V32000 in bf16: 3.13 ms without and
// 3.23 ms with what a backward needs (1.37 / 1.33 PFLOP/s), backward 6.35 ms (1.35; dx 0.71 at 5.9 TB/s, the GEMMs 2.74 and 2.80),
// 10.9 to 11.3 ms together in a sustained loop.  At small H the logits' epilogue sets the pace: H512 N3108 97 us without, 118 with
// (0.06 of MMAs).
#include "head_gemm.cuh"

namespace hawk {

__global__ void __launch_bounds__(256)
score_reduce_kernel(const float4* __restrict__ score, const float* __restrict__ correct, const int64_t* __restrict__ tokens,
                    const __nv_bfloat16* __restrict__ weight, const __nv_bfloat16* __restrict__ act, float* __restrict__ logprob,
                    float* __restrict__ entropy, float2* __restrict__ stats, int N, int H, int V, int groups,
                    const int* __restrict__ status) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= N) return;
  const float4* g = score + (long long)row * groups;
  const int64_t token = tokens[row];
  float own = 0.f;
  if (token >= 0 && token < V) {
    const __nv_bfloat16 *a = act + (long long)row * H, *w = weight + token * H;
#pragma unroll 4
    for (int i = lane * 8; i < H; i += 256) {
      float av[8], wv[8];
      VecIO<__nv_bfloat16, 8>::load(a + i, av);
      VecIO<__nv_bfloat16, 8>::load(w + i, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) own = fmaf(av[j], wv[j], own);
    }
  }
  float m = -INFINITY;
  for (int i = lane; i < groups; i += 32) m = fmaxf(m, g[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = 0.f, sx = 0.f;
  for (int i = lane; i < groups; i += 32) {
    const float4 v = g[i];
    const float t = (v.x - m) * kLog2e, k = ex2_approx(t);
    s = fmaf(v.y, k, s);
    // the group's terms are relative to its own maximum: each moves by t; far below, k is 0 and t finite
    sx = fmaf(fmaf(v.y, t, v.z), k, sx);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    sx += __shfl_xor_sync(0xffffffffu, sx, o);
    own += __shfl_xor_sync(0xffffffffu, own, o);
  }
  if (lane == 0) {
    const float nan = __int_as_float(0x7fc00000);
    if (token >= 0 && token < V) {
      const float t0 = (correct[row] - m) * kLog2e, t1 = (own - m) * kLog2e, e0 = ex2_approx(t0), e1 = ex2_approx(t1);
      s = (s - e0) + e1;
      sx = (sx - e0 * t0) + e1 * t1;
    } else {
      own = nan;
    }
    const float logs = logf(s);
    float lp = (own - m) - logs, ent = logs - 0.6931471805599453f * sx / s;
    if (token < 0) lp = ent = 0.f;
    if (*status != 0) lp = ent = nan;  // a GEMM gave up a wait (this call's, or an earlier one nobody has looked at)
    logprob[row] = lp;
    entropy[row] = ent;
    stats[row] = make_float2(m, logs);
  }
}

constexpr int kDxThreads = 512;
// d x of one row per block, 8 columns (16 bytes of e, of one group) per thread and step
__global__ void __launch_bounds__(kDxThreads)
score_dx_kernel(const __half* __restrict__ e, const float4* __restrict__ score, const float2* __restrict__ stats,
                const float* __restrict__ logprob, const float* __restrict__ entropy, const int64_t* __restrict__ tokens,
                const float* __restrict__ g_lp, const float* __restrict__ g_ent, __nv_bfloat16* __restrict__ dx, long long ld, int V,
                int groups) {
  const long long row = blockIdx.x;
  const int64_t token = tokens[row];
  const int nvec = (V + 7) / 8;  // ld is a multiple of 8; what lies behind V is never read
  __nv_bfloat16* out = dx + row * ld;
  if (token < 0) {
    for (int i = threadIdx.x; i < nvec; i += kDxThreads) reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const __half* in = e + row * ld;
  const float4* g = score + row * groups;
  const float2 st = stats[row];
  const float lp = logprob[row], H = entropy[row], gl = g_lp ? g_lp[row] : 0.f, gh = g_ent ? g_ent[row] : 0.f;
  const bool known = token < V;
#pragma unroll 4
  for (int i = threadIdx.x; i < nvec; i += kDxThreads) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(in) + i);
    const float off = (__ldg(&g[i / (EPI_COLS / 8)].x) - st.x) - st.y;  // log p of the group's maximum
    const float f = known ? ex2_approx(off * kLog2e) : __int_as_float(0x7fc00000);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float d[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 ev = unpack_f16x2(w[q]);
      float c0 = gl, c1 = gl;
      if (gh != 0.f) {  // the same for all of the row
        c0 = fmaf(gh, fmaf(fmaxf(__log2f(ev.x), -200.f), 0.6931471805599453f, off) + H, gl);  // e = 0: a finite factor
        c1 = fmaf(gh, fmaf(fmaxf(__log2f(ev.y), -200.f), 0.6931471805599453f, off) + H, gl);
      }
      d[2 * q] = -ev.x * f * c0;
      d[2 * q + 1] = -ev.y * f * c1;
    }
    const int64_t at = token - (int64_t)i * 8;
    if (at >= 0 && at < 8) {
      const float own = fmaf(-gl, expm1f(lp), -gh * expf(lp) * (lp + H));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j == (int)at) d[j] = own;
    }
    VecIO<__nv_bfloat16, 8>::store(out + (long long)i * 8, d);
  }
}

// act with the left-out rows zeroed: d x is 0 there, but 0 times what they hold need not be
__global__ void __launch_bounds__(256)
keep_rows_kernel(const __nv_bfloat16* __restrict__ act, const int64_t* __restrict__ tokens, __nv_bfloat16* __restrict__ out, long long vectors,
                 int per_row) {
  for (long long i = (long long)blockIdx.x * 1024 + threadIdx.x, end = min(vectors, (long long)(blockIdx.x + 1) * 1024); i < end; i += 256)
    reinterpret_cast<uint4*>(out)[i] =
        tokens[i / per_row] < 0 ? make_uint4(0u, 0u, 0u, 0u) : __ldg(reinterpret_cast<const uint4*>(act) + i);
}

// ---- host --------------------------------------------------------------------------------------------------
// What the forward leaves: bf16 copies of fp32 operands, the groups' statistics and the rows', e (only for a backward)
struct ScoreSaved {
  size_t wb, ab, score, stats, correct, e, total;
  long long ldV;
  int groups;
};
static ScoreSaved score_saved(long long N, long long H, long long V, int w_dtype, int a_dtype, bool keep) {
  ScoreSaved L;
  L.ldV = (V + 7) & ~7LL;
  L.groups = (int)((V + EPI_COLS - 1) / EPI_COLS);
  size_t o = 0;
  L.wb = o;      o += w_dtype == HAWK_F32 ? up256((size_t)V * H * 2) : 0;
  L.ab = o;      o += a_dtype == HAWK_F32 ? up256((size_t)N * H * 2) : 0;
  L.score = o;   o += up256((size_t)N * L.groups * sizeof(float4));
  L.stats = o;   o += up256((size_t)N * sizeof(float2));
  L.correct = o; o += up256((size_t)N * 4);
  L.e = o;       o += keep ? up256((size_t)N * L.ldV * 2) : 0;
  L.total = o;
  return L;
}
struct ScoreScratch {
  size_t dx, act, partial, total;
};
static ScoreScratch score_scratch(long long N, long long H, long long V, int a_dtype, bool want_dw, bool want_da) {
  ScoreScratch L;
  size_t o = 0, part = 0;
  L.dx = o;      o += up256((size_t)N * ((V + 7) & ~7LL) * 2);
  L.act = o;     o += want_dw ? up256((size_t)N * H * 2) : 0;
  if (want_da && plan_grad(N, H, V).splits > 1) part = (size_t)plan_grad(N, H, V).splits * N * H * 4;
  if (want_dw && plan_grad(V, H, N).splits > 1) part = std::max<size_t>(part, (size_t)plan_grad(V, H, N).splits * V * H * 4);
  L.partial = o; o += up256(part);
  L.total = o;
  return L;
}

static int check_score(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype) {
  HAWK_REQUIRE(valid_dtype(w_dtype) && valid_dtype(a_dtype), HAWK_ERR_DTYPE);
  HAWK_REQUIRE(N >= 1 && V >= 1 && H >= 8 && H % 8 == 0, HAWK_ERR_SHAPE);
  HAWK_REQUIRE(N < (1LL << 31) - 512 && V < (1LL << 31) - 512 && H < (1LL << 31) - 512, HAWK_ERR_SHAPE);
  return HAWK_OK;
}

}  // namespace hawk

using namespace hawk;

extern "C" size_t hawk_linear_logprobs_saved_bytes(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int want_grad) {
  if (N < 1 || H < 1 || V < 1) return 0;
  return score_saved(N, H, V, w_dtype, a_dtype, want_grad != 0).total;
}

extern "C" size_t hawk_linear_logprobs_scratch_bytes(int64_t N, int64_t H, int64_t V, int a_dtype, int want_dw, int want_da) {
  if (N < 1 || H < 1 || V < 1) return 0;
  return score_scratch(N, H, V, a_dtype, want_dw != 0, want_da != 0).total;
}

// the forward (want_dw = want_da = 0): a cast per fp32 operand, the GEMM and the reduction; the backward: d x, the copy of act, a
// GEMM and where K is split a sum for each gradient, the look at the status word
extern "C" int hawk_linear_logprobs_kernels(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int want_dw, int want_da) {
  if (N < 1 || H < 1 || V < 1) return 0;
  if (!want_dw && !want_da) return (w_dtype == HAWK_F32) + (a_dtype == HAWK_F32) + 2;
  int n = 2;
  if (want_dw) n += plan_grad(V, H, N).splits > 1 ? 3 : 2;
  if (want_da) n += plan_grad(N, H, V).splits > 1 ? 2 : 1;
  return n;
}

extern "C" int hawk_linear_logprobs(const void* weight, const void* act, const int64_t* tokens, float* logprob, float* entropy, void* saved,
                                    size_t saved_bytes, int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int want_grad,
                                    int* status, void* stream) {
  HAWK_REQUIRE(weight && act && tokens && logprob && entropy && status, HAWK_ERR_NULL);
  int rc = check_score(N, H, V, w_dtype, a_dtype);
  if (rc != HAWK_OK) return rc;
  const ScoreSaved S = score_saved(N, H, V, w_dtype, a_dtype, want_grad != 0);
  HAWK_REQUIRE(saved && saved_bytes >= S.total, HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(saved, 256) && aligned(weight, 16) && aligned(act, 16) && aligned(tokens, 8) && aligned(logprob, 4) &&
                   aligned(entropy, 4),
               HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* sv = static_cast<unsigned char*>(saved);
  const __nv_bfloat16* wb = static_cast<const __nv_bfloat16*>(weight);
  const __nv_bfloat16* ab = static_cast<const __nv_bfloat16*>(act);
  if (w_dtype == HAWK_F32) {
    rc = hawk_cast_f32_bf16(static_cast<const float*>(weight), sv + S.wb, V * H, stream);
    if (rc != HAWK_OK) return rc;
    wb = reinterpret_cast<const __nv_bfloat16*>(sv + S.wb);
  }
  if (a_dtype == HAWK_F32) {
    rc = hawk_cast_f32_bf16(static_cast<const float*>(act), sv + S.ab, N * H, stream);
    if (rc != HAWK_OK) return rc;
    ab = reinterpret_cast<const __nv_bfloat16*>(sv + S.ab);
  }
  // a token outside [0, V) is in no tile: its logit stays this NaN
  auto* correct = reinterpret_cast<float*>(sv + S.correct);
  if (cudaMemsetAsync(correct, 0xFF, (size_t)N * sizeof(float), st) != cudaSuccess) {
    (void)cudaGetLastError();
    return HAWK_ERR_LAUNCH;
  }
  EpiParams ep{};
  ep.score = reinterpret_cast<float4*>(sv + S.score);
  ep.groups = S.groups;
  ep.correct = correct;
  ep.labels = reinterpret_cast<const long long*>(tokens);
  if (want_grad)
    rc = launch_gemm<EPI_SCORE_KEEP, 1, false, false>(ab, H, wb, H, sv + S.e, false, S.ldV, (int)N, (int)V, (int)H, 1, ep, status, st);
  else
    rc = launch_gemm<EPI_SCORE, 1, false, false>(ab, H, wb, H, nullptr, false, S.ldV, (int)N, (int)V, (int)H, 1, ep, status, st);
  if (rc != HAWK_OK) return rc;
  score_reduce_kernel<<<(unsigned)((N + 7) / 8), 256, 0, st>>>(ep.score, correct, tokens, wb, ab, logprob, entropy,
                                                               reinterpret_cast<float2*>(sv + S.stats), (int)N, (int)H, (int)V, S.groups,
                                                               status);
  return launch_status();
}

extern "C" int hawk_linear_logprobs_bwd(const void* weight, const void* act, const int64_t* tokens, const void* saved, size_t saved_bytes,
                                        const float* logprob, const float* entropy, const float* g_logprob, const float* g_entropy,
                                        void* dweight, int dw_dtype, void* dact, int da_dtype, void* scratch, size_t scratch_bytes,
                                        int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int* status, void* stream) {
  HAWK_REQUIRE(weight && act && tokens && logprob && entropy && status && (dweight || dact), HAWK_ERR_NULL);
  HAWK_REQUIRE(valid_dtype(dw_dtype) && valid_dtype(da_dtype), HAWK_ERR_DTYPE);
  int rc = check_score(N, H, V, w_dtype, a_dtype);
  if (rc != HAWK_OK) return rc;
  const ScoreSaved S = score_saved(N, H, V, w_dtype, a_dtype, true);
  const ScoreScratch L = score_scratch(N, H, V, a_dtype, dweight != nullptr, dact != nullptr);
  HAWK_REQUIRE(saved && saved_bytes >= S.total && scratch && scratch_bytes >= L.total, HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(saved, 256) && aligned(scratch, 256) && aligned(dweight, 16) && aligned(dact, 16) && aligned(weight, 16) &&
                   aligned(act, 16) && aligned(tokens, 8) && aligned(logprob, 4) && aligned(entropy, 4) && aligned(g_logprob, 4) &&
                   aligned(g_entropy, 4),
               HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto* sv = static_cast<const unsigned char*>(saved);
  auto* sc = static_cast<unsigned char*>(scratch);
  const auto* wb = static_cast<const __nv_bfloat16*>(w_dtype == HAWK_F32 ? static_cast<const void*>(sv + S.wb) : weight);
  const auto* ab = static_cast<const __nv_bfloat16*>(a_dtype == HAWK_F32 ? static_cast<const void*>(sv + S.ab) : act);
  auto* dx = reinterpret_cast<__nv_bfloat16*>(sc + L.dx);
  auto* part = reinterpret_cast<float*>(sc + L.partial);
  score_dx_kernel<<<(unsigned)N, kDxThreads, 0, st>>>(reinterpret_cast<const __half*>(sv + S.e),
                                                      reinterpret_cast<const float4*>(sv + S.score),
                                                      reinterpret_cast<const float2*>(sv + S.stats), logprob, entropy, tokens, g_logprob,
                                                      g_entropy, dx, S.ldV, (int)V, S.groups);
  rc = launch_status();
  if (rc != HAWK_OK) return rc;
  if (dact) {  // d act [N,H] = dx [N,V] . W [V,H]: A K-major, B MN-major (W's rows are the K index)
    rc = grad_gemm<false, true>(dx, S.ldV, wb, H, dact, da_dtype, nullptr, (int)N, (int)H, (int)V, part, status, st);
    if (rc != HAWK_OK) return rc;
  }
  if (dweight) {  // d weight [V,H] = dx^T . act [N,H]: A and B MN-major (the rows of dx and act are the K index)
    auto* kept = reinterpret_cast<__nv_bfloat16*>(sc + L.act);
    const long long vectors = N * H / 8;
    keep_rows_kernel<<<(unsigned)((vectors + 1023) / 1024), 256, 0, st>>>(ab, tokens, kept, vectors, (int)(H / 8));
    rc = launch_status();
    if (rc != HAWK_OK) return rc;
    rc = grad_gemm<true, true>(dx, S.ldV, kept, H, dweight, dw_dtype, nullptr, (int)V, (int)H, (int)N, part, status, st);
    if (rc != HAWK_OK) return rc;
  }
  ce_poison_on_abort_kernel<<<1, 1, 0, st>>>(status, dweight, dw_dtype == HAWK_BF16, dact, da_dtype == HAWK_BF16);
  return launch_status();
}
