// Log probability and entropy of tokens from activations and the head's weight, x = act W^T, and both gradients.  The logits
// are never rounded and never in memory:
//   0. rows    those that name a token, listed in order and their activations copied together (in bf16): the products below
//      take only them, as many as the list's length on the device says, so padding and prompts cost nothing: of 32760 rows of 2048
//      (V32000) forward and backward take 9.7 ms all named, 5.3 with half of them left out, 1.2 with 9 of 10.  48 us with all
//      of them named, and the scatter of d act as long again; the same launch casts an fp32 weight.
//   1. GEMM (head_gemm.cuh) whose epilogue reduces every row's 128 columns, from the fp32 accumulators, to their maximum m_g,
//      the sum of e = e^(x - m_g) and the sum of e (x - m_g) log2 e; the token's logit is picked out on the way.  Where a
//      gradient is wanted it stores e, in fp16: at most 1, so its rounding is 2^-12 of a probability (2^-25 of the group's largest
//      below 2^-14 of it) whatever the logits' size (a bf16 logit of 20 is off by 0.06, 6 % of its probability), and exactly 1 at
//      each group's maximum, so that the probability of a token that is all but certain is as exact as the sums.
//   2. reduce  a warp per row over its groups: m, log s, log probability and entropy.  The token's own logit is formed once more,
//      as a plain fp32 dot product: the tensor core truncates its running sum at every step of 16 products, which leaves a large
//      logit a little too small (2e-5 of 16 after 2048 products), and a log probability near 0 would be nothing but that.  The
//      sums get its term anew as well.  Elements at a group's maximum are counted apart where little else may be in the group, and
//      log s is log1p of the rest, so that 1 - p of a token that is all but certain is as exact as the logits.  N rows of act and
//      weight read: 67 us of 11 ms at N32760 H2048 V32000.
// Backward, from e and the groups' maxima (2 N V bytes kept instead of a third GEMM: forming the logits again takes 2 N H V
// flops, 3.1 ms at N32760 H2048 V32000 where writing and reading e takes 1):
//   3. d x     d x_j = -p_j (g_lp + g_H (log p_j + H)) with p_j = e_j e^(m_g - m - log s), and at the token from its exact log
//      probability, g_lp (1 - p) as -expm1 (log p_j of the others is that of the rounded e_j, 2^-12 off: where the two terms of a
//      small vocabulary nearly cancel, that much of g_H p_j is left); bf16 for the products, out of place: a second backward finds e as it was.  The token's
//      element is most of its row, so the row is first scaled, by up to 2, to where that element is a bf16 number, and d act's
//      row is scaled back as it leaves the product: its error is then that of its own rounding alone (1.7e-3 in norm where two
//      roundings left 2.4e-3).  d W takes the row's activations scaled back, a copy rounded to bf16 once more.  Each row has a scale
//      of its own (dithered): where the upstream gradients are alike (a mean), so are the tokens' elements, and one scale
//      for all, the nearest bf16 number's, would leave a common factor in the whole d W (0.34 % at 255 rows if the activations stayed as
//      they are, 0.09 % with them scaled back, since they lie on bf16's grid), where independent roundings average out.  Few
//      rows d W takes twice, as two bf16 numbers to each of fp32, from a scale within 2^-8 of 1 (kTwiceRows).
//   4. two GEMMs, d act = dx W and d W = dx^T act; d act's rows go back to their places.
// Bound by the tensor pipe: 2 N H V flops forward, 4 N H V backward.  Measured at N32760 H2048 V32000 in bf16, all rows named:
// 3.13 ms without and 3.28 ms with what a backward needs (1.37 / 1.31 PFLOP/s), backward 6.2 to 6.5 ms (1.34; dx 0.7, the
// GEMMs 2.74 and 2.80), 10.3 ms together in a sustained loop with a tenth left out.  At small H the logits' epilogue sets the pace:
// H512 N3108 110 us without, 132 with (0.06 of MMAs).
#include "head_gemm.cuh"

namespace hawk {

// What the forward finds out about its rows, on the device
struct ScoreRows {
  int* count;        // how many name a token: the compact rows 0 .. count - 1 below; behind it the K rows of the d W product
  int* row;          // [N] compact row -> row
  int64_t* token;    // [N] compact row -> token (>= 0)
};
// The d W product reads whole K blocks of BK compact rows, zeros behind the last one.  Where few rows are named it reads each twice: as
// many rows follow with what rounding d x to bf16 left, and act again, as it is.  (Sums of few terms do not average their roundings: d W
// of 8 to 64 rows was 1.2 to 1.76 times as far off as a single rounding leaves it, and is 1.00 now; from 200 rows on 1.35 to 1.5, in
// thousands 1.41 to 1.46.  The backward of 31 / 128 rows at H2048 V32000 takes 93 / 106 us instead of 88 / 96.)
constexpr int kTwiceRows = 128;
__host__ __device__ constexpr int64_t whole_blocks(int64_t rows) { return (rows + BK - 1) / BK * BK; }
__device__ __forceinline__ int padded_count(int count) { return (int)whole_blocks(max(count, 1)); }
__device__ __forceinline__ bool twice(int count) { return count <= kTwiceRows; }
// rows that d x and the activations beside it have room for
__host__ __device__ constexpr int64_t room_rows(int64_t N) {
  return whole_blocks(N) > 2 * kTwiceRows ? whole_blocks(N) : 2 * whole_blocks(N) < 2 * kTwiceRows ? 2 * whole_blocks(N) : 2 * kTwiceRows;
}

// The first row_blocks blocks list `per` rows each (at most one to a thread): a block counts the named tokens before its own by
// itself, so there is no second launch and no order between blocks.  That is N^2 / (2 per) tokens read from L2 in all: 75 MB at
// N = 32760, of the 270 that are copied, but 64 ms at 10 M rows; longer lists are counted by block first (`counts`, null otherwise) and
// a block adds up the counts before its own.  The forward of short rows (H16 V64) without / with the count: 4096 rows 23.6 / 26 us, 16384
// 35.8 / 35.9, 32768 50 / 46, 65536 81 / 67, 131072 140 / 108.  The other blocks cast the weight.
constexpr int64_t kCountedRows = 32768;
__global__ void __launch_bounds__(256) score_count_kernel(const int64_t* __restrict__ tokens, int* __restrict__ counts, int N, int per) {
  const int row = blockIdx.x * per + threadIdx.x;
  const int n = __syncthreads_count((int)threadIdx.x < per && row < N && __ldg(tokens + min(row, N - 1)) >= 0);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

template <typename T>
__global__ void __launch_bounds__(256)
score_prepare_kernel(const int64_t* __restrict__ tokens, const T* __restrict__ act, ScoreRows rows, __nv_bfloat16* __restrict__ compact,
                     float* __restrict__ correct, float* __restrict__ logprob, float* __restrict__ entropy, int N, int H, int per,
                     int row_blocks, const int* __restrict__ counts, const float* __restrict__ weight, __nv_bfloat16* __restrict__ wb, long long wvec) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= row_blocks) {
    const long long at = ((long long)blockIdx.x - row_blocks) * 1024 + tid;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long i = at + q * 256;
      if (i < wvec) {
        float v[8];
        VecIO<float, 8>::load(weight + i * 8, v);
        VecIO<__nv_bfloat16, 8>::store(wb + i * 8, v);
      }
    }
    return;
  }
  __shared__ int sums[2][8], source[256];
  const int first = blockIdx.x * per, own = min(per, N - first);
  int before = 0;
  if (counts) {
#pragma unroll 8
    for (int i = tid; i < (int)blockIdx.x; i += 256) before += __ldg(counts + i);
  } else {
#pragma unroll 8
    for (int i = tid; i < first; i += 256) before += __ldg(tokens + i) >= 0;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  const int64_t token = tid < own ? __ldg(tokens + first + tid) : -1;
  const uint32_t named = __ballot_sync(0xffffffffu, token >= 0);
  if (lane == 0) {
    sums[0][warp] = before;
    sums[1][warp] = __popc(named);
  }
  __syncthreads();
  before = 0;
  int at = __popc(named & ((1u << lane) - 1)), total = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before += sums[0][w];
    total += sums[1][w];
    if (w < warp) at += sums[1][w];
  }
  if (tid < own) {
    const int row = first + tid;
    correct[row] = __int_as_float(0x7fc00000);  // a token >= V is in no tile: its logit stays this NaN
    if (token >= 0) {
      rows.row[before + at] = row;
      rows.token[before + at] = token;
      source[at] = row;
    } else {
      logprob[row] = entropy[row] = 0.f;
    }
  }
  if (tid == 0 && first + own == N) {
    const int n = before + total;
    rows.count[0] = n;
    rows.count[1] = twice(n) ? 2 * padded_count(n) : n;
  }
  __syncthreads();
  const int vecs = H / 8, all = total * vecs;
#pragma unroll 4
  for (int i = tid; i < all; i += 256) {
    const int r = i / vecs, c = (i - r * vecs) * 8;
    float v[8];
    VecIO<T, 8>::load(act + (long long)source[r] * H + c, v);
    VecIO<__nv_bfloat16, 8>::store(compact + (long long)(before + r) * H + c, v);
  }
}

// a warp to a compact row; `act` compact
__global__ void __launch_bounds__(256)
score_reduce_kernel(const float4* __restrict__ score, const float* __restrict__ correct, ScoreRows rows,
                    const __nv_bfloat16* __restrict__ weight, const __nv_bfloat16* __restrict__ act, float* __restrict__ logprob,
                    float* __restrict__ entropy, float2* __restrict__ stats, int H, int V, int groups,
                    const int* __restrict__ status) {
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= *rows.count) return;
  const float4* g = score + (long long)r * groups;
  const int64_t token = rows.token[r];
  float own = 0.f;
  if (token < V) {
    const __nv_bfloat16 *a = act + (long long)r * H, *w = weight + token * H;
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
  float s = 0.f, sx = 0.f, ties = 0.f;  // ties: elements at the row's maximum that their group's sum leaves out
  for (int i = lane; i < groups; i += 32) {
    const float4 v = g[i];
    const float t = (v.x - m) * kLog2e, k = ex2_approx(t), all = v.y + v.w;
    if (v.x == m) {
      s += v.y;
      ties += v.w;
    } else {
      s = fmaf(all, k, s);
    }
    // the group's terms are relative to its own maximum: each moves by t; far below, k is 0 and t finite
    sx = fmaf(fmaf(all, t, v.z), k, sx);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    sx += __shfl_xor_sync(0xffffffffu, sx, o);
    ties += __shfl_xor_sync(0xffffffffu, ties, o);
    own += __shfl_xor_sync(0xffffffffu, own, o);
  }
  if (lane == 0) {
    const float nan = __int_as_float(0x7fc00000), c = correct[r];
    float lp = nan, rest = (ties - 1.f) + s, logs = log1pf(rest), base = logs;  // rest: the sum less 1
    sx *= -0.6931471805599453f;
    if (token < V) {
      const float d = own - m, t0 = (c - m) * kLog2e, t1 = d * kLog2e, e0 = ex2_approx(t0), e1 = ex2_approx(t1);
      const bool tied = c == m && ties > 0.f;
      const float others = tied ? rest : (s - e0) + ties;
      rest = tied ? rest + expm1f(d) : (ties - 1.f) + ((s - e0) + e1);
      logs = log1pf(rest);
      sx += e0 * (c - m);
      if (d > -1.f) {  // the token has a good part of the sum: from the others, and from where they lie below it
        lp = -log1pf(others * ex2_approx(-t1));
        base = -lp;
        sx = fmaf(others, d, sx);
      } else {
        lp = d - logs;
        base = logs;
        sx -= e1 * d;
      }
    }
    float ent = base + sx / (rest + 1.f);
    if (*status != 0) lp = ent = nan;  // a GEMM gave up a wait (this call's, or an earlier one nobody has looked at)
    logprob[rows.row[r]] = lp;
    entropy[rows.row[r]] = ent;
    stats[r] = make_float2(m, logs);
  }
}

// the bf16 number of v's sign and exponent whose mantissa is row r's: 7 bits of a multiple of the golden ratio, evenly spread
__device__ __forceinline__ float dithered(float v, uint32_t r) {
  return __uint_as_float((__float_as_uint(v) & 0xff800000u) | r * 2654435769u >> 25 << 16);
}

// the token's element of d x and what it is stored as: where it is exact in bf16 the row is scaled by own16 / own
struct TokenElement {
  float own, own16, shrink, grow;
  __device__ __forceinline__ TokenElement(float lp, float H, float gl, float gh, uint32_t r, bool two) {
    own = fmaf(-gl, expm1f(lp), -gh * expf(lp) * (lp + H));
    const bool scaled = fabsf(own) > 1e-30f && fabsf(own) < 1e37f;
    own16 = scaled && !two ? dithered(own, r) : __bfloat162float(__float2bfloat16(own));
    shrink = scaled ? own16 / own : 1.f;
    grow = scaled ? own / own16 : 1.f;
  }
};

// d x of a share of one compact row per block, 8 columns (16 bytes of e, of one group) per vector, all of a thread's requested before
// what the row's factors are known, pairs of fp32 operations, and no call in the loop.  16380 rows of 32000: 355 us (5.9 TB/s), 1548 rows 36;
// a row to a block of 512 threads in a loop with the token's element among the others 403 and 42.
// The blocks behind write the activations that the d W product takes with it, a warp to a row (3108 rows of 2048: 3 us more, by the
// first block of each row 10).
constexpr int kDxThreads = 256, kDxVectors = 4, kDxShare = kDxThreads * kDxVectors;
__global__ void __launch_bounds__(kDxThreads)
score_dx_kernel(const __half* __restrict__ e, const float4* __restrict__ score, const float2* __restrict__ stats,
                const float* __restrict__ logprob, const float* __restrict__ entropy, ScoreRows rows,
                const float* __restrict__ g_lp, const float* __restrict__ g_ent, __nv_bfloat16* __restrict__ dx, float* __restrict__ row_scale,
                const __nv_bfloat16* __restrict__ act, __nv_bfloat16* __restrict__ dw_act, long long ld, int V, int width, int groups,
                uint32_t shares, uint32_t dx_blocks) {
  if (blockIdx.x >= dx_blocks) {
    const int r = (int)(blockIdx.x - dx_blocks) * 8 + (int)(threadIdx.x >> 5), count = *rows.count, padded = padded_count(count);
    if (r >= padded) return;
    const bool named = r < count, two = twice(count);
    const int row = named ? rows.row[r] : 0;
    const TokenElement t(logprob[row], entropy[row], g_lp ? g_lp[row] : 0.f, g_ent ? g_ent[row] : 0.f, r, two);
    const uint4* from = reinterpret_cast<const uint4*>(act + (long long)r * width);
    uint4* to = reinterpret_cast<uint4*>(dw_act + (long long)r * width);
    uint4* again = reinterpret_cast<uint4*>(dw_act + (long long)(padded + r) * width);
#pragma unroll 4
    for (int i = threadIdx.x & 31; i < width / 8; i += 32) {
      uint4 a = named ? __ldg(from + i) : make_uint4(0u, 0u, 0u, 0u);
      if (two) {
        again[i] = a;
      } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = mul2(unpack_bf16x2(w[k]), f2(t.grow));
          w[k] = pack_bf16x2(v.x, v.y);
        }
      }
      to[i] = a;
    }
    return;
  }
  const uint32_t r = blockIdx.x / shares;
  const int i0 = (int)(blockIdx.x - r * shares) * kDxShare + (int)threadIdx.x;
  const int nvec = (V + 7) / 8;  // ld is a multiple of 8; what lies behind V is never read
  const uint4* in = reinterpret_cast<const uint4*>(e + r * ld);
  const float4* g = score + (long long)r * groups;
  __nv_bfloat16* out = dx + r * ld;
  const int count = *rows.count;
  __nv_bfloat16* rest = twice(count) ? out + padded_count(count) * ld : nullptr;
  if ((int)r >= count) {
    if ((int)r >= padded_count(count)) return;
#pragma unroll
    for (int q = 0; q < kDxVectors; ++q)
      if (i0 + q * kDxThreads < nvec) {
        reinterpret_cast<uint4*>(out)[i0 + q * kDxThreads] = make_uint4(0u, 0u, 0u, 0u);
        if (rest) reinterpret_cast<uint4*>(rest)[i0 + q * kDxThreads] = make_uint4(0u, 0u, 0u, 0u);
      }
    return;
  }
  uint4 raw[kDxVectors];
  float mg[kDxVectors];
#pragma unroll
  for (int q = 0; q < kDxVectors; ++q) {
    const int i = i0 + q * kDxThreads;
    if (i < nvec) {
      raw[q] = __ldg(in + i);
      mg[q] = __ldg(&g[i / (EPI_COLS / 8)].x);
    }
  }
  const int row = rows.row[r];
  const int64_t token = rows.token[r];
  const float2 st = stats[r];
  const float lp = logprob[row], H = entropy[row], gl = g_lp ? g_lp[row] : 0.f, gh = g_ent ? g_ent[row] : 0.f;
  const bool known = token < V;
  const TokenElement el(lp, H, gl, gh, r, rest != nullptr);
  const float own = el.own, own16 = el.own16, shrink = el.shrink, grow = el.grow;
  if (blockIdx.x == r * shares && threadIdx.x == 0) row_scale[r] = grow;
#pragma unroll
  for (int q = 0; q < kDxVectors; ++q) {
    const int i = i0 + q * kDxThreads;
    if (i >= nvec) break;
    const float off = (mg[q] - st.x) - st.y;  // log p of the group's maximum
    const float2 f = f2(known ? -ex2_approx(off * kLog2e) * shrink : __int_as_float(0x7fc00000)), k0 = f2(off + H);
    const uint32_t w[4] = {raw[q].x, raw[q].y, raw[q].z, raw[q].w};
    float d[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 ev = unpack_f16x2(w[k]);
      float2 c = f2(gl);
      if (gh != 0.f) {  // the same for all of the row.  2^-40: a finite factor where e = 0, nothing to the others (2^-24 at least)
        const float2 l = add2(ev, f2(0x1p-40f));
        c = fma2(f2(gh), fma2(make_float2(__log2f(l.x), __log2f(l.y)), f2(0.6931471805599453f), k0), c);
      }
      c = mul2(mul2(ev, f), c);
      d[2 * k] = c.x;
      d[2 * k + 1] = c.y;
    }
    VecIO<__nv_bfloat16, 8>::store(out + (long long)i * 8, d);
    if (rest) {
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = fmaf(grow, d[j], -__bfloat162float(__float2bfloat16(d[j])));
      VecIO<__nv_bfloat16, 8>::store(rest + (long long)i * 8, d);
    }
  }
  // the token's own element anew, by the thread that wrote it
  const int64_t in_share = token / 8 - (i0 - (int)threadIdx.x);
  if (known && in_share >= 0 && in_share < kDxShare && (int)threadIdx.x == (int)in_share % kDxThreads) {
    out[token] = __float2bfloat16(own16);
    if (rest) rest[token] = __float2bfloat16(own - own16);
  }
}

// d act from its compact rows: the sum over the splits of K, to the rows that they belong to, and zeros to the others.  A warp to 256
// columns of a row, a vector of 8 to a lane, or to 1024 where there is nothing to add up.  N32760 H2048 in bf16 48 us (a thread to a vector, which divides 64-bit numbers: 68)
struct ScatterPlan {  // what the GEMM knew when it planned its splits (part_rows 0: one, no partial sums)
  int tile_rows, n_tiles, kblocks, planned, part_rows, pairs;
};
template <typename TC, typename TO, int kVecs>
__global__ void __launch_bounds__(256)
score_scatter_kernel(const TC* __restrict__ part, ScatterPlan plan, const int64_t* __restrict__ tokens, ScoreRows rows, TO* __restrict__ out,
                     uint32_t units, uint32_t chunks, int H, const int* __restrict__ status, void* dw, int dw_bf16) {
  const uint32_t unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const bool failed = *status != 0;  // a GEMM gave up a wait: NaN in the rows of d act, and in d weight's first element
  if (failed && dw && blockIdx.x == 0 && threadIdx.x == 0) {
    if (dw_bf16) *static_cast<__nv_bfloat16*>(dw) = __float2bfloat16(__int_as_float(0x7fc00000));
    else *static_cast<float*>(dw) = __int_as_float(0x7fc00000);
  }
  const int r = (int)(unit / chunks), c0 = ((int)(unit - r * chunks) * 32 * kVecs + (threadIdx.x & 31)) * 8;
  const bool mine = r < *rows.count;
  if (tokens[r] < 0) {
    const float zero[8] = {};
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
      if (c0 + q * 256 < H) VecIO<TO, 8>::store(out + (long long)r * H + c0 + q * 256, zero);
  }
  if (!mine) return;
  float v[kVecs][8];
  const TC* in = part + (long long)r * H + c0;
#pragma unroll
  for (int q = 0; q < kVecs; ++q)
    if (c0 + q * 256 < H) VecIO<TC, 8>::load(in + q * 256, v[q]);
  int splits = 1;
  long long stride = 0;
  if (plan.part_rows) {
    const CountedRows c(*rows.count, plan.tile_rows, plan.n_tiles, plan.kblocks, plan.planned, plan.part_rows, plan.pairs);
    splits = c.splits;
    stride = (long long)c.stride * H;
  }
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    in += stride;
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
      if (c0 + q * 256 < H) {
        float u[8];
        VecIO<TC, 8>::load(in + q * 256, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[q][j] += u[j];
      }
  }
  TO* to = out + (long long)rows.row[r] * H + c0;
#pragma unroll
  for (int q = 0; q < kVecs; ++q)
    if (c0 + q * 256 < H) {
      if (failed) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[q][j] = __int_as_float(0x7fc00000);
      }
      VecIO<TO, 8>::store(to + q * 256, v[q]);
    }
}

// ---- host --------------------------------------------------------------------------------------------------
// What the forward leaves: the rows that name a token, their activations, an fp32 weight in bf16, the groups' statistics and the
// rows', e (only for a backward)
struct ScoreSaved {
  size_t wb, ab, count, row, token, score, stats, correct, e, total;
  long long ldV;
  int groups;
};
static ScoreSaved score_saved(long long N, long long H, long long V, int w_dtype, bool keep) {
  ScoreSaved L;
  L.ldV = (V + 7) & ~7LL;
  L.groups = (int)((V + EPI_COLS - 1) / EPI_COLS);
  size_t o = 0;
  L.wb = o;      o += w_dtype == HAWK_F32 ? up256((size_t)V * H * 2) : 0;
  L.ab = o;      o += up256((size_t)N * H * 2);
  L.count = o;   o += 256;
  L.row = o;     o += up256((size_t)N * 4);
  L.token = o;   o += up256((size_t)N * 8);
  L.score = o;   o += up256((size_t)N * L.groups * sizeof(float4));
  L.stats = o;   o += up256((size_t)N * sizeof(float2));
  L.correct = o; o += up256((size_t)N * 4);
  L.e = o;       o += keep ? up256((size_t)N * L.ldV * 2) : 0;
  L.total = o;
  return L;
}
static ScoreRows score_rows(const ScoreSaved& S, const void* saved) {
  auto* p = const_cast<unsigned char*>(static_cast<const unsigned char*>(saved));
  return ScoreRows{reinterpret_cast<int*>(p + S.count), reinterpret_cast<int*>(p + S.row), reinterpret_cast<int64_t*>(p + S.token)};
}
struct ScoreScratch {
  size_t dx, row_scale, act, partial, total;
};
// d act of up to this many rows leaves partial sums in fp32 over splits of K that its kernel plans for the rows that are named (3108 rows
// of 2048, V32000, nine of ten left out: backward 386 -> 143 us, half 519 -> 393).  Of more rows the product leaves what it is asked for, as
// the sums cost where many are named and the splits are fewer in any case: 32760 rows of 2048, d x and d act, planned so / without,
// all named 3654 / 3558 us, a quarter 1022 / 1002, a tenth 532 / 577, a hundredth 206 / 491.  Just above the border the loss is largest: 8193
// rows, all 925 / 907, a quarter 388 / 376, a tenth 157 / 347
constexpr int64_t kPlannedRows = 8192;
static int da_part_rows(int64_t N, const GradPlan& plan) {  // 0: no partial sums
  const int64_t rows = plan.splits * ((N + 31) / 32 * 32);
  return (N <= kPlannedRows || plan.splits > 1) && rows < (1LL << 31) ? (int)rows : 0;
}
static ScoreScratch score_scratch(long long N, long long H, long long V, bool want_dw, bool want_da) {
  ScoreScratch L;
  size_t o = 0, part = 0;
  L.dx = o;      o += up256((size_t)room_rows(N) * ((V + 7) & ~7LL) * 2);
  L.row_scale = o; o += up256((size_t)N * 4);
  L.act = o;     o += want_dw ? up256((size_t)room_rows(N) * H * 2) : 0;
  if (want_da) part = (size_t)std::max<int64_t>(N, da_part_rows(N, plan_grad(N, H, V))) * H * 4;  // its compact rows, in fp32 at most
  const long long splits = want_dw ? plan_grad(V, H, room_rows(N)).splits : 1;
  if (splits > 1) part = std::max<size_t>(part, (size_t)splits * V * H * 4);
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
  (void)a_dtype;
  return score_saved(N, H, V, w_dtype, want_grad != 0).total;
}

extern "C" size_t hawk_linear_logprobs_scratch_bytes(int64_t N, int64_t H, int64_t V, int a_dtype, int want_dw, int want_da) {
  if (N < 1 || H < 1 || V < 1) return 0;
  (void)a_dtype;
  return score_scratch(N, H, V, want_dw != 0, want_da != 0).total;
}

// the forward (want_dw = want_da = 0): the rows (counted before in long lists) and casts, the GEMM and the reduction; the backward:
// d x, d weight's GEMM and, where K is split, the sum, d act's GEMM and the scatter, which looks at the status word, too
extern "C" int hawk_linear_logprobs_kernels(int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int want_dw, int want_da) {
  (void)w_dtype;
  (void)a_dtype;
  if (N < 1 || H < 1 || V < 1) return 0;
  if (!want_dw && !want_da) return N > kCountedRows ? 4 : 3;
  return 1 + (want_da ? 2 : 1) + (want_dw ? (plan_grad(V, H, room_rows(N)).splits > 1 ? 2 : 1) : 0);
}

extern "C" int hawk_linear_logprobs(const void* weight, const void* act, const int64_t* tokens, float* logprob, float* entropy, void* saved,
                                    size_t saved_bytes, int64_t N, int64_t H, int64_t V, int w_dtype, int a_dtype, int want_grad,
                                    int* status, void* stream) {
  HAWK_REQUIRE(weight && act && tokens && logprob && entropy && status, HAWK_ERR_NULL);
  int rc = check_score(N, H, V, w_dtype, a_dtype);
  if (rc != HAWK_OK) return rc;
  const ScoreSaved S = score_saved(N, H, V, w_dtype, want_grad != 0);
  HAWK_REQUIRE(saved && saved_bytes >= S.total, HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(aligned(saved, 256) && aligned(weight, 16) && aligned(act, 16) && aligned(tokens, 8) && aligned(logprob, 4) &&
                   aligned(entropy, 4),
               HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* sv = static_cast<unsigned char*>(saved);
  const ScoreRows rows = score_rows(S, saved);
  auto* ab = reinterpret_cast<__nv_bfloat16*>(sv + S.ab);
  auto* wcopy = reinterpret_cast<__nv_bfloat16*>(sv + S.wb);
  const auto* wb = w_dtype == HAWK_F32 ? wcopy : static_cast<const __nv_bfloat16*>(weight);
  auto* correct = reinterpret_cast<float*>(sv + S.correct);
  const int per = (int)std::min<int64_t>(256, std::max<int64_t>(8, (N + 4 * sm_count() - 1) / (4 * sm_count())));  // 4 blocks to an SM
  const int64_t row_blocks = (N + per - 1) / per, wvec = w_dtype == HAWK_F32 ? V * H / 8 : 0, blocks = row_blocks + (wvec + 1023) / 1024;
  HAWK_REQUIRE(blocks < (1LL << 31) && (int64_t)per * H < (1LL << 31), HAWK_ERR_SHAPE);
  const auto* wf = static_cast<const float*>(weight);
  int* counts = nullptr;
  if (N > kCountedRows) {
    counts = reinterpret_cast<int*>(sv + S.score);  // free until the GEMM writes it, and 16 bytes to a row at least
    score_count_kernel<<<(unsigned)row_blocks, 256, 0, st>>>(tokens, counts, (int)N, per);
    rc = launch_status();
    if (rc != HAWK_OK) return rc;
  }
  if (a_dtype == HAWK_F32)
    score_prepare_kernel<<<(unsigned)blocks, 256, 0, st>>>(tokens, static_cast<const float*>(act), rows, ab, correct, logprob, entropy, (int)N,
                                                           (int)H, per, (int)row_blocks, counts, wf, wcopy, wvec);
  else
    score_prepare_kernel<<<(unsigned)blocks, 256, 0, st>>>(tokens, static_cast<const __nv_bfloat16*>(act), rows, ab, correct, logprob, entropy,
                                                           (int)N, (int)H, per, (int)row_blocks, counts, wf, wcopy, wvec);
  rc = launch_status();
  if (rc != HAWK_OK) return rc;
  EpiParams ep{};
  ep.score = reinterpret_cast<float4*>(sv + S.score);
  ep.groups = S.groups;
  ep.correct = correct;
  ep.labels = reinterpret_cast<const long long*>(rows.token);
  ep.count = rows.count;
  if (want_grad)
    rc = launch_gemm<EPI_SCORE_KEEP, 1, false, false>(ab, H, wb, H, sv + S.e, false, S.ldV, (int)N, (int)V, (int)H, 1, ep, status, st);
  else
    rc = launch_gemm<EPI_SCORE, 1, false, false>(ab, H, wb, H, nullptr, false, S.ldV, (int)N, (int)V, (int)H, 1, ep, status, st);
  if (rc != HAWK_OK) return rc;
  score_reduce_kernel<<<(unsigned)((N + 7) / 8), 256, 0, st>>>(ep.score, correct, rows, wb, ab, logprob, entropy,
                                                               reinterpret_cast<float2*>(sv + S.stats), (int)H, (int)V, S.groups,
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
  const ScoreSaved S = score_saved(N, H, V, w_dtype, true);
  const ScoreScratch L = score_scratch(N, H, V, dweight != nullptr, dact != nullptr);
  HAWK_REQUIRE(saved && saved_bytes >= S.total && scratch && scratch_bytes >= L.total, HAWK_ERR_WORKSPACE);
  HAWK_REQUIRE(N * (H / 256 + 1) < (1LL << 31) && whole_blocks(N) * (V / (8 * kDxShare) + 2) < (1LL << 31), HAWK_ERR_SHAPE);
  HAWK_REQUIRE(aligned(saved, 256) && aligned(scratch, 256) && aligned(dweight, 16) && aligned(dact, 16) && aligned(weight, 16) &&
                   aligned(act, 16) && aligned(tokens, 8) && aligned(logprob, 4) && aligned(entropy, 4) && aligned(g_logprob, 4) &&
                   aligned(g_entropy, 4),
               HAWK_ERR_ALIGN);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto* sv = static_cast<const unsigned char*>(saved);
  auto* sc = static_cast<unsigned char*>(scratch);
  const auto* wb = static_cast<const __nv_bfloat16*>(w_dtype == HAWK_F32 ? static_cast<const void*>(sv + S.wb) : weight);
  const auto* ab = reinterpret_cast<const __nv_bfloat16*>(sv + S.ab);
  const ScoreRows rows = score_rows(S, saved);
  auto* dx = reinterpret_cast<__nv_bfloat16*>(sc + L.dx);
  auto* row_scale = reinterpret_cast<float*>(sc + L.row_scale);
  auto* dw_act = reinterpret_cast<__nv_bfloat16*>(sc + L.act);
  auto* part = reinterpret_cast<float*>(sc + L.partial);
  const int64_t shares = ((V + 7) / 8 + kDxShare - 1) / kDxShare;
  const int64_t dx_blocks = whole_blocks(N) * shares, act_blocks = dweight ? whole_blocks(N) / 8 : 0;
  score_dx_kernel<<<(unsigned)(dx_blocks + act_blocks), kDxThreads, 0, st>>>(reinterpret_cast<const __half*>(sv + S.e),
                                                                 reinterpret_cast<const float4*>(sv + S.score),
                                                                 reinterpret_cast<const float2*>(sv + S.stats), logprob, entropy, rows,
                                                                 g_logprob, g_entropy, dx, row_scale, ab, dw_act, S.ldV, (int)V, (int)H,
                                                                 S.groups, (uint32_t)shares, (uint32_t)dx_blocks);
  rc = launch_status();
  if (rc != HAWK_OK) return rc;
  if (dweight) {  // d weight [V,H] = dx^T . act [N,H]: A and B MN-major (the compact rows of dx and their activations are the K index)
    rc = grad_gemm<true, true>(dx, S.ldV, dw_act, H, dweight, dw_dtype, nullptr, (int)V, (int)H, (int)room_rows(N), rows.count + 1, part, status, st);
    if (rc != HAWK_OK) return rc;
  }
  if (dact) {  // d act [N,H] = dx [N,V] . W [V,H]: A K-major, B MN-major (W's rows are the K index); compact rows
    const GradPlan plan = plan_grad(N, H, V);
    EpiParams ep{};
    ep.part_rows = da_part_rows(N, plan);
    const int splits = ep.part_rows ? plan.splits : 1;
    ep.out_bf16 = !ep.part_rows && da_dtype == HAWK_BF16;
    ep.count = rows.count;
    ep.row_scale = row_scale;
    rc = plan.mh == 2 ? launch_gemm<EPI_OUT, 2, false, true>(dx, S.ldV, wb, H, part, !ep.out_bf16, H, (int)N, (int)H, (int)V, splits, ep, status, st)
                      : launch_gemm<EPI_OUT, 1, false, true>(dx, S.ldV, wb, H, part, !ep.out_bf16, H, (int)N, (int)H, (int)V, splits, ep, status, st);
    if (rc != HAWK_OK) return rc;
    const int cols = ep.part_rows ? 256 : 1024;
    const int64_t chunks = (H + cols - 1) / cols, units = N * chunks;
    const unsigned blocks = (unsigned)((units + 7) / 8);
    const ScatterPlan how{BM * plan.mh, (int)((H + BN - 1) / BN), (int)((V + BK - 1) / BK), plan.splits, ep.part_rows, sm_count() / 2};
    const auto scatter = [&](auto kern, auto* from, auto* to) {
      kern<<<blocks, 256, 0, st>>>(from, how, tokens, rows, to, (uint32_t)units, (uint32_t)chunks, (int)H, status, dweight, dw_dtype == HAWK_BF16);
    };
    using bf16 = __nv_bfloat16;
    if (ep.out_bf16) scatter(score_scatter_kernel<bf16, bf16, 4>, reinterpret_cast<bf16*>(part), static_cast<bf16*>(dact));
    else if (da_dtype == HAWK_BF16) scatter(score_scatter_kernel<float, bf16, 1>, part, static_cast<bf16*>(dact));
    else if (ep.part_rows) scatter(score_scatter_kernel<float, float, 1>, part, static_cast<float*>(dact));
    else scatter(score_scatter_kernel<float, float, 4>, part, static_cast<float*>(dact));
    return launch_status();
  }
  ce_poison_on_abort_kernel<<<1, 1, 0, st>>>(status, dweight, dw_dtype == HAWK_BF16, nullptr, 0);
  return launch_status();
}
