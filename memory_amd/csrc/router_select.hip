// Selection of chapters as a mixture of experts routes: scores, a bias for balance, groups, top-k.
//   s_c  = softmax of the logits over the selectable chapters c >= S, or sigmoid(z_c)
//   key  = s_c + b_c  (b: the balance bias, which steers the selection and nothing else); a masked logit
//          (-inf) has key -inf, NaN sorts above everything (as in torch)
//   groups: the C - S chapters in G runs of equal length; a group's score is the sum of its `best` largest
//          keys, the top_groups groups with the largest scores stay (ties: lower group)
//   the k largest keys of the groups that stay, keys descending, equal keys by ascending chapter
//   w = scale * s / max(sum of the selected s, 1e-12), or scale * s
// Keys are compared in f64: neighbours of a few thousand scores differ by less than f32 resolves.  Without a bias
// a key grows with its logit, and the logits themselves are compared.  (A group's score adds two keys and needs
// them.)
//
// Backward, ds_j = scale (dw_j - [sum > 1e-12] (sum_i dw_i s_i) / D) / D with D = max(sum, 1e-12), or scale dw_j:
//   sigmoid: dz_j = ds_j s_j (1 - s_j) on the selected, 0 elsewhere
//   softmax: dz_c = s_c (ds_c [selected] - sum_j ds_j s_j); the sum is 0 for renormalised weights.
//
// One workgroup per row, every key of the row in LDS as an ordered 64-bit integer: the k-th largest by eight
// passes over bytes, then the selected in order.
#include <algorithm>

#include "moc_common.h"

namespace moc {
namespace {

constexpr int kSelThreads = 256;
constexpr int kSelMaxK = 1024;
constexpr int kSelMaxG = 1024;
constexpr int kSelMaxC = 16384;

// doubles (and NaN) to integers of the same order; 0 stays free for "not selectable"
__device__ __forceinline__ uint64_t key64(double v) {
  if (v != v) return ~0ull;
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);   // (-0 and 0 are equal)
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double key64_inv(uint64_t k) {
  if (k == ~0ull) return __builtin_nan("");
  return __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}

struct SelArgs {
  const float *z, *bias;
  int64_t R, ldz;
  int n, S, k, sigmoid, G, top, best, renorm;
  float scale;
  int32_t* idx;
  float *w, *s_sel, *row_stats;
};

template <int NT> __device__ __forceinline__ double blk_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}

__global__ __launch_bounds__(kSelThreads) void router_select_kernel(SelArgs a) {
  constexpr int NT = kSelThreads;
  extern __shared__ char lds[];
  uint64_t* keys = (uint64_t*)lds;                       // [n]
  uint64_t* gkey = keys + a.n;                           // [G]
  uint64_t* sel_key = gkey + a.G;                        // [k]
  float* sel_s = (float*)(sel_key + a.k);                // [k]
  int32_t* sel_id = (int32_t*)(sel_s + a.k);             // [k]
  uint8_t* keep = (uint8_t*)(sel_id + a.k);              // [G]
  __shared__ double red[NT / 64];
  __shared__ int hist[256];
  __shared__ int pick[4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* z = a.z + r * a.ldz + a.S;
  const float* b = a.bias ? a.bias + a.S : nullptr;
  const int n = a.n, per = n / a.G;
  const bool by_logit = !b && (a.G == a.top || a.best == 1);

  double m = 0.0, Z = 1.0;
  float mf = -INFINITY;
  if (!a.sigmoid) {
    bool nan = false;
    for (int c = tid; c < n; c += NT) {
      nan |= z[c] != z[c];
      mf = fmaxf(mf, z[c]);
    }
    mf = wave_max(mf);
    __syncthreads();
    if (lane == 0) red[wave] = mf;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) mf = fmaxf(mf, (float)red[i]);
    m = mf;
    double s = 0.0;
    for (int c = tid; c < n; c += NT) s += exp((double)z[c] - m);   // (every logit -inf: NaN, as the formula)
    Z = blk_sum<NT>(s, red);
    if (a.row_stats && tid == 0) {
      a.row_stats[2 * r] = mf;
      a.row_stats[2 * r + 1] = (float)Z;
    }
  }
  auto score = [&](float v) -> double {
    return a.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : exp((double)v - m) / Z;
  };
  for (int c = tid; c < n; c += NT) {
    const float v = z[c];
    const double key = by_logit || v == -INFINITY ? (double)v : score(v) + (b ? (double)b[c] : 0.0);
    keys[c] = key64(key);
  }
  __syncthreads();
  if (a.top < a.G) {
    // a group's best keys (their ordered integers pick them, their values are added), one wave per group
    for (int g = wave; g < a.G; g += NT / 64) {
      uint64_t k1 = 0, k2 = 0;   // the lane's two largest
      for (int i = lane; i < per; i += 64) {
        const uint64_t v = keys[g * per + i];
        if (v > k1) { k2 = k1; k1 = v; }
        else if (v > k2) k2 = v;
      }
      for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t p1 = __shfl_xor((unsigned long long)k1, o, 64), p2 = __shfl_xor((unsigned long long)k2, o, 64);
        const uint64_t lo = min(k1, p1);
        k1 = max(k1, p1);
        k2 = max(lo, max(k2, p2));
      }
      if (lane == 0) {
        const double v1 = key64_inv(k1), v2 = key64_inv(k2);
        // (a masked second key leaves the first alone)
        gkey[g] = a.best == 1 || k2 == 0 || v2 == -INFINITY ? key64(v1) : key64(v1 + v2);
      }
    }
    __syncthreads();
    for (int g = tid; g < a.G; g += NT) {
      int rank = 0;
      for (int j = 0; j < a.G; ++j) rank += gkey[j] > gkey[g] || (gkey[j] == gkey[g] && j < g);
      keep[g] = rank < a.top;
    }
    __syncthreads();
    for (int c = tid; c < n; c += NT)
      if (!keep[c / per]) keys[c] = 0;
    __syncthreads();
  }
  // the k-th largest key, byte by byte from the top
  uint64_t prefix = 0;
  int want = a.k;   // the want-th largest among the keys that share the prefix
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    __syncthreads();
    for (int c = tid; c < n; c += NT) {
      const uint64_t v = keys[c];
      if (shift == 56 || (v >> (shift + 8)) == prefix) atomicAdd(&hist[(int)((v >> shift) & 255)], 1);
    }
    __syncthreads();
    if (wave == 0) {
      int cnt[4], mine = 0;
      for (int i = 0; i < 4; ++i) { cnt[i] = hist[4 * lane + i]; mine += cnt[i]; }
      int above = mine;   // counts in the bins of this lane and higher lanes
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_down(above, o, 64);
        if (lane + o < 64) above += t;
      }
      above -= mine;
      for (int i = 3; i >= 0; --i) {
        if (above < want && above + cnt[i] >= want) {
          pick[0] = 4 * lane + i;
          pick[1] = want - above;
        }
        above += cnt[i];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint64_t)pick[0];
    want = pick[1];
    __syncthreads();
  }
  // every key above the k-th, and of those equal to it the `want` with the lowest ids
  if (tid == 0) pick[2] = 0;
  __syncthreads();
  for (int c = tid; c < n; c += NT)
    if (keys[c] > prefix) {
      const int p = atomicAdd(&pick[2], 1);
      sel_key[p] = keys[c];
      sel_id[p] = c;
    }
  __syncthreads();
  if (wave == 0) {
    int at = a.k - want;
    for (int c0 = 0; c0 < n && at < a.k; c0 += 64) {
      const bool eq = c0 + lane < n && keys[c0 + lane] == prefix;
      const uint64_t mask = __ballot(eq);
      const int p = at + __popcll(mask & ((1ull << lane) - 1));
      if (eq && p < a.k) {
        sel_key[p] = prefix;
        sel_id[p] = c0 + lane;
      }
      at += __popcll(mask);
    }
  }
  __syncthreads();
  // their order and scores
  double mine[(kSelMaxK + NT - 1) / NT];
  int rank[(kSelMaxK + NT - 1) / NT];
  double sum = 0.0;
#pragma unroll
  for (int q = 0; q < (kSelMaxK + NT - 1) / NT; ++q) {
    const int i = tid + NT * q;
    if (i < a.k) {
      const uint64_t ki = sel_key[i];
      const int32_t ii = sel_id[i];
      int rk = 0;
      for (int j = 0; j < a.k; ++j) rk += sel_key[j] > ki || (sel_key[j] == ki && sel_id[j] < ii);
      rank[q] = rk;
      mine[q] = score(z[ii]);
      sum += mine[q];
    }
  }
  sum = blk_sum<NT>(sum, red);
  const double D = a.renorm ? (sum > 1e-12 ? sum : (sum == sum ? 1e-12 : sum)) : 1.0;
#pragma unroll
  for (int q = 0; q < (kSelMaxK + NT - 1) / NT; ++q) {
    const int i = tid + NT * q;
    if (i < a.k) {
      const int64_t o = r * a.k + rank[q];
      a.idx[o] = sel_id[i] + a.S;
      a.w[o] = (float)((double)a.scale * mine[q] / D);
      if (a.s_sel) a.s_sel[o] = (float)mine[q];
    }
  }
}

struct SelBwdArgs {
  const float *z, *dw, *s_sel, *row_stats;
  const int32_t* idx;
  int64_t R, ldz, C;
  int S, k, sigmoid, renorm;
  float scale;
  float* dz;
};

// One workgroup per row: the row of zeros (or of the softmax's dense part), then the selected entries.
__global__ __launch_bounds__(kSelThreads) void router_select_bwd_kernel(SelBwdArgs a) {
  constexpr int NT = kSelThreads;
  __shared__ double red[NT / 64];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  double sum = 0.0, dot = 0.0;
  for (int j = tid; j < a.k; j += NT) {
    const double s = a.s_sel[r * a.k + j];
    sum += s;
    dot += s * (double)a.dw[r * a.k + j];
  }
  sum = blk_sum<NT>(sum, red);
  dot = blk_sum<NT>(dot, red);
  const bool clamped = !(sum > 1e-12);
  const double D = a.renorm ? (clamped && sum == sum ? 1e-12 : sum) : 1.0;
  // sum_j ds_j s_j of the softmax
  const double t = a.sigmoid || (a.renorm && !clamped) ? 0.0 : (double)a.scale * dot / D;
  auto ds = [&](int j) {
    const double g = a.dw[r * a.k + j];
    return (double)a.scale * (a.renorm && !clamped ? (g - dot / D) / D : g / D);
  };
  float* row = a.dz + r * a.C;
  if (t == 0.0) {
    for (int64_t c = tid; c < a.C; c += NT) row[c] = 0.f;
  } else {
    const float m = a.row_stats[2 * r], Z = a.row_stats[2 * r + 1];
    const float ft = (float)t;
    for (int64_t c = tid; c < a.C; c += NT) row[c] = c < a.S ? 0.f : -expf(a.z[r * a.ldz + c] - m) / Z * ft;
  }
  __syncthreads();
  for (int j = tid; j < a.k; j += NT) {
    const double s = a.s_sel[r * a.k + j];
    row[a.idx[r * a.k + j]] = (float)(a.sigmoid ? ds(j) * s * (1.0 - s) : s * (ds(j) - t));
  }
}

// counts[c] += selections of c; one thread per selection, integer adds.
__global__ __launch_bounds__(256) void select_count_kernel(const int32_t* __restrict__ idx, int64_t n, int64_t C,
                                                           int32_t* __restrict__ counts) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int32_t c = idx[i];
  if (c >= 0 && c < C) atomicAdd(&counts[c], 1);
}
__global__ __launch_bounds__(256) void select_clear_kernel(int32_t* __restrict__ counts, int64_t C) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < C) counts[i] = 0;
}
// bias[c] += rate * sign(mean count - count[c]) for the routed chapters c >= S (mean over them; compared as
// integers: count * (C - S) against the total).
__global__ __launch_bounds__(1024) void balance_update_kernel(const int32_t* __restrict__ counts, int64_t C, int S, float rate,
                                                              float* __restrict__ bias) {
  __shared__ long long part[16];
  long long s = 0;
  for (int64_t c = S + threadIdx.x; c < C; c += 1024) s += counts[c];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  long long total = 0;
  for (int i = 0; i < 16; ++i) total += part[i];
  for (int64_t c = S + threadIdx.x; c < C; c += 1024) {
    const long long v = (long long)counts[c] * (C - S);
    bias[c] += v < total ? rate : v > total ? -rate : 0.f;
  }
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" {

int moc_router_select(const float* logits, int64_t ldz, int64_t R, int64_t C, int S, int k, int score, const float* bias,
                      int groups, int top_groups, int group_best, int renormalize, float scale, int32_t* idx, float* w,
                      float* s_sel, float* row_stats, hipStream_t stream) {
  MOC_REQUIRE(R >= 0 && C > 0 && C <= kSelMaxC, MOC_ERR_UNSUPPORTED, "moc_router_select: R=%lld C=%lld (C up to %d)",
              (long long)R, (long long)C, kSelMaxC);
  MOC_REQUIRE(R < ((int64_t)1 << 31), MOC_ERR_UNSUPPORTED, "moc_router_select: R=%lld", (long long)R);
  MOC_REQUIRE(S >= 0 && S < C, MOC_ERR_ARG, "moc_router_select: exclude_prefix_chapters %d of %lld", S, (long long)C);
  MOC_REQUIRE(score == MOC_SCORE_SOFTMAX || score == MOC_SCORE_SIGMOID, MOC_ERR_ARG, "moc_router_select: score %d", score);
  const int64_t n = C - S;
  MOC_REQUIRE(groups >= 1 && groups <= kSelMaxG && n % groups == 0 && top_groups >= 1 && top_groups <= groups, MOC_ERR_ARG,
              "moc_router_select: %lld chapters in %d groups, %d kept", (long long)n, groups, top_groups);
  MOC_REQUIRE(group_best == 1 || (group_best == 2 && n / groups >= 2), MOC_ERR_ARG, "moc_router_select: group_best %d",
              group_best);
  MOC_REQUIRE(k >= 1 && k <= kSelMaxK && k <= top_groups * (n / groups), MOC_ERR_ARG,
              "moc_router_select: k=%d of %lld selectable (up to %d)", k, (long long)(top_groups * (n / groups)), kSelMaxK);
  MOC_REQUIRE(ldz >= C, MOC_ERR_ARG, "moc_router_select: row stride %lld", (long long)ldz);
  if (R == 0) return MOC_OK;
  MOC_REQUIRE(logits && idx && w, MOC_ERR_ARG, "moc_router_select: null pointer");
  SelArgs a{logits, bias, R, ldz, (int)n, S, k, score == MOC_SCORE_SIGMOID, groups, top_groups, group_best,
            renormalize != 0, scale, idx, w, s_sel, row_stats};
  const size_t lds = (size_t)n * 8 + (size_t)groups * 9 + (size_t)k * 16;
  MOC_HIP(hipFuncSetAttribute((const void*)router_select_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(router_select_kernel, dim3((unsigned)R), dim3(kSelThreads), lds, stream, a);
  return check_launch("router_select_kernel");
}

int moc_router_select_bwd(const float* logits, int64_t ldz, const int32_t* idx, const float* s_sel, const float* row_stats,
                          const float* dw, int64_t R, int64_t C, int S, int k, int score, int renormalize, float scale,
                          float* dlogits, hipStream_t stream) {
  MOC_REQUIRE(R >= 0 && R < ((int64_t)1 << 31) && C > 0 && C <= kSelMaxC && S >= 0 && S < C && k >= 1 && k <= kSelMaxK &&
                  k <= C - S && ldz >= C,
              MOC_ERR_ARG, "moc_router_select_bwd: R=%lld C=%lld S=%d k=%d", (long long)R, (long long)C, S, k);
  MOC_REQUIRE(score == MOC_SCORE_SOFTMAX || score == MOC_SCORE_SIGMOID, MOC_ERR_ARG, "moc_router_select_bwd: score %d", score);
  if (R == 0) return MOC_OK;
  MOC_REQUIRE(logits && idx && s_sel && dw && dlogits && (score == MOC_SCORE_SIGMOID || row_stats), MOC_ERR_ARG,
              "moc_router_select_bwd: null pointer");
  SelBwdArgs a{logits, dw, s_sel, row_stats, idx, R, ldz, C, S, k, score == MOC_SCORE_SIGMOID, renormalize != 0, scale, dlogits};
  hipLaunchKernelGGL(router_select_bwd_kernel, dim3((unsigned)R), dim3(kSelThreads), 0, stream, a);
  return check_launch("router_select_bwd_kernel");
}

int moc_router_balance(const int32_t* idx, int64_t n, int64_t C, int S, float rate, int32_t* counts, float* bias,
                       hipStream_t stream) {
  MOC_REQUIRE(n >= 0 && n < ((int64_t)1 << 38) && C > 0 && C <= kSelMaxC && S >= 0 && S < C, MOC_ERR_ARG,
              "moc_router_balance: n=%lld C=%lld S=%d", (long long)n, (long long)C, S);
  MOC_REQUIRE(counts && bias && (idx || n == 0), MOC_ERR_ARG, "moc_router_balance: null pointer");
  hipLaunchKernelGGL(select_clear_kernel, dim3((unsigned)((C + 255) / 256)), dim3(256), 0, stream, counts, C);
  if (n > 0)
    hipLaunchKernelGGL(select_count_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, idx, n, C, counts);
  hipLaunchKernelGGL(balance_update_kernel, dim3(1), dim3(1024), 0, stream, counts, C, S, rate, bias);
  return check_launch("balance_update_kernel");
}

}  // extern "C"
