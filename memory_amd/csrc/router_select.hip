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
//   softmax: dz_c = s_c (ds_c [selected] - sum_j ds_j s_j); the sum is 0 for renormalised weights.  ds_c - sum_j ds_j s_j is
//   formed as ds_c (1 - sum_j s_j) + sum_j (ds_c - ds_j) s_j with the mass that is not selected from the forward.
//
// Rows are held in registers by one wave, or by four where there are few; what does not fit them, or cannot be decided
// from f32 keys with a few exact ones, goes to a workgroup with every exact key in LDS.
#include <cfloat>

#include <algorithm>

#include "moc_common.h"

namespace moc {
namespace {

constexpr int kSelThreads = 256;
constexpr int kSelMaxK = 1024;
constexpr int kSelMaxG = 1024;
constexpr int kSelMaxC = 16384;
// Up to which four waves take a row, one behind it.  Sigmoid with a bias, four waves / one, us: 4,097 chapters in 8 groups, 16
// selected: 7.2 / 10.3 for 64 rows, 10.9 / 11.1 for 1,024, 19.1 / 14.4 for 2,048; 64 selected: 10.5 / 27.6, 16.0 / 28.9,
// 27.6 / 33.5; 257 chapters, 8 selected: 5.2 / 5.6, 7.3 / 5.8, 11.6 / 6.5.
constexpr int64_t kSelFewRows = 1024;

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

// the softmax's maximum, sum, and the part of its mass that is not selected (sel: the selected's part of the sum)
__device__ __forceinline__ void put_row_stats(const SelArgs& a, int64_t r, float m, double Z, double sel) {
  a.row_stats[3 * r] = m;
  a.row_stats[3 * r + 1] = (float)Z;
  a.row_stats[3 * r + 2] = (float)((Z > sel ? Z - sel : 0.0) / Z);
}

// a chapter's exact score (m, Z: the row's maximum and sum for softmax); one exponential and one quotient in the code
__device__ __forceinline__ double score64(float x, int sigmoid, float m, double Z) {
  const double e = exp(sigmoid ? -(double)x : (double)x - (double)m);
  return (sigmoid ? 1.0 : e) / (sigmoid ? 1.0 + e : Z);
}

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

// One row on a workgroup, any shape: every key of the row in LDS as an ordered 64-bit integer, the k-th largest by
// eight passes over bytes, then the selected in order.  Every thread calls it.
__device__ __forceinline__ void select_row(const SelArgs& a, int64_t r, char* lds) {
  constexpr int NT = kSelThreads;
  uint64_t* keys = (uint64_t*)lds;                       // [n]
  uint64_t* gkey = keys + a.n;                           // [G]
  uint64_t* sel_key = gkey + a.G;                        // [k]
  float* sel_s = (float*)(sel_key + a.k);                // [k]
  int32_t* sel_id = (int32_t*)(sel_s + a.k);             // [k]
  uint8_t* keep = (uint8_t*)(sel_id + a.k);              // [G]
  __shared__ double red[NT / 64];
  __shared__ int hist[256];
  __shared__ int pick[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* z = a.z + r * a.ldz + a.S;
  const float* b = a.bias ? a.bias + a.S : nullptr;
  const int n = a.n, per = n / a.G;
  const bool by_logit = !b && (a.G == a.top || a.best == 1);

  double Z = 1.0;
  float mf = -INFINITY;
  if (!a.sigmoid) {
    for (int c = tid; c < n; c += NT) mf = fmaxf(mf, z[c]);
    mf = wave_max(mf);
    __syncthreads();
    if (lane == 0) red[wave] = mf;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) mf = fmaxf(mf, (float)red[i]);
    double s = 0.0;
    for (int c = tid; c < n; c += NT) s += exp((double)z[c] - (double)mf);   // (every logit -inf: NaN, as the formula)
    Z = blk_sum<NT>(s, red);
  }
  auto score = [&](float v) { return score64(v, a.sigmoid, mf, Z); };
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
  // their order, and scores and weights in that order (the list's own order is not fixed, a sum over it would not be)
  int32_t* id_at = (int32_t*)keys;   // (the keys are done)
  for (int i = tid; i < a.k; i += NT) {
    const uint64_t ki = sel_key[i];
    const int32_t ii = sel_id[i];
    int rk = 0;
    for (int j = 0; j < a.k; ++j) rk += sel_key[j] > ki || (sel_key[j] == ki && sel_id[j] < ii);
    sel_s[rk] = (float)score(z[ii]);
    id_at[rk] = ii;
  }
  __syncthreads();
  double sum = 0.0;
  for (int i = tid; i < a.k; i += NT) sum += (double)sel_s[i];
  sum = blk_sum<NT>(sum, red);
  if (a.row_stats) {
    double e = 0.0;
    for (int i = tid; i < a.k; i += NT) e += exp((double)z[id_at[i]] - (double)mf);
    e = blk_sum<NT>(e, red);
    if (tid == 0) put_row_stats(a, r, mf, Z, e);
  }
  const double D = a.renorm ? (sum > 1e-12 ? sum : (sum == sum ? 1e-12 : sum)) : 1.0;
  for (int i = tid; i < a.k; i += NT) {
    const int64_t o = r * a.k + i;
    a.idx[o] = id_at[i] + a.S;
    a.w[o] = (float)((double)a.scale * (double)sel_s[i] / D);
    if (a.s_sel) a.s_sel[o] = sel_s[i];
  }
}

__global__ __launch_bounds__(kSelThreads) void router_select_kernel(SelArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  select_row(a, blockIdx.x, lds);
}

inline size_t select_row_lds(int n, int G, int k) { return (size_t)n * 8 + (size_t)G * 9 + (size_t)k * 16; }

// --------------------------------------------------------- rows in registers
// Rows of up to 64 * 72 (NW = 1) logits with k <= 64, and up to 64 groups: a team of NW waves holds the row's keys in
// registers as f32, E per lane, a group's chapters on lanes of its own (four consecutive ones per load).
//   1. keys in f32, within eps = kSelEps + 2^-24 |key| of the exact ones (the bound below); per lane the two largest, and four
//      maxima (NW = 1; one for NW = 4): 256 per row.
//   2. the groups' scores from the lanes' pairs; groups too close to the cut for these keys are scored again from
//      exact keys of their few largest.
//   3. t = a lower bound of the k-th largest of the 256 maxima: k keys are >= t.  With fewer live maxima than k, t by
//      bisection over the keys themselves.
//   4. every key >= t - 2 eps is a candidate (a few dozen; more than 256: select_row).  Only these are evaluated in
//      f64 and ranked exactly.
// Why no selected chapter is missed: k keys are >= t in f32, so the exact k-th largest is >= t - eps, and a chapter at
// or above that has an f32 key >= t - 2 eps.
// Error of the keys, with v_exp_f32 and v_rcp_f32 good to 1 ulp (2^-23).  Sigmoid: the argument z log2(e) is off by
// 1.5 |z| 2^-24 (its rounding and the constant's), which moves s by |z| s (1 - s) 1.5 2^-24 < 0.34 2^-24; the exponential moves
// it by s (1 - s) 2^-23 <= 0.5 2^-24; 1 + e and the reciprocal by 3 2^-24 s: below 4 2^-24 = 2^-22.  Softmax: the
// argument is off by 3 2^-24 |z - m| (difference, product, constant), which moves p by |z - m| p 3 2^-24 <= 1.2 2^-24 with
// p <= 1 (x e^-x <= 0.37), the exponential and 1 / Z by 2 2^-24 p each...: together below 2^-21.  The bias' addition
// rounds by 2^-24 |key|.
// The softmax's sum Z itself is off by (3 sum p |z - m| + 2) 2^-24 of it, below 20 2^-24 for up to 6,144 chapters (sum
// p |z - m| = y log(n / y) / (1 + y) <= 5.9, n chapters of one logit that together weigh y times the largest).  It moves all keys
// of a row to the same side, by p times it, below 9 2^-24; a difference of two keys, whose own errors are below 1 and
// 4 2^-24 where p is that large, stays within twice the bound above.
constexpr float kSelEps = 0x1p-21f;
constexpr double kSelSumErr = 0x1p-19;
constexpr int kSelMaxima = 256;
constexpr int kSelCand = 256;
constexpr int kSelTeamK = 64;

enum { kKeyLogit, kKeySigmoid, kKeySoftmax };

template <int NW> struct SelTeam {
  uint64_t key[kSelCand];
  int32_t id[kSelCand];
  float score[kSelCand];
  uint32_t maxima[kSelMaxima];
  float top[64 * NW][2];
  double part[NW];
  int count[NW];
};

__device__ __forceinline__ uint32_t key32(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key32_inv(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

// set bits of m below this lane
__device__ __forceinline__ int lanes_before(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}
// the value of lane i (the same i in every lane)
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); }
__device__ __forceinline__ float lane_value(float v, int i) { return __uint_as_float(lane_value(__float_as_uint(v), i)); }
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int i) {
  return (uint64_t)lane_value((uint32_t)(v >> 32), i) << 32 | lane_value((uint32_t)v, i);
}
// cross-lane steps of a wave reduction by DPP and row permutes, without LDS: step 0 .. 5 pairs lanes 1, 2, 4 (half
// rows mirrored), 8 (rows mirrored), 16 and 32 apart
template <int kStep> __device__ __forceinline__ uint32_t lane_step(uint32_t v) {
  if constexpr (kStep < 4) {
    constexpr int kCtrl = kStep == 0 ? 0xB1 : kStep == 1 ? 0x4E : kStep == 2 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kCtrl, 0xf, 0xf, true);
  } else {
    uint32_t a = v, b = v;
    if constexpr (kStep == 4) asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    else asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    // one of the two holds the lane's own value, the other its partner's
    return (threadIdx.x & (kStep == 4 ? 16 : 32)) ? a : b;
  }
}
template <typename F> __device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, F f) {
  v = f(v, lane_step<0>(v));
  v = f(v, lane_step<1>(v));
  v = f(v, lane_step<2>(v));
  v = f(v, lane_step<3>(v));
  v = f(v, lane_step<4>(v));
  return f(v, lane_step<5>(v));
}
template <int kStep> __device__ __forceinline__ double lane_step64(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  return __longlong_as_double((long long)((uint64_t)lane_step<kStep>((uint32_t)(u >> 32)) << 32 | lane_step<kStep>((uint32_t)u)));
}
__device__ __forceinline__ double lanes_sum(double v) {
  v += lane_step64<0>(v);
  v += lane_step64<1>(v);
  v += lane_step64<2>(v);
  v += lane_step64<3>(v);
  v += lane_step64<4>(v);
  return v + lane_step64<5>(v);
}
__device__ __forceinline__ float lanes_max(float v) {
  return __uint_as_float(lanes_reduce(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}

template <int NW> __device__ __forceinline__ void team_sync() {
  if constexpr (NW == 1) wave_lds_sync();
  else __syncthreads();
}
template <int NW> __device__ __forceinline__ double team_sum(double v, SelTeam<NW>& sm, int wave) {
  v = lanes_sum(v);
  if constexpr (NW > 1) {
    team_sync<NW>();
    if ((threadIdx.x & 63) == 0) sm.part[wave] = v;
    team_sync<NW>();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += sm.part[i];
  }
  return v;
}
template <int NW> __device__ __forceinline__ float team_max(float v, SelTeam<NW>& sm, int wave) {
  v = lanes_max(v);
  if constexpr (NW > 1) {
    team_sync<NW>();
    if ((threadIdx.x & 63) == 0) sm.part[wave] = (double)v;
    team_sync<NW>();
#pragma unroll
    for (int i = 0; i < NW; ++i) v = fmaxf(v, (float)sm.part[i]);
  }
  return v;
}
template <int NW> __device__ __forceinline__ int team_add(int v, SelTeam<NW>& sm, int wave) {
  if constexpr (NW > 1) {
    team_sync<NW>();
    if ((threadIdx.x & 63) == 0) sm.count[wave] = v;
    team_sync<NW>();
    v = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += sm.count[i];
  }
  return v;
}

// bit 4 j + e: v[j][e] >= cut
template <int E> __device__ __forceinline__ void lane_bits(const float (&v)[E / 4][4], float cut, uint32_t (&bits)[(E + 31) / 32]) {
#pragma unroll
  for (int i = 0; i < (E + 31) / 32; ++i) bits[i] = 0;
#pragma unroll
  for (int j = 0; j < E / 4; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) bits[(4 * j + e) >> 5] |= (v[j][e] >= cut ? 1u : 0u) << ((4 * j + e) & 31);
}

// True where the row is done, false where select_row has to take it (the same in every lane of the team).
template <int NW, int E, int MODE>
__device__ __forceinline__ bool select_team(const SelArgs& a, int64_t r, SelTeam<NW>& sm, int tl) {
  constexpr int TL = 64 * NW, E4 = E / 4, Q = 4 / NW;
  const int lane = tl & 63, wave = tl >> 6;
  const bool grouped = a.top < a.G;
  const int Ge = grouped ? a.G : 1, per = a.n / Ge, lpg = TL / Ge;
  const int grp = tl / lpg, pos = tl - grp * lpg;
  const bool active = grp < Ge;
  const int mine = active ? per : 0;   // chapters of the lane's group
  const int c0 = active ? grp * per : 0;
  const float* z = a.z + r * a.ldz + a.S;
  const float* b = a.bias ? a.bias + a.S : nullptr;
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  // The lane's chapters of its group, four consecutive ones per load, in whatever is behind the group too; a load
  // that would pass the row's end takes the row's last four.  What is behind the group, or another load's, is dropped.
  const int last4 = a.n - 4 - c0;
  auto chapter = [&](int q) { return min(4 * (pos + lpg * (q >> 2)), last4) + (q & 3); };   // within the group
  auto load4 = [&](const float* base, int j) {
    return *reinterpret_cast<const f32x4u*>(reinterpret_cast<const char*>(base) + 4u * (uint32_t)(c0 + chapter(4 * j)));
  };
  float v[E4][4];
#pragma unroll
  for (int j = 0; j < E4; ++j) {
    const f32x4u t = load4(z, j);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[j][e] = t[e];
  }
  if (per != lpg * E || TL != Ge * lpg) {   // (the same in every lane)
#pragma unroll
    for (int j = 0; j < E4; ++j) {
      const int at = chapter(4 * j), from = 4 * (pos + lpg * j) - at, to = mine - at;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = e >= from && e < to ? v[j][e] : -INFINITY;
    }
  }
  // softmax statistics
  float m = -INFINITY;
  double Z = 1.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < E4; ++j) m = fmaxf(m, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
    m = team_max<NW>(m, sm, wave);
    if (!(m > -INFINITY && m < INFINITY)) return false;
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < E4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f((v[j][e] - m) * 1.4426950408889634f);
        s += (double)p;
        if constexpr (MODE == kKeySoftmax) v[j][e] = v[j][e] == -INFINITY ? -INFINITY : p;
      }
    Z = team_sum<NW>(s, sm, wave);
  }
  // keys
  if constexpr (MODE != kKeyLogit) {
    const float rz = MODE == kKeySoftmax ? (float)(1.0 / Z) : 1.f;
#pragma unroll
    for (int j = 0; j < E4; ++j) {
      float w[4] = {0.f, 0.f, 0.f, 0.f};
      if (b) {
        const f32x4u t = load4(b, j);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = t[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = v[j][e];
        float s;
        if constexpr (MODE == kKeySigmoid) s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
        else s = x * rz;
        v[j][e] = x == -INFINITY ? -INFINITY : s + w[e];
      }
    }
  }
  // the lane's maxima (NaN stays in them) and its two largest keys
  float mx[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    mx[e] = v[0][e];
#pragma unroll
    for (int j = 1; j < E4; ++j) mx[e] = fmax_fast(mx[e], v[j][e]);
  }
  float k1 = fmax_fast(fmax_fast(mx[0], mx[1]), fmax_fast(mx[2], mx[3]));
  const bool odd = !(k1 < INFINITY);   // NaN or infinity
  if (team_add<NW>(__popcll(__ballot(odd)), sm, wave) != 0) return false;
  uint64_t keep = ~0ull;
  if (grouped) {
    float k2 = -INFINITY;
    if (a.best == 2) {
      k1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < E4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          k2 = __builtin_amdgcn_fmed3f(k1, k2, v[j][e]);
          k1 = fmaxf(k1, v[j][e]);
        }
    }
    sm.top[tl][0] = k1;
    sm.top[tl][1] = k2;
    team_sync<NW>();
    // (every wave for itself) lane g: group g's score, its rank, and how clear the cut is
    float g1 = -INFINITY, g2 = -INFINITY;
    if (lane < Ge) {
      for (int i = 0; i < lpg; ++i) {
        const float t1 = sm.top[lane * lpg + i][0], t2 = sm.top[lane * lpg + i][1];
        g2 = fmaxf(__builtin_amdgcn_fmed3f(g1, g2, t1), t2);
        g1 = fmaxf(g1, t1);
      }
    }
    const float sc = a.best == 2 && g2 > -INFINITY ? g1 + g2 : g1;
    int rank = 0;
    for (int i = 0; i < Ge; ++i) {
      const float o = lane_value(sc, i);
      rank += o > sc || (o == sc && i < lane);
    }
    const bool in = lane < Ge;
    keep = __ballot(in && rank < a.top);
    if constexpr (MODE != kKeyLogit) {
      // groups whose score is within the errors of the last one kept and the first one dropped are scored again
      // from exact keys: of those, the best by (score, lower group) stay
      const float last = __shfl(sc, __builtin_ctzll(__ballot(in && rank == a.top - 1)), 64);
      const float first = __shfl(sc, __builtin_ctzll(__ballot(in && rank == a.top)), 64);
      // (the error of a score: two keys and their sum)
      float err = in && sc > -INFINITY ? 0x1p-24f * (fabsf(g1) + (g2 > -INFINITY ? fabsf(g2) : 0.f) + fabsf(sc)) : 0.f;
      err = 2.f * kSelEps + lanes_max(err);
      if (!(last - first > 2.f * err)) {
        if (!(first > -INFINITY)) return false;
        const uint64_t near = __ballot(in && sc >= first - 2.f * err && sc <= last + 2.f * err);
        const uint64_t sure = __ballot(in && sc > last + 2.f * err);
        uint64_t score = 0;   // lane g: group g's exact score, ordered
        float most = 0.f;     // and the largest of its chapters' scores in it
        for (uint64_t todo = near; todo; todo &= todo - 1) {
          const int g = __builtin_ctzll(todo);
          const float lo = __shfl(a.best == 2 ? g2 : g1, g, 64);
          const float cut = lo - 2.f * (kSelEps + 0x1p-24f * fabsf(lo));
          uint64_t e1 = 0, e2 = 0;   // the lane's two largest exact keys of the group
          float sg = 0.f;            // the largest score among the group's keys in question
          if (active && grp == g) {
            uint32_t bits[(E + 31) / 32];
            lane_bits<E>(v, fmaxf(cut, -FLT_MAX), bits);
#pragma unroll
            for (int i = 0; i < (E + 31) / 32; ++i)
              for (uint32_t w = bits[i]; w; w &= w - 1) {
                const int c = c0 + chapter(32 * i + __builtin_ctz(w));
                const double sc64 = score64(z[c], a.sigmoid, m, Z);
                const uint64_t k = key64(sc64 + (b ? (double)b[c] : 0.0));
                e2 = k > e1 ? e1 : k > e2 ? k : e2;
                e1 = k > e1 ? k : e1;
                if constexpr (MODE == kKeySoftmax) sg = fmaxf(sg, (float)sc64);
              }
          }
#pragma unroll
          for (int o = 32; o >= 1; o >>= 1) {
            const uint64_t p1 = __shfl_xor((unsigned long long)e1, o, 64), p2 = __shfl_xor((unsigned long long)e2, o, 64);
            const uint64_t low = min(e1, p1);
            e1 = max(e1, p1);
            e2 = max(low, max(e2, p2));
          }
          if constexpr (NW > 1) {
            team_sync<NW>();
            if (lane == 0) {
              sm.key[2 * wave] = e1;
              sm.key[2 * wave + 1] = e2;
            }
            team_sync<NW>();
            e1 = e2 = 0;
            for (int i = 0; i < 2 * NW; ++i) {
              const uint64_t k = sm.key[i];
              e2 = k > e1 ? e1 : k > e2 ? k : e2;
              e1 = k > e1 ? k : e1;
            }
          }
          const double s1 = key64_inv(e1);
          if (lane == g) score = a.best == 1 || e2 == 0 ? e1 : key64(s1 + key64_inv(e2));
          if constexpr (MODE == kKeySoftmax) {
            sg = team_max<NW>(sg, sm, wave);
            if (lane == g) most = sg;
          }
        }
        const int room = a.top - __popcll(sure);
        int place = 0;
        for (uint64_t todo = near; todo; todo &= todo - 1) {
          const int g = __builtin_ctzll(todo);
          const uint64_t o = __shfl((unsigned long long)score, g, 64);
          place += o > score || (o == score && g < lane);
        }
        const uint64_t chosen = __ballot((near >> lane & 1) && place < room);
        keep = sure | chosen;
        if constexpr (MODE == kKeySoftmax) {
          // Z's error moves two groups' totals by as much of the difference of their scores, which biases may hide: it is
          // below twice the larger score.  A pair across the cut that is no further apart goes to exact sums.
          if (b) {
            bool unclear = false;
            for (uint64_t todo = near & ~chosen; todo; todo &= todo - 1) {
              const int g = __builtin_ctzll(todo);
              const double o = key64_inv(__shfl((unsigned long long)score, g, 64));
              const float om = __shfl(most, g, 64);
              unclear |= (chosen >> lane & 1) && key64_inv(score) - o <= 2.0 * kSelSumErr * (double)fmaxf(most, om);
            }
            if (__any(unclear)) return false;   // (the same in every wave)
          }
        }
      }
    }
  }
  const bool live = active && (keep >> (grp & 63) & 1) != 0;
  // (maxima of live lanes that hold chapters)
  const int maxima = (grouped ? a.top : 1) * (Q == 4 ? min(4 * lpg, per) : min(lpg, (per + 3) / 4));
  uint32_t T = 0;
  if (maxima >= a.k) {
    if constexpr (Q == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = live ? __uint_as_float(key32(mx[e])) : 0.f;
    } else {
      sm.maxima[tl] = live ? key32(fmax_fast(fmax_fast(mx[0], mx[1]), fmax_fast(mx[2], mx[3]))) : 0u;
      team_sync<NW>();
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(sm.maxima[lane + 64 * e]);
    }
    // from the bits that the live maxima do not share; t may lie below the k-th maximum, by the low byte or as long as
    // not many more maxima are above it
    uint32_t hi = 0, lo = ~0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = __float_as_uint(mx[e]);
      hi = max(hi, u);
      lo = u ? min(lo, u) : lo;
    }
    hi = lanes_reduce(hi, [](uint32_t x, uint32_t y) { return max(x, y); });
    lo = lanes_reduce(lo, [](uint32_t x, uint32_t y) { return min(x, y); });
    const int top = 31 - __builtin_clz((hi ^ lo) | 0x100u);
    T = hi & ~((2u << top) - 1);
    for (int bit = top; bit >= 8; --bit) {
      const uint32_t t = T | 1u << bit;
      int cnt = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) cnt += __popcll(__ballot(__float_as_uint(mx[e]) >= t));
      if (cnt >= a.k) {
        T = t;
        if (cnt <= a.k + (a.k >> 2)) break;
      }
    }
  } else {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = T | 1u << bit;
      const float tf = key32_inv(t);
      int cnt = 0;
      if (live && t > 0x007fffffu) {
#pragma unroll
        for (int j = 0; j < E4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) cnt += v[j][e] >= tf;
      }
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) cnt += __shfl_xor(cnt, o, 64);
      cnt = team_add<NW>(cnt, sm, wave);
      if (cnt >= a.k) {
        T = t;
        if (cnt <= 2 * a.k + 32) break;
      }
    }
  }
  if (T <= 0x007fffffu) return false;   // fewer than k keys above -inf
  const float t0 = key32_inv(T), thr = MODE == kKeyLogit ? t0 : t0 - 2.f * (kSelEps + 0x1p-24f * fabsf(t0));
  // candidates: the lane's as bits, then a list in lane order
  uint32_t bits[(E + 31) / 32];
  lane_bits<E>(v, thr, bits);
  int cnt = 0;
#pragma unroll
  for (int i = 0; i < (E + 31) / 32; ++i) {
    bits[i] = live ? bits[i] : 0u;
    cnt += __popc(bits[i]);
  }
  int base = 0, ncand = 0;
  if constexpr (NW > 1) {
    // where the wave's candidates go: behind those of the waves before it
    const int mine_all = (int)lanes_reduce((uint32_t)cnt, [](uint32_t x, uint32_t y) { return x + y; });
    team_sync<NW>();
    if (lane == 0) sm.count[wave] = mine_all;
    team_sync<NW>();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      base += i < wave ? sm.count[i] : 0;
      ncand += sm.count[i];
    }
    if (ncand > kSelCand) return false;
  }
  // one candidate per lane and round
#pragma unroll
  for (int i = 0; i < (E + 31) / 32; ++i) {
    uint32_t w = bits[i];
    for (uint64_t has = __ballot(w != 0); has; has = __ballot(w != 0)) {
      const int p = base + lanes_before(has);
      if (w && p < kSelCand) sm.id[p] = c0 + chapter(32 * i + __builtin_ctz(w));
      w &= w - 1;
      base += __popcll(has);
    }
  }
  if constexpr (NW == 1) {
    ncand = base;
    if (ncand > kSelCand) return false;
  }
  team_sync<NW>();
  // exact keys of the candidates
  constexpr int NC = kSelCand / TL;
  for (int p = tl; p < ncand; p += TL) {
    const int c = sm.id[p];
    const float x = z[c];
    const double s = score64(x, a.sigmoid, m, Z);
    sm.key[p] = key64(MODE == kKeyLogit ? (double)x : s + (b ? (double)b[c] : 0.0));
    sm.score[p] = (float)s;
  }
  team_sync<NW>();
  uint64_t key[NC];
  float sc[NC];
  int32_t id[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int p = tl + TL * i;
    key[i] = p < ncand ? sm.key[p] : 0;
    sc[i] = p < ncand ? sm.score[p] : 0.f;
    id[i] = p < ncand ? sm.id[p] : 0;
  }
  int rank[NC];
  bool unclear = false;
#pragma unroll
  for (int i = 0; i < NC; ++i) rank[i] = tl + TL * i < ncand ? 0 : kSelCand;
  auto against = [&](uint64_t kj, int32_t ij) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (TL * i < ncand) {   // (the same in every lane)
        rank[i] += kj > key[i] || (kj == key[i] && ij < id[i]);
        if constexpr (MODE == kKeySoftmax) {
          // Z's error moves a pair of keys by as much of their scores' difference
          const double gap = fabs(key64_inv(kj) - key64_inv(key[i]));
          unclear |= tl + TL * i < ncand && ij != id[i] && gap <= kSelSumErr * (double)sc[i] && z[ij] != z[id[i]];
        }
      }
    }
  };
  if constexpr (NW == 1) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      for (int j = 0; j < min(TL, ncand - TL * i); ++j) against(lane_value(key[i], j), (int32_t)lane_value((uint32_t)id[i], j));
  } else {
#pragma unroll 4
    for (int j = 0; j < ncand; ++j) against(sm.key[j], sm.id[j]);
  }
  if constexpr (MODE == kKeySoftmax) {
    if (team_add<NW>(__popcll(__ballot(unclear)), sm, wave) != 0) return false;
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < NC; ++i) sum += rank[i] < a.k ? (double)sc[i] : 0.0;
  sum = team_sum<NW>(sum, sm, wave);
  if constexpr (MODE != kKeySigmoid) {
    if (a.row_stats) {
      // (the same bits that the selected have in Z)
      double e = 0.0;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        e += rank[i] < a.k ? (double)__builtin_amdgcn_exp2f((z[id[i]] - m) * 1.4426950408889634f) : 0.0;
      e = team_sum<NW>(e, sm, wave);
      if (tl == 0) put_row_stats(a, r, m, Z, e);
    }
  }
  const double f = (double)a.scale / (a.renorm ? fmax(sum, 1e-12) : 1.0);
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (rank[i] < a.k) {
      const int64_t o = r * a.k + rank[i];
      a.idx[o] = id[i] + a.S;
      a.w[o] = (float)((double)sc[i] * f);
      if (a.s_sel) a.s_sel[o] = sc[i];
    }
  return true;
}

// Four waves: four rows (NW = 1) or one (NW = 4); rows that select_team leaves are then taken by the whole workgroup.
// Bound, few rows: dependent steps (the bisection for the k-th key, the ranks of the candidates): 16 rows of 4,097, k = 64, four
// waves each 10.6 us, the waves waiting for 0.54 of it.  Many rows: the VALU, at work for 0.57 to 0.61 of the time: 8,192 rows of
// 4,097, k = 16 44 us (3.0 TB/s; HBM moves these 134 MB in 26); 16,001 rows of 257, k = 8, softmax with a backward's statistics
// 32 us, the same steps of a wave whose lanes hold four or five logits.  2,039 rows of 4,097 17.6 us, two rounds of waves.
template <int NW, int E, int MODE>
__global__ __launch_bounds__(kSelThreads, E <= 64 ? 3 : 2) void router_select_team_kernel(SelArgs a) {
  constexpr int kTeams = 4 / NW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int left[kTeams];
  SelTeam<NW>* teams = (SelTeam<NW>*)lds;
  const int team = NW == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int tl = NW == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const int64_t r0 = (int64_t)blockIdx.x * kTeams, r = r0 + team;
  const bool done = r >= a.R || select_team<NW, E, MODE>(a, r, teams[team], tl);
  if (tl == 0) left[team] = !done;
  __syncthreads();
  for (int t = 0; t < kTeams; ++t)
    if (left[t]) {
      select_row(a, r0 + t, lds);
      __syncthreads();
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

// A team of NT threads per row (a wave: four rows per workgroup): the row of zeros, or of the softmax's dense part, then
// the selected entries over it.  Bound by the stores: 8,192 x 4,097 (134 MB) 22 to 24 us by card, a plain fill of as much
// 18.2.  With the softmax's dense part (16,001 x 257) 14 us, where reading the logits and writing takes 6.4.
template <int NT>
__global__ __launch_bounds__(kSelThreads) void router_select_bwd_kernel(SelBwdArgs a) {
  constexpr int kRows = kSelThreads / NT;
  __shared__ double red[NT / 64];
  const int64_t r = (int64_t)blockIdx.x * kRows + (NT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  if (r >= a.R) return;
  const int tid = NT == 64 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  double sum = 0.0, dot = 0.0;
  for (int j = tid; j < a.k; j += NT) {
    const double s = a.s_sel[r * a.k + j];
    sum += s;
    dot += s * (double)a.dw[r * a.k + j];
  }
  if constexpr (NT == 64) {
    sum = lanes_sum(sum);
    dot = lanes_sum(dot);
  } else {
    sum = blk_sum<NT>(sum, red);
    dot = blk_sum<NT>(dot, red);
  }
  const bool clamped = !(sum > 1e-12);
  const double D = a.renorm ? (clamped && sum == sum ? 1e-12 : sum) : 1.0;
  // sum_j ds_j s_j of the softmax
  const double t = a.sigmoid || (a.renorm && !clamped) ? 0.0 : (double)a.scale * dot / D;
  const double f = (double)a.scale / D, shift = a.renorm && !clamped ? dot / D : 0.0;   // ds_j = f (dw_j - shift)
  float* row = a.dz + r * a.C;
  double rest = 0.0;   // of the softmax's mass: what is not selected
  if (t == 0.0) {
    for (int64_t c = tid; c < a.C; c += NT) row[c] = 0.f;
  } else {
    const float m = a.row_stats[3 * r];
    const float ft = (float)(-t / (double)a.row_stats[3 * r + 1]);
    rest = (double)a.row_stats[3 * r + 2];
    for (int64_t c = tid; c < a.C; c += NT) row[c] = c < a.S ? 0.f : expf(a.z[r * a.ldz + c] - m) * ft;
  }
  // (the row's stores are done before the entries')
  if constexpr (NT == 64) __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  else __syncthreads();
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
  for (int j = tid; j < a.k; j += NT) {
    const double s = a.s_sel[r * a.k + j], ds = f * ((double)a.dw[r * a.k + j] - shift);
    const int32_t c = a.idx[r * a.k + j];
    if (a.sigmoid) {
      // s (1 - s) from the logit, e^-|z| / (1 + e^-|z|)^2: a score near 1 that was rounded to f32 has lost 1 - s
      const double e = exp(-fabs((double)a.z[r * a.ldz + c])), q = 1.0 + e;
      row[c] = (float)(ds * (e / (q * q)));
    } else {
      // (1 - sum s from the rest of the row: a score near 1 that was rounded to f32 has lost it)
      row[c] = (float)(s * (t == 0.0 ? ds : ds * rest + (ds * sum - t)));
    }
  }
}

// counts[c] += selections of c; one thread per selection, integer adds (their order changes nothing).
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
// integers: count * (C - S) against the total).  With the clearing and the counting 16 us for 131,072 ids of 4,097 chapters,
// three launches at their latency, once a training step.
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

template <int NW, int E> int select_team_launch(const SelArgs& a, int mode, hipStream_t stream) {
  const size_t lds = std::max(sizeof(SelTeam<NW>) * (4 / NW), select_row_lds(a.n, a.G, a.k));
  const dim3 grid((unsigned)((a.R + 4 / NW - 1) / (4 / NW)));
  if (mode == kKeyLogit)
    hipLaunchKernelGGL((router_select_team_kernel<NW, E, kKeyLogit>), grid, dim3(kSelThreads), lds, stream, a);
  else if (mode == kKeySigmoid)
    hipLaunchKernelGGL((router_select_team_kernel<NW, E, kKeySigmoid>), grid, dim3(kSelThreads), lds, stream, a);
  else
    hipLaunchKernelGGL((router_select_team_kernel<NW, E, kKeySoftmax>), grid, dim3(kSelThreads), lds, stream, a);
  return check_launch("router_select_team_kernel");
}

int select_launch(const SelArgs& a, hipStream_t stream) {
  const bool grouped = a.top < a.G;
  const int Ge = grouped ? a.G : 1;
  // a group's score adds two keys: scores are needed then, or where a bias is added to them
  const int mode = !a.bias && (!grouped || a.best == 1) ? kKeyLogit : a.sigmoid ? kKeySigmoid : kKeySoftmax;
  const int NW = a.R <= kSelFewRows ? 4 : 1;
  // elements per lane: four consecutive chapters of the lane's group per load
  const int lanes = 64 * NW / std::max(Ge, 1);
  const int e = lanes > 0 ? 4 * ((a.n / Ge + 4 * lanes - 1) / (4 * lanes)) : 1 << 30;
  if (a.k <= kSelTeamK && Ge <= 64 && a.n / Ge >= 4 && e <= (NW == 1 ? 72 : 24)) {
    if (NW == 4) {
      if (e <= 4) return select_team_launch<4, 4>(a, mode, stream);
      if (e <= 16) return select_team_launch<4, 16>(a, mode, stream);
      return select_team_launch<4, 24>(a, mode, stream);
    }
    if (e <= 4) return select_team_launch<1, 4>(a, mode, stream);
    if (e <= 16) return select_team_launch<1, 16>(a, mode, stream);
    if (e <= 32) return select_team_launch<1, 32>(a, mode, stream);
    if (e <= 64) return select_team_launch<1, 64>(a, mode, stream);
    return select_team_launch<1, 72>(a, mode, stream);
  }
  const size_t lds = select_row_lds(a.n, a.G, a.k);
  if (lds > 65536)
    MOC_HIP(hipFuncSetAttribute((const void*)router_select_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(router_select_kernel, dim3((unsigned)a.R), dim3(kSelThreads), lds, stream, a);
  return check_launch("router_select_kernel");
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
  return select_launch(a, stream);
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
  if (R > kSelFewRows)
    hipLaunchKernelGGL(router_select_bwd_kernel<64>, dim3((unsigned)((R + 3) / 4)), dim3(kSelThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(router_select_bwd_kernel<kSelThreads>, dim3((unsigned)R), dim3(kSelThreads), 0, stream, a);
  return check_launch("router_select_bwd_kernel");
}

int moc_router_balance(const int32_t* idx, int64_t n, int64_t C, int S, float rate, int32_t* counts, float* bias,
                       hipStream_t stream) {
  MOC_REQUIRE(n >= 0 && n < ((int64_t)1 << 31) && C > 0 && C <= kSelMaxC && S >= 0 && S < C, MOC_ERR_ARG,
              "moc_router_balance: n=%lld C=%lld S=%d", (long long)n, (long long)C, S);
  MOC_REQUIRE(counts && bias && (idx || n == 0), MOC_ERR_ARG, "moc_router_balance: null pointer");
  hipLaunchKernelGGL(select_clear_kernel, dim3((unsigned)((C + 255) / 256)), dim3(256), 0, stream, counts, C);
  if (n > 0)
    hipLaunchKernelGGL(select_count_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, idx, n, C, counts);
  hipLaunchKernelGGL(balance_update_kernel, dim3(1), dim3(1024), 0, stream, counts, C, S, rate, bias);
  return check_launch("balance_update_kernel");
}

}  // extern "C"
