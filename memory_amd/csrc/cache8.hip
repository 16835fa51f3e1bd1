// Attention over a decode cache held in 8 bits: K / V tiles of every chapter in e4m3 (OCP), one f32 scale per
// (chapter, kv head) for K and one for V.
//
// For sequence b with slots (chapter c, weight omega) and a query row q of kv head hk:
//   s_j = omega * ks[c, hk] * scale * (q . k8_j),  o = sum_j softmax_j(s) * omega * vs[c, hk] * v8_j
// i.e. the decode attention of decode.hip over K = ks k8, V = vs v8; the scales are one factor per 64-key tile and
// fold into the logit factor and the probabilities, so the products run on the 8-bit values, widened to bf16 (exact).
//
// Layout: k_tiles[c][hk][key][dim] and v_tiles[c][hk][dim][pos], position 16 g + 4 kb + x of a dim holding key
// 16 kb + 4 g + x.  That is the key order of the probabilities in the matrix accumulator (lane group g, values x of
// key block kb), so that a lane's keys of one dim are 16 consecutive bytes: every operand of both products is one
// 16-byte load per lane straight into registers, and V needs no transpose.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "moc_common.h"

namespace moc {
namespace {

constexpr int kC8Dh = 64;
constexpr int kC8Tile = 64 * 64;   // elements (= bytes) of a tile
constexpr float kC8Max = 448.f;    // largest e4m3 value

// the maximum over the wave (NaN stays)
__device__ __forceinline__ float wave_max_nan(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmax_fast(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float c8_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// eight e4m3 values (two words) as bf16, exact
__device__ __forceinline__ bf16x8 c8_widen(uint32_t a, uint32_t b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true)};
  return __builtin_bit_cast(bf16x8, v);
}

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
// the same as f16 (exact as well: e4m3 spans 2^-9 .. 448)
__device__ __forceinline__ f16x8 c8_widen_f16(uint32_t a, uint32_t b) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const f16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false),
                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true)};
  return __builtin_bit_cast(f16x8, v);
}
__device__ __forceinline__ void mma16(f32x4& c, const f16x8& a, const f16x8& b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ------------------------------------------------------------------ quantising
// One workgroup per tile (blockIdx.y: K or V).  scale = 2^ceil(log2(amax / 448)) of the largest finite magnitude (1
// for a tile of zeros): x / scale is then exact and every element is rounded once, to nearest even.  Infinities
// become +-448 scale, NaN stays NaN.  Bound: HBM (read once into registers, a tile's maximum through LDS): 4,097 chapters of 12
// heads in bf16 206 us, 5.9 TB/s, in f32 350 us, 5.8 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void cache8_pack_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                          uint8_t* __restrict__ k8, uint8_t* __restrict__ v8,
                                                          float* __restrict__ k_scale, float* __restrict__ v_scale) {
  __shared__ float red[4];
  __shared__ uint8_t tile[64 * 68];
  const int64_t t = blockIdx.x;
  const bool is_v = blockIdx.y == 1;
  const T* src = (is_v ? v : k) + t * kC8Tile + 16 * threadIdx.x;   // row threadIdx / 4, elements 16 (threadIdx % 4) ..
  float x[16];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = to_f(src[i]);
    const float m = fabsf(x[i]);
    amax = m < INFINITY && m > amax ? m : amax;
  }
  amax = wave_max(amax);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  // the exponent e with 448 2^(e-1) < amax <= 448 2^e, within what 2^e and 2^-e can hold
  int e = 0;
  if (amax > 0.f) {
    e = ilogbf(amax) - 8;                       // 2^8 <= 448 < 2^9
    if (ldexpf(amax, -e) > kC8Max) ++e;
    e = max(-120, min(120, e));
  }
  const float inv = ldexpf(1.f, -e);
  if (threadIdx.x == 0) (is_v ? v_scale : k_scale)[t] = ldexpf(1.f, e);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[j] = x[4 * i + j] * inv;
      y[j] = y[j] > kC8Max ? kC8Max : y[j] < -kC8Max ? -kC8Max : y[j];   // (NaN passes)
    }
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
  }
  if (!is_v) {
    V16 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.w[i] = w[i];
    st16(k8 + t * kC8Tile + 16 * threadIdx.x, o);
    return;
  }
  const int key = threadIdx.x >> 2, pos = 16 * ((key >> 2) & 3) + 4 * (key >> 4) + (key & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[(16 * (threadIdx.x & 3) + 4 * i + j) * 68 + pos] = (uint8_t)(w[i] >> (8 * j));
  __syncthreads();
  V16 o;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o.w[i] = *reinterpret_cast<const uint32_t*>(tile + (threadIdx.x >> 2) * 68 + 16 * (threadIdx.x & 3) + 4 * i);
  st16(v8 + t * kC8Tile + 16 * threadIdx.x, o);
}

// ------------------------------------------------------------------ few queries: one wave per (chapter, kv head)
// Each selected tile is read once however many sequences chose it (the chapter plan over the (sequence, slot) edges),
// as decode.hip does.  Rows of a unit: edge, query token, head of the kv group; 16 at a time.
//   S^T = K Q^T (lane = query row), softmax over the 64 keys, O^T = V^T P^T, normalised rows to part rows
// [edge][token][head][64] with their log-sum-exp and value factor omega vs; cache8_combine_kernel merges the slots.
// Probabilities (at most 1) and part rows (averages of e4m3 values, at most 448) are rounded to f16, 2^-11 where bf16
// would round by 2^-8 at the same bytes: with bf16 the result was 1.7 times as far from the exact one as its own
// rounding.
// Bound: HBM, or latency where the units are few.  Eight loads of 16 bytes per lane hold the whole tile pair.  64 sequences
// with 65 of 4,097 chapters, 12 heads (256 MB of tiles): 40 us, 6.3 TB/s, where a copy of 1 GiB reaches 5.2 (part of the tiles
// stays in the last-level cache); one sequence: 4 us.  37 sequences of 16 heads on 4: 17 us, most of it the one wave per kv head
// that takes the shared chapter's 148 rows, ten blocks of about 1 us one after the other.
constexpr int kC8Waves = 4;

struct C8Unit {
  const bf16* q;
  const uint8_t *k8, *v8;
  const float *ks, *vs, *omega;
  const int32_t *uniq, *n_uniq, *csr_off, *csr_edge, *row_tab;
  f16* o_part;
  float2* lse_part;
  int64_t max_u;
  int L, H, HK, NS;
  uint32_t ns_mul, ns_shift;   // e / NS = e ns_mul >> ns_shift for e < 2^31
  float scale_log2;
};

__global__ __launch_bounds__(64 * kC8Waves) void cache8_unit_kernel(C8Unit a) {
  const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = (int64_t)blockIdx.x * kC8Waves + wave;
  const int64_t u = unit / a.HK;
  const int hk = (int)(unit % a.HK);
  if (u >= a.max_u) return;
  const int G = a.H / a.HK, GL = G * a.L;
  // the first 16 rows' edges come with the plan entries, not after them
  const int eid = a.row_tab[u * 16 + c16 / GL];
  const int nu = a.n_uniq[0];
  const int64_t c = a.uniq[u];
  const int p0 = a.csr_off[u], cnt = a.csr_off[u + 1] - p0;
  if (u >= nu) return;
  const int nrows = cnt * GL;
  const int64_t tile = c * a.HK + hk;
  V16 kw[4], vw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) kw[i] = ld16(a.k8 + tile * kC8Tile + 64 * (16 * i + c16) + 16 * g);
#pragma unroll
  for (int i = 0; i < 4; ++i) vw[i] = ld16(a.v8 + tile * kC8Tile + 64 * (16 * i + c16) + 16 * g);
  const float ks = a.ks[tile] * a.scale_log2, vs = a.vs[tile];
  // a row block's operands: its edges two blocks ahead, its queries one (a chapter that every sequence selects has many)
  struct Rows {
    bf16x8 qf[2];
    int64_t row;
    float w;
  };
  // row r0 + c16 is row `rem` of edge number j of the chapter; both move on by 16 rows without a division
  const int step_j = 16 / GL, step_rem = 16 % GL;
  int j = c16 / GL, rem = c16 % GL;
  auto move_on = [&] {
    j += step_j;
    rem += step_rem;
    if (rem >= GL) {
      rem -= GL;
      ++j;
    }
  };
  auto fetch = [&](int e, int rm) {
    Rows x;
    x.qf[0] = x.qf[1] = zero_frag<bf16>();
    x.row = -1;
    x.w = 1.f;
    if (e >= 0) {
      const int l = a.L == 1 ? 0 : rm / G, at = l * a.H + hk * G + (a.L == 1 ? rm : rm % G);   // (token, head)
      const int64_t lh = (int64_t)a.L * a.H;
      x.row = e * lh + at;
      x.w = a.omega[e];
      const int64_t seq = (int64_t)(((uint64_t)(uint32_t)e * a.ns_mul) >> a.ns_shift);
      const bf16* qp = a.q + (seq * lh + at) * kC8Dh + 16 * g;
      x.qf[0] = Load8<bf16, bf16>::run(qp);
      x.qf[1] = Load8<bf16, bf16>::run(qp + 8);
    }
    return x;
  };
  Rows cur = fetch(c16 < nrows ? eid : -1, rem);
  move_on();
  int ahead = 16 + c16 < nrows ? a.csr_edge[p0 + j] : -1, ahead_rem = rem;
  for (int r0 = 0; r0 < nrows; r0 += 16) {
    Rows next = cur;
    if (r0 + 16 < nrows) {   // (the same in every lane)
      next = fetch(ahead, ahead_rem);
      move_on();
      ahead = r0 + 32 + c16 < nrows ? a.csr_edge[p0 + j] : -1;
      ahead_rem = rem;
    }
    const bf16x8 (&qf)[2] = cur.qf;
    const int64_t row = cur.row;
    const float w = cur.w;
    // S^T: lane = query row r0 + c16, keys 16 kb + 4 g + x; dims 16 g + 8 ks of both operands
    f32x4 st[4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      st[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
      mma(st[kb], c8_widen(kw[kb].w[0], kw[kb].w[1]), qf[0]);
      mma(st[kb], c8_widen(kw[kb].w[2], kw[kb].w[3]), qf[1]);
    }
    float mx = st[0][0];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int x = 0; x < 4; ++x) mx = fmax_fast(mx, st[kb][x]);
    const float cf = w * ks;
    mx = quad_max_pl(mx);
    const float m = mx * cf;
    float ps = 0.f;
    f16x8 pf[2];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p = c8_exp2((st[kb][x] - mx) * cf);   // (at most 1, however large the logits)
        ps += p;
        pf[kb >> 1][4 * (kb & 1) + x] = (f16)p;
      }
    const float l = quad_sum_pl(ps);
    // O^T: lane = query row, dims 16 db + 4 g + x
    f32x4 o[4];
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
      mma16(o[db], c8_widen_f16(vw[db].w[0], vw[db].w[1]), pf[0]);
      mma16(o[db], c8_widen_f16(vw[db].w[2], vw[db].w[3]), pf[1]);
    }
    if (row >= 0) {
      const float inv = 1.f / l;
      f16* op = a.o_part + row * kC8Dh;
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        f16x4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = (f16)(o[db][x] * inv);
        *reinterpret_cast<f16x4*>(op + 16 * db + 4 * g) = v;
      }
      if (g == 0) a.lse_part[row] = make_float2(m + __builtin_amdgcn_logf(l), w * vs);
    }
    cur = next;
  }
}

// out = sum_s 2^(lse_s - M) f_s o_s / sum_s 2^(lse_s - M) over a row's slots: one wave per row, lane s holding slot s's
// statistics, eight lanes of 16 bytes per part row.  A skipped slot's entries were never written: its factor is 0 and what
// was read of its row is dropped by a select.  Bound: latency of two dependent loads (one sequence of 12 heads 4 us; 64
// sequences, 6.4 MB of part rows, 5.8 us).
__global__ __launch_bounds__(256) void cache8_combine_kernel(const f16* __restrict__ o_part, const float2* __restrict__ lse_part,
                                                             const int32_t* __restrict__ edge_u, int NS, int rpe, int64_t rows,
                                                             bf16* __restrict__ out) {
  const int lane = threadIdx.x & 63, sg = lane >> 3, ch = lane & 7;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int64_t e0 = row / rpe * NS;
  const int r = (int)(row % rpe);
  constexpr int kSlots = 72;   // of a round: nine loads per lane, all in flight before the statistics are used
  float M = -INFINITY, den = 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < NS; s0 += kSlots) {
    const int n = min(kSlots, NS - s0);
    f16x8 v[kSlots / 8];
#pragma unroll
    for (int i = 0; i < kSlots / 8; ++i)
      v[i] = 8 * i + sg < n ? *reinterpret_cast<const f16x8*>(o_part + ((e0 + s0 + 8 * i + sg) * rpe + r) * kC8Dh + 8 * ch) : f16x8{};
    float2 st[2];   // slots lane and 64 + lane of the round
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t e = e0 + s0 + lane + 64 * q;
      st[q] = make_float2(-INFINITY, 0.f);
      if (lane + 64 * q < n) {
        const int u = edge_u[e];
        const float2 t = lse_part[e * rpe + r];
        if (u >= 0) st[q] = t;
      }
    }
    const float Mn = fmax_fast(M, wave_max_nan(fmax_fast(st[0].x, st[1].x)));
    const float scale = M == Mn ? 1.f : c8_exp2(M - Mn);   // (NaN passes)
    float a[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float p = st[q].x == -INFINITY ? 0.f : c8_exp2(st[q].x - Mn);
      den = (q == 0 ? den * scale : den) + p;
      a[q] = st[q].x == -INFINITY ? 0.f : p * st[q].y;
    }
    M = Mn;
#pragma unroll
    for (int x = 0; x < 8; ++x) acc[x] *= scale;
#pragma unroll
    for (int i = 0; i < kSlots / 8; ++i) {
      const float aj = __shfl(8 * i < 64 ? a[0] : a[1], (8 * i + sg) & 63, 64);
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[x] += aj != 0.f ? aj * (float)v[i][x] : 0.f;
    }
  }
  den = wave_sum(den);
#pragma unroll
  for (int o = 8; o < 64; o <<= 1)
#pragma unroll
    for (int x = 0; x < 8; ++x) acc[x] += __shfl_xor(acc[x], o, 64);
  if (lane < 8) {
    const float inv = den == 0.f ? 0.f : 1.f / den;
    bf16x8 v;
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = (bf16)(acc[x] * inv);
    *reinterpret_cast<bf16x8*>(out + row * kC8Dh + 8 * lane) = v;
  }
}

// ------------------------------------------------------------------ many queries: running softmax over the slots
// One workgroup = 256 query rows (token, head of the kv group) of one (sequence, kv head), 8 waves x 32 rows; the
// heads of a group share every tile.  A tile pair is 8 KB of e4m3: each thread loads eight bytes of K and of V one slot
// ahead (two ahead took more registers than there are: 200 us), widens them once and puts them into LDS, K as bf16 and V
// as f16, double-buffered, for all waves (four waves of 16 bytes: 191 us against 183).  Probabilities are f16: with bf16 the
// kernel took 183 us for 4 x 2,048 tokens of 16 heads in place of 188 to 194, at 1.4 times the error against float64
// (0.0024; 0.0017 is what rounding the result to bf16 alone gives).  163 to 177 us a call in a row of calls, 178 to 188 alone, by card:
// 790 to 857 TFLOP/s, 0.65 to 0.70 of a large matrix product's rate.  Bound: the exponentials and the products, which hardly overlap (matrix units busy 0.34,
// VALU 0.6 of the time).  Running maximum (raised lazily) and sum as in the sequence attention (xattn_fwd.hip).
constexpr int kC8Threads = 512;
constexpr int kC8Rows = kC8Threads / 2;   // 32 per wave
constexpr float kC8Slack = 8.f;

struct C8Prompt {
  const bf16* q;
  const uint8_t *k8, *v8;
  const float *ks, *vs, *omega;
  const int32_t* idx;
  bf16* out;
  float *part, *lse;
  int64_t C;
  int B, L, H, HK, NS, nsplit;
  float scale_log2;
};

__global__ __launch_bounds__(kC8Threads, 4) void cache8_prompt_kernel(C8Prompt a) {
  using Tile = SwzTile<bf16, 64>;
  __shared__ __attribute__((aligned(16))) char sK[2][8192];
  __shared__ __attribute__((aligned(16))) char sV[2][8192];
  const int G = a.H / a.HK;
  const int64_t rows = (int64_t)a.L * G;
  const int64_t nqb = (rows + kC8Rows - 1) / kC8Rows;
  const int64_t t = xcd_tile((int64_t)a.B * a.HK * a.nsplit * nqb);
  if (t < 0) return;
  const int64_t bh = t / (a.nsplit * nqb);
  const int b = (int)(bh / a.HK), hk = (int)(bh % a.HK), sp = (int)((t / nqb) % a.nsplit);
  const int s_begin = (int)((int64_t)a.NS * sp / a.nsplit), s_end = (int)((int64_t)a.NS * (sp + 1) / a.nsplit);
  const int64_t q0 = (t % nqb) * kC8Rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c16 = lane & 15;

  // query rows (of the sequence: token * H + head; -1 past the end) and their fragments
  const bf16* qb0 = a.q + (int64_t)b * a.L * a.H * kC8Dh;
  auto query_row = [&](int qb) {
    const int r = (int)q0 + 32 * wave + 16 * qb + c16;
    return r < rows ? r / G * a.H + hk * G + r % G : -1;
  };
  bf16x8 qf[2][2];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int qr = query_row(qb);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      qf[qb][ks] = qr >= 0 ? Load8<bf16, bf16>::run(qb0 + (int64_t)qr * kC8Dh + 32 * ks + 8 * g) : zero_frag<bf16>();
  }
  float m[2] = {-INFINITY, -INFINITY}, lsum[2] = {0.f, 0.f};
  float F = 0.f, inv_F = INFINITY, f_min = 0.f;   // (f_min: 2^-90 of the largest factor met)
  f16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (f16)1.f;
  f32x4 o[4][2];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int32_t* ids = a.idx + (int64_t)b * a.NS;
  const float* om = a.omega + (int64_t)b * a.NS;
  auto slot_tile = [&](int s) -> int64_t {
    const int64_t c = ids[s];
    return c >= 0 && c < a.C ? c * a.HK + hk : -1;
  };
  uint2 kr, vr;
  auto fetch = [&](int64_t tile) {
    kr = *reinterpret_cast<const uint2*>(a.k8 + tile * kC8Tile + 8 * tid);
    vr = *reinterpret_cast<const uint2*>(a.v8 + tile * kC8Tile + 8 * tid);
  };
  const int st_off = Tile::off(tid >> 3, 8 * (tid & 7));
  auto stage = [&](int buf) {
    *reinterpret_cast<bf16x8*>(sK[buf] + st_off) = c8_widen(kr.x, kr.y);
    *reinterpret_cast<f16x8*>(sV[buf] + st_off) = c8_widen_f16(vr.x, vr.y);
  };
  // a slot's logit and value factors are loaded with its tile, its chapter id one slot before that
  int64_t cur = slot_tile(s_begin);
  int64_t next = s_begin + 1 < s_end ? slot_tile(s_begin + 1) : -1;
  float c = 0.f, f = 0.f;
  if (cur >= 0) {
    fetch(cur);
    c = om[s_begin] * a.ks[cur] * a.scale_log2;
    f = om[s_begin] * a.vs[cur];
    stage(0);
  }
  __syncthreads();
  auto slots = [&](auto busy) {
  for (int s = s_begin; s < s_end; ++s) {
    const int buf = (s - s_begin) & 1;
    float w1 = 0.f, ks1 = 0.f, vs1 = 0.f;
    if (next >= 0) {
      fetch(next);
      w1 = om[s + 1];
      ks1 = a.ks[next];
      vs1 = a.vs[next];
    }
    const int64_t after = s + 2 < s_end ? slot_tile(s + 2) : -1;
    if constexpr (decltype(busy)::value) if (cur >= 0) {
      f32x4 st[4][2];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) st[kb][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const bf16x8 ka = Tile::frag(sK[buf], 16 * kb + c16, 32 * ks + 8 * g);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) mma(st[kb][qb], ka, qf[qb][ks]);
        }
      // a lane's keys tell whether a row's reference has to rise; only then is the row's maximum formed
      float mx[2];
      bool grow = false;
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        mx[qb] = st[0][qb][0];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int x = 0; x < 4; ++x) mx[qb] = fmax_fast(mx[qb], st[kb][qb][x]);
        grow |= mx[qb] * c > m[qb] + kC8Slack;   // (c >= 0)
      }
      if (__any(grow)) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const float cm = quad_max_pl(mx[qb]) * c;
          const float mn = cm > m[qb] + kC8Slack ? cm : m[qb];
          const float alpha = c8_exp2(m[qb] - mn);
          m[qb] = mn;
          lsum[qb] *= alpha;
#pragma unroll
          for (int db = 0; db < 4; ++db) o[db][qb] *= alpha;
        }
      }
      // O is held in units of F, a value factor omega vs met before; a slot's probabilities carry f / F, in the
      // exponent.  Within 2^-1 .. 2^6 of F they stay below 2^14, and one that f16's smallest step rounds away is
      // below 2^-24 of the row's largest; past that F becomes f.  f = 0 leaves O alone and counts in the sum, and so
      // does an f below 2^-90 of the largest factor met, so that F stays above that and O in f32's range (448 2^90
      // times the sum of the probabilities), however the factors fall from slot to slot.
      float r = f * inv_F;
      const bool none = f == 0.f || f < f_min;
      f_min = fmaxf(f_min, f * 0x1p-90f);
      if (!none && !(r > 0x1p-1f && r < 0x1p6f)) {   // (the first slot; NaN too)
        const float beta = F / f;
        F = f;
        inv_F = 1.f / f;
        r = 1.f;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) o[db][qb] *= beta;
      }
      r = none ? 1.f : r;
      const float lr = __builtin_amdgcn_logf(r), rr = __builtin_amdgcn_rcpf(r);
      // Past 2^22 the product's rounding in m shows in the exponent (the difference below is fused): there the logits are
      // rounded alike and subtracted first, and are at most kC8Slack.
      float cc = c;
      float off[2] = {m[0] - lr, m[1] - lr};
      if (__any(fmax_fast(fabsf(m[0]), fabsf(m[1])) > 0x1p22f)) {
#pragma clang fp contract(off)
        cc = 1.f;
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          off[qb] = -lr;
#pragma unroll
          for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int x = 0; x < 4; ++x) st[kb][qb][x] = st[kb][qb][x] * c - m[qb];
        }
      }
      f16x8 pf[2][2];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            pf[qb][h][x] = (f16)c8_exp2(st[2 * h][qb][x] * cc - off[qb]);
            pf[qb][h][4 + x] = (f16)c8_exp2(st[2 * h + 1][qb][x] * cc - off[qb]);
          }
        // row sums of the rounded probabilities, in units of r
        f32x4 ls = f32x4{0.f, 0.f, 0.f, 0.f};
        mma16(ls, ones, pf[qb][0]);
        mma16(ls, ones, pf[qb][1]);
        lsum[qb] += ls[0] * rr;
      }
      if (!none)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          const f16x8 va = __builtin_bit_cast(f16x8, Tile::frag(sV[buf], 16 * db + c16, 16 * g + 8 * h));
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) mma16(o[db][qb], va, pf[qb][h]);
        }
    }
    if (next >= 0) stage(buf ^ 1);
    cur = next;
    next = after;
    c = w1 * ks1 * a.scale_log2;
    f = w1 * vs1;
    __syncthreads();
  }
  };
  // a wave without rows only helps to stage the tiles
  if (q0 + 32 * wave < rows) slots(std::true_type{});
  else slots(std::false_type{});
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int qr = query_row(qb);
    if (qr < 0) continue;
    const int64_t row = (int64_t)b * a.L * a.H + qr;
    const float inv = lsum[qb] > 0.f ? F / lsum[qb] : lsum[qb];   // (no slot: 0; NaN passes)
    if (a.nsplit > 1) {
      const int64_t at = (int64_t)sp * a.B * a.L * a.H + row;
#pragma unroll
      for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(a.part + at * kC8Dh + 16 * db + 4 * g) = o[db][qb] * inv;
      if (g == 0) a.lse[at] = lsum[qb] > 0.f ? m[qb] + log2f(lsum[qb]) : lsum[qb] == 0.f ? -INFINITY : lsum[qb];
    } else {
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        bf16x4 v;
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = (bf16)(o[db][qb][x] * inv);
        *reinterpret_cast<bf16x4*>(a.out + row * kC8Dh + 16 * db + 4 * g) = v;
      }
    }
  }
}

// out = sum_i 2^(lse_i - M) o_i / sum_i 2^(lse_i - M) over the splits of a row: 16 lanes of 4 dims per row.
// 6,108 rows: 4.5 us, latency.
__global__ __launch_bounds__(256) void cache8_merge_kernel(const float* __restrict__ part, const float* __restrict__ lse,
                                                           int nsplit, int64_t rows, bf16* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i >> 4;
  if (row >= rows) return;
  const int ch = (int)(i & 15);
  float M = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < nsplit; ++s) M = fmax_fast(M, lse[s * rows + row]);
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  if (!(M == -INFINITY)) {
#pragma unroll 8
    for (int s = 0; s < nsplit; ++s) {
      const float w = c8_exp2(lse[s * rows + row] - M);
      den += w;
      acc += w * *reinterpret_cast<const f32x4*>(part + (s * rows + row) * kC8Dh + 4 * ch);
    }
    acc *= 1.f / den;
  }
  bf16x4 v;
#pragma unroll
  for (int x = 0; x < 4; ++x) v[x] = (bf16)acc[x];
  *reinterpret_cast<bf16x4*>(out + row * kC8Dh + 4 * ch) = v;
}

// Slots of a row block split over workgroups, up to one per CU: a prompt of 509 tokens of 12 heads 24 + 7 us with its
// merge; two per CU 25 + 13 (the f32 part rows), 144 in all 27 + 5.  Blocks of few rows, whose part rows are small: two.
int c8_splits(int64_t B, int64_t L, int H, int HK, int NS) {
  const int64_t rows = L * (H / HK), tiles = B * HK * ((rows + kC8Rows - 1) / kC8Rows);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(NS, 32), (rows <= 64 ? 512 : 256) / std::max<int64_t>(tiles, 1)));
}

// Whether the unit form is taken for several tokens: by estimated times (us).  Unit form: one wave takes the 16-row
// blocks of a chapter that every sequence selects one after the other, ~1 us each, and part rows are written and
// read.  Row blocks: ~1.2 us per slot and workgroup of a CU, and the merge.  Measured, unit form / row blocks, at 65 of 4,097
// chapters: 1 x 64 tokens of 12 heads 17 / 22 us, 4 x 64 35 / 23, 16 x 16 37 / 60, 16 x 64 109 / 60, 64 x 8 80 / 185; 16 heads on
// 4: 8 x 4 18 / 20, 8 x 16 42 / 20, 37 x 8 88 / 41, 37 x 16 165 / 44.
bool c8_units(int64_t B, int64_t L, int H, int HK, int NS) {
  if (L == 1) return true;
  if (B * NS * L >= ((int64_t)1 << 31) / (H / HK)) return false;
  const double rows = (double)L * (H / HK), tiles = (double)B * HK * std::ceil(rows / kC8Rows);
  const double units = 9 + B * rows / 16 + (double)B * NS * L * H * 256 / 5e6;
  const int ns = c8_splits(B, L, H, HK, NS);
  const double blocks = 10 + 1.2 * NS / ns * std::max(1.0, tiles * ns / 256) + (ns > 1 ? 5 : 0);
  return units <= blocks;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
struct C8Ws {
  size_t o_part = 0, lse_part, bytes;
  C8Ws(int64_t B, int64_t L, int H, int HK, int NS) {
    const size_t rows = (size_t)B * L * H;
    if (c8_units(B, L, H, HK, NS)) {
      lse_part = up256(rows * NS * kC8Dh * 2);
      bytes = lse_part + up256(rows * NS * 8);
    } else {
      const int ns = c8_splits(B, L, H, HK, NS);
      lse_part = ns > 1 ? up256(rows * ns * kC8Dh * 4) : 0;
      bytes = ns > 1 ? lse_part + up256(rows * ns * 4) : 0;
    }
  }
};

bool c8_shape_ok(int64_t B, int64_t L, int H, int HK, int NS) {
  if (B < 0 || L <= 0 || H <= 0 || HK <= 0 || H % HK != 0 || NS <= 0) return false;
  const int64_t cap = (int64_t)1 << 31;
  if (B >= cap / NS || L >= ((int64_t)1 << 25) / H) return false;   // edges, and rows of a sequence
  if (c8_units(B, L, H, HK, NS)) return B * NS * L < cap / (H / HK) && B * L * H < cap;   // rows of a unit
  return B * HK * c8_splits(B, L, H, HK, NS) * ((L * (H / HK) + kC8Rows - 1) / kC8Rows) < cap && B * L * H < cap * 8;
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" {

int moc_cache8_pack(int dtype, const void* k, const void* v, int64_t tiles, void* k_tiles, void* v_tiles, float* k_scale,
                    float* v_scale, hipStream_t stream) {
  MOC_REQUIRE(tiles >= 0 && tiles < ((int64_t)1 << 31), MOC_ERR_ARG, "moc_cache8_pack: %lld tiles", (long long)tiles);
  if (tiles == 0) return MOC_OK;
  MOC_REQUIRE(k && v && k_tiles && v_tiles && k_scale && v_scale, MOC_ERR_ARG, "moc_cache8_pack: null pointer");
  MOC_REQUIRE((((uintptr_t)k_tiles | (uintptr_t)v_tiles) & 15) == 0, MOC_ERR_ARG, "moc_cache8_pack: unaligned tiles");
  const dim3 grid((unsigned)tiles, 2);
  if (dtype == MOC_BF16)
    hipLaunchKernelGGL(cache8_pack_kernel<bf16>, grid, dim3(256), 0, stream, (const bf16*)k, (const bf16*)v, (uint8_t*)k_tiles,
                       (uint8_t*)v_tiles, k_scale, v_scale);
  else if (dtype == MOC_F32)
    hipLaunchKernelGGL(cache8_pack_kernel<float>, grid, dim3(256), 0, stream, (const float*)k, (const float*)v,
                       (uint8_t*)k_tiles, (uint8_t*)v_tiles, k_scale, v_scale);
  else
    return set_error(MOC_ERR_UNSUPPORTED, "moc_cache8_pack: dtype %d", dtype);
  return check_launch("cache8_pack_kernel");
}

size_t moc_cache8_attend_workspace(int64_t B, int64_t L, int H, int HK, int NS) {
  return c8_shape_ok(B, L, H, HK, NS) && B > 0 ? C8Ws(B, L, H, HK, NS).bytes : 0;
}

int moc_cache8_attend(const moc_cache8_args* a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  MOC_REQUIRE(a, MOC_ERR_ARG, "moc_cache8_attend: null pointer");
  MOC_REQUIRE(c8_shape_ok(a->B, a->L, a->H, a->HK, a->NS) && a->C > 0 && a->max_u >= 0 &&
                  a->max_u * a->HK < ((int64_t)1 << 32),
              MOC_ERR_ARG, "moc_cache8_attend: B=%lld L=%lld H=%d HK=%d NS=%d C=%lld", (long long)a->B, (long long)a->L, a->H,
              a->HK, a->NS, (long long)a->C);
  if (a->B == 0) return MOC_OK;
  MOC_REQUIRE(a->q && a->k_tiles && a->v_tiles && a->k_scale && a->v_scale && a->idx && a->omega && a->uniq && a->n_uniq &&
                  a->csr_off && a->csr_edge && a->edge_u && a->row_tab && a->out,
              MOC_ERR_ARG, "moc_cache8_attend: null pointer");
  MOC_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->k_tiles | (uintptr_t)a->v_tiles | (uintptr_t)a->out) & 15) == 0, MOC_ERR_ARG,
              "moc_cache8_attend: 16-byte aligned q / tiles / out");
  const C8Ws y(a->B, a->L, a->H, a->HK, a->NS);
  MOC_REQUIRE(y.bytes == 0 || (workspace && workspace_bytes >= y.bytes && ((uintptr_t)workspace & 15) == 0), MOC_ERR_ARG,
              "moc_cache8_attend: workspace %zu < %zu bytes, or unaligned", workspace_bytes, y.bytes);
  char* ws = (char*)workspace;
  const float sl2 = a->scale * 1.4426950408889634f;
  if (c8_units(a->B, a->L, a->H, a->HK, a->NS)) {
    const int64_t units = a->max_u * a->HK;
    if (units > 0) {
      C8Unit k{(const bf16*)a->q, (const uint8_t*)a->k_tiles, (const uint8_t*)a->v_tiles, a->k_scale, a->v_scale, a->omega,
               a->uniq, a->n_uniq, a->csr_off, a->csr_edge, a->row_tab, (f16*)(ws + y.o_part), (float2*)(ws + y.lse_part),
               a->max_u, (int)a->L, a->H, a->HK, a->NS, 0, 0, sl2};
      // division by NS as a product: with s = ceil(log2 NS), floor(2^(31 + s) / NS) + 1 < 2^32 is exact below 2^31
      int s = 0;
      while ((1 << s) < a->NS) ++s;
      k.ns_shift = 31 + s;
      k.ns_mul = (uint32_t)(((uint64_t)1 << (31 + s)) / a->NS + 1);
      hipLaunchKernelGGL(cache8_unit_kernel, dim3((unsigned)((units + kC8Waves - 1) / kC8Waves)), dim3(64 * kC8Waves), 0,
                         stream, k);
      if (int rc = check_launch("cache8_unit_kernel")) return rc;
    }
    const int64_t rows = a->B * a->L * a->H;
    hipLaunchKernelGGL(cache8_combine_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, (const f16*)(ws + y.o_part),
                       (const float2*)(ws + y.lse_part), a->edge_u, a->NS, (int)(a->L * a->H), rows, (bf16*)a->out);
    return check_launch("cache8_combine_kernel");
  }
  const int nsplit = c8_splits(a->B, a->L, a->H, a->HK, a->NS);
  const int64_t nqb = (a->L * (a->H / a->HK) + kC8Rows - 1) / kC8Rows, tiles = a->B * a->HK * nsplit * nqb;
  C8Prompt p{(const bf16*)a->q, (const uint8_t*)a->k_tiles, (const uint8_t*)a->v_tiles, a->k_scale, a->v_scale, a->omega, a->idx,
             (bf16*)a->out, (float*)ws, (float*)(ws + y.lse_part), a->C, (int)a->B, (int)a->L, a->H, a->HK, a->NS, nsplit, sl2};
  hipLaunchKernelGGL(cache8_prompt_kernel, dim3(xcd_grid(tiles)), dim3(kC8Threads), 0, stream, p);
  if (int rc = check_launch("cache8_prompt_kernel")) return rc;
  if (nsplit == 1) return MOC_OK;
  const int64_t rows = a->B * a->L * a->H;
  hipLaunchKernelGGL(cache8_merge_kernel, dim3((unsigned)((rows * 16 + 255) / 256)), dim3(256), 0, stream, (const float*)p.part,
                     (const float*)p.lse, nsplit, rows, (bf16*)a->out);
  return check_launch("cache8_merge_kernel");
}

}  // extern "C"
