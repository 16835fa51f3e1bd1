// Norms of heads with the rotation by position, forward and backward, bound by HBM (each row read once, written once).
//   u = x / sqrt(mean(x^2) + eps) * w;   pair (a, b) of angle t = position * f:  (a cos t - b sin t, b cos t + a sin t)
//   backward: du turns dy back, g = du w, dx = rstd (g - xh mean(g xh)) with xh = x rstd, dw = sum du xh.
//
// A lane owns eight pairs of a head: with halves rotated elements p .. p + 7 and R / 2 + p .. + 7, with interleaved
// pairs (and behind the rotated part) sixteen in a row, so a pair never leaves its lane and the norm's sums are over
// the few neighbouring lanes of the head.  The angles are a token's, not a head's: a workgroup works each one out
// once (f64 product and reduction, whose error of 2^-53 times the position in turns stays below f32's for positions up
// to 2^28; then sin and cos in f32) and its rows read them from LDS.
//
// Measured (forward; backward with the weights' sums): 16 us (62 MB, 3.9 TB/s; a copy of much more runs at 5.2) and 28 + 4
// for 8,192 + 12,000 rows of 12 heads of 64; 33 us (167 MB, 5.0 TB/s) and 63 + 6 (250 MB, 3.9) for 8,156 rows of 32 and 8
// heads of 128 with a weight per head; 5 us for one token, a launch with its angles.
#include "moc_common.h"

namespace moc {

constexpr int kHrThreads = 256;
constexpr int kHrAngles = 4096;    // angles of a workgroup's tokens (32 KB)

struct HrSeg {
  moc_head_rows r;
  int64_t tokens;          // B * L
  int toks;                // of a workgroup's step
  int first;               // first workgroup of the set
  float* part;             // backward: [workgroups][columns] of dw, columns D or H * D
};
struct HrArgs {
  HrSeg seg[3];
  const double* inv_freq;
  int nseg, D, R, R2, interleaved, lph, form;   // R2: pairs, lph: lanes per head, form: HrForm of all rows
  float eps;
};

// Sum over the 2^k lanes of a head
__device__ __forceinline__ float hr_sum(float v, int lph) {
  auto add = [](float x, auto ctrl) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  if (lph > 1) v = add(v, std::integral_constant<int, 0xB1>());    // quad_perm [1, 0, 3, 2]
  if (lph > 2) v = add(v, std::integral_constant<int, 0x4E>());    // quad_perm [2, 3, 0, 1]
  if (lph > 4) v = add(v, std::integral_constant<int, 0x141>());   // row_half_mirror
  if (lph > 8) v = add(v, std::integral_constant<int, 0x140>());   // row_mirror
  if (lph > 16) v += __shfl_xor(v, 16, 64);
  return v;
}

// How rows are read and written: in 16-byte pieces (kWide: every run of eight starts on one, and eight pairs turn
// together or not at all), in the same vectors at 4-byte boundaries (kLoose: any number of rotated dims and odd strides;
// a lane that straddles the rotated part's end still goes one by one), or element by element.  Measured, 16,384 rows of
// 16 bf16 heads of 128 (forward, backward): 31 and 57 us with 128 rotated, 72 rotated 65 and 109 us loose against 118 and
// 196 one by one, 72 rotated in pairs 36 and 64 against 129 and 213.
enum HrForm { kByOne, kLoose, kWide };
typedef uint32_t hr_u32x4 __attribute__((ext_vector_type(4)));
typedef hr_u32x4 hr_loose4 __attribute__((aligned(4)));

// The lane's elements: a = first eight (or even places), b = the others, as a row's two runs of eight
template <typename T, int FORM>
__device__ __forceinline__ void hr_load(const T* p, int e0, int e1, int D, float (&x)[16]) {
  if constexpr (FORM == kWide) {
    ChunkLoadF<T>::run(p + e0, x);
    ChunkLoadF<T>::run(p + e1, x + 8);
  } else if constexpr (FORM == kLoose) {
    constexpr int N = 8 * (int)sizeof(T) / 16;       // vectors of a run
    hr_u32x4 v[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = reinterpret_cast<const hr_loose4*>(p + e0)[i];
      v[N + i] = reinterpret_cast<const hr_loose4*>(p + e1)[i];
    }
    T t[16];
    __builtin_memcpy(t, v, sizeof(t));
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = to_f(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = e0 + i < D ? to_f(p[e0 + i]) : 0.f;
      x[8 + i] = e1 + i < D ? to_f(p[e1 + i]) : 0.f;
    }
  }
}
template <typename T> struct HrStore;
template <> struct HrStore<bf16> {
  static __device__ __forceinline__ void run(bf16* p, const float* v) {
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (bf16)v[i];
    *reinterpret_cast<bf16x8*>(p) = o;
  }
};
template <> struct HrStore<float> {
  static __device__ __forceinline__ void run(float* p, const float* v) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
};

// Where a lane's pairs lie.  In a head of any even D the lane j has pairs 8 j .. 8 j + 7 (of D / 2): rotated halves are
// two runs R / 2 apart, everything else one run of sixteen.  A lane whose pairs straddle the end of the rotated part
// (R not a multiple of 16) takes them one by one: `mixed`.
struct HrLane {
  int p0;         // first pair
  int e0, e1;     // first elements of the two runs
  bool turns, mixed;
};
__device__ __forceinline__ HrLane hr_lane(const HrArgs& a, int j) {
  HrLane l;
  l.p0 = 8 * j;
  l.turns = l.p0 < a.R2;
  l.mixed = !a.interleaved && l.turns && l.p0 + 8 > a.R2;
  const bool halves = l.turns && !a.interleaved;
  l.e0 = halves ? l.p0 : 2 * l.p0;
  l.e1 = halves ? a.R2 + l.p0 : 2 * l.p0 + 8;
  return l;
}
// elements of pair i of a mixed lane
__device__ __forceinline__ void hr_pair(const HrArgs& a, int p, int& e0, int& e1) {
  if (p < a.R2) {
    e0 = p;
    e1 = a.R2 + p;
  } else {
    e0 = 2 * p;
    e1 = 2 * p + 1;
  }
}

template <typename T, int FORM>
__device__ __forceinline__ void hr_read(const HrArgs& a, const HrLane& l, const T* p, float (&x)[16]) {
  if (FORM != kWide && l.mixed) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int e0, e1;
      hr_pair(a, l.p0 + i, e0, e1);
      x[i] = e0 < a.D ? to_f(p[e0]) : 0.f;
      x[8 + i] = e1 < a.D ? to_f(p[e1]) : 0.f;
    }
  } else {
    hr_load<T, FORM>(p, l.e0, l.e1, a.D, x);
  }
}
template <typename T, int FORM>
__device__ __forceinline__ void hr_write(const HrArgs& a, const HrLane& l, T* p, const float (&y)[16]) {
  if (FORM != kWide && l.mixed) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int e0, e1;
      hr_pair(a, l.p0 + i, e0, e1);
      if (e0 < a.D) p[e0] = from_f<T>(y[i]);
      if (e1 < a.D) p[e1] = from_f<T>(y[8 + i]);
    }
  } else if constexpr (FORM == kWide) {
    HrStore<T>::run(p + l.e0, y);
    HrStore<T>::run(p + l.e1, y + 8);
  } else if constexpr (FORM == kLoose) {
    constexpr int N = 8 * (int)sizeof(T) / 16;
    T t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = from_f<T>(y[i]);
    hr_u32x4 v[2 * N];
    __builtin_memcpy(v, t, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      reinterpret_cast<hr_loose4*>(p + l.e0)[i] = v[i];
      reinterpret_cast<hr_loose4*>(p + l.e1)[i] = v[N + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (l.e0 + i < a.D) p[l.e0 + i] = from_f<T>(y[i]);
      if (l.e1 + i < a.D) p[l.e1 + i] = from_f<T>(y[8 + i]);
    }
  }
}

// Turns the lane's pairs by +-angle (dir): pairs lie (i, 8 + i) in halves and mixed lanes, (2 i, 2 i + 1) interleaved.
// Pairs behind the rotated part are left alone: turned by 0, an infinity or NaN in one element would reach the other.
template <int FORM>
__device__ __forceinline__ void hr_turn(const HrArgs& a, const HrLane& l, const float2* cs, float dir, float (&x)[16]) {
  if (!l.turns) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = FORM == kWide || l.p0 + i < a.R2;
    const float2 t = in ? cs[l.p0 + i] : float2{1.f, 0.f};
    const float s = t.y * dir;
    auto turn = [&](float& u, float& v) {
      const float y = u * t.x - v * s, z = v * t.x + u * s;
      u = in ? y : u;
      v = in ? z : v;
    };
    if (a.interleaved)
      turn(x[2 * i], x[2 * i + 1]);
    else
      turn(x[i], x[8 + i]);
  }
}

__device__ __forceinline__ int64_t hr_position(const moc_head_rows& r, int64_t b, int64_t l) {
  int64_t p = l * r.pstep;
  if (r.positions) {
    const int64_t at = b * r.pb + l * r.pl;
    p += r.pos32 ? (int64_t)((const int32_t*)r.positions)[at] : ((const int64_t*)r.positions)[at];
  }
  return p;
}

// cos and sin of tokens t0 .. t0 + n - 1 of a set, [token][pair]
__device__ __forceinline__ void hr_angles(const HrArgs& a, const HrSeg& s, int64_t t0, int n, float2* cs) {
  for (int i = threadIdx.x; i < n * a.R2; i += kHrThreads) {
    const int64_t t = t0 + i / a.R2;
    const double turns = (double)hr_position(s.r, t / s.r.L, t % s.r.L) * (a.inv_freq[i % a.R2] * 0.15915494309189533577);
    float sn, cn;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
    cs[i] = float2{cn, sn};
  }
}

__device__ __forceinline__ int hr_segment(const HrArgs& a) {
  int s = 0;
  while (s + 1 < a.nseg && (int)blockIdx.x >= a.seg[s + 1].first) ++s;
  return s;
}

template <typename T, int FORM>
__global__ __launch_bounds__(kHrThreads) void head_rotate_fwd_kernel(HrArgs a) {
  extern __shared__ float2 cs[];
  const int si = hr_segment(a);
  const HrSeg& s = a.seg[si];
  const moc_head_rows& r = s.r;
  const int64_t t0 = (int64_t)(blockIdx.x - s.first) * s.toks;
  const int n = (int)(s.tokens - t0 < s.toks ? s.tokens - t0 : s.toks);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = lane % a.lph, sub = lane / a.lph, hpw = 64 / a.lph;
  const HrLane ln = hr_lane(a, j);
  const bool lane_on = 16 * j < a.D;
  const int rows = n * r.H;
  auto read = [&](int row, float (&x)[16]) {
    const uint32_t tk = (uint32_t)row / (uint32_t)r.H, h = row - tk * r.H;
    const uint32_t t = (uint32_t)t0 + tk, b = t / (uint32_t)r.L, l = t - b * (uint32_t)r.L;
    hr_read<T, FORM>(a, ln, (const T*)r.x + b * r.xb + l * r.xl + h * r.xh, x);
  };
  // (a row is requested before the angles are worked out, and then a row ahead of the one in hand)
  float next[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) next[i] = 0.f;
  int row = wave * hpw + sub;
  if (lane_on && row < rows) read(row, next);
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = 1.f;
  if (r.w && !r.w_head && lane_on) hr_read<float, FORM>(a, ln, r.w, w);
  if (r.rotate) {
    hr_angles(a, s, t0, n, cs);
    __syncthreads();
  }
  for (; row < rows; row += 4 * hpw) {
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = next[i];
    if (lane_on && row + 4 * hpw < rows) read(row + 4 * hpw, next);
    const uint32_t tk = (uint32_t)row / (uint32_t)r.H, h = row - tk * r.H;
    const uint32_t t = (uint32_t)t0 + tk, b = t / (uint32_t)r.L, l = t - b * (uint32_t)r.L;
    if (r.norm) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) sq += x[i] * x[i];
      const float rstd = 1.f / sqrtf(hr_sum(sq, a.lph) / (float)a.D + a.eps);
      if (r.w_head && lane_on) hr_read<float, FORM>(a, ln, r.w + (int64_t)h * a.D, w);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = x[i] * rstd * w[i];
    }
    if (r.rotate) hr_turn<FORM>(a, ln, cs + tk * a.R2, 1.f, x);
    int64_t at = b * r.yb + l * r.yl;
    if (r.page) {       // (a table without columns has no address: it is the page that says where rows go)
      const int64_t p = hr_position(r, b, l), pg = p < 0 ? r.max_pages : p / r.page;
      const int id = pg < r.max_pages ? r.table[b * r.tb + pg] : -1;
      if (id < 0 || id >= r.num_pages) continue;     // (the whole head's lanes)
      at = id * r.yb + (p % r.page) * r.yl;
    }
    if (lane_on) hr_write<T, FORM>(a, ln, (T*)r.y + at + h * r.yh, x);
  }
}

// Backward: a workgroup goes over its share of the tokens, `toks` at a time, for one group of heads (those of a wave's
// lanes, so that a lane's sums for dw belong to one head); its sums of dw go to its row of `part`.
template <typename T, int FORM>
__global__ __launch_bounds__(kHrThreads) void head_rotate_bwd_kernel(HrArgs a, int wgs0, int wgs1, int wgs2) {
  extern __shared__ float2 cs[];                      // the angles, and at the end
  float (*red)[64 * 16] = reinterpret_cast<float (*)[64 * 16]>(cs);   // the waves' sums of dw
  const int si = hr_segment(a);
  const HrSeg& s = a.seg[si];
  const moc_head_rows& r = s.r;
  const int wgs = si == 0 ? wgs0 : si == 1 ? wgs1 : wgs2, wg = blockIdx.x - s.first;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = lane % a.lph, sub = lane / a.lph, hpw = 64 / a.lph;
  const HrLane ln = hr_lane(a, j);
  const bool lane_on = 16 * j < a.D;
  // weight per head: workgroups of one head group; else a row is any head of any token
  const int ngrp = r.w_head ? (r.H + hpw - 1) / hpw : 1;
  const int grp = wg % ngrp, slice = wg / ngrp, nslice = wgs / ngrp;
  const int h_lane = grp * hpw + sub;
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    w[i] = 1.f;
    dw[i] = 0.f;
  }
  if (r.w && lane_on && (!r.w_head || h_lane < r.H))
    hr_read<float, FORM>(a, ln, r.w + (r.w_head ? (int64_t)h_lane * a.D : 0), w);
  const int64_t steps = (s.tokens + s.toks - 1) / s.toks;
  const int per = r.w_head ? hpw : r.H;               // rows of a token that the workgroup takes
  for (int64_t st = slice; st < steps; st += nslice) {
    const int64_t t0 = st * s.toks;
    const int n = (int)(s.tokens - t0 < s.toks ? s.tokens - t0 : s.toks), rows = n * per;
    auto at = [&](int row, uint32_t& tk, uint32_t& h, uint32_t& b, uint32_t& l) {
      tk = (uint32_t)row / (uint32_t)per;
      h = r.w_head ? (uint32_t)h_lane : row - tk * per;
      const uint32_t t = (uint32_t)t0 + tk;
      b = t / (uint32_t)r.L;
      l = t - b * (uint32_t)r.L;
    };
    auto read = [&](int row, float (&g)[16], float (&x)[16]) {
      uint32_t tk, h, b, l;
      at(row, tk, h, b, l);
      if (!lane_on || h >= (uint32_t)r.H) return;
      hr_read<T, FORM>(a, ln, (const T*)r.dy + b * r.yb + l * r.yl + h * r.yh, g);
      if (r.norm) hr_read<T, FORM>(a, ln, (const T*)r.x + b * r.xb + l * r.xl + h * r.xh, x);
    };
    float gn[16], xn[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) gn[i] = xn[i] = 0.f;
    int row = wave * hpw + sub;
    if (row < rows) read(row, gn, xn);
    if (r.rotate) {
      __syncthreads();
      hr_angles(a, s, t0, n, cs);
      __syncthreads();
    }
    for (; row < rows; row += 4 * hpw) {
      float g[16], x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        g[i] = gn[i];
        x[i] = xn[i];
      }
      if (row + 4 * hpw < rows) read(row + 4 * hpw, gn, xn);
      uint32_t tk, h, b, l;
      at(row, tk, h, b, l);
      if (h >= (uint32_t)r.H) continue;
      if (r.rotate) hr_turn<FORM>(a, ln, cs + tk * a.R2, -1.f, g);
      if (r.norm) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sq += x[i] * x[i];
        const float rstd = 1.f / sqrtf(hr_sum(sq, a.lph) / (float)a.D + a.eps);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] *= rstd;
          dw[i] += g[i] * x[i];
          g[i] *= w[i];
          dot += g[i] * x[i];
        }
        const float mean = hr_sum(dot, a.lph) / (float)a.D;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = rstd * (g[i] - x[i] * mean);
      }
      if (r.dx && lane_on) hr_write<T, FORM>(a, ln, (T*)r.dx + ((t0 + tk) * r.H + h) * a.D, g);
    }
  }
  if (!s.part) return;
  // this workgroup's sums: over its waves, and over the heads where they share the weight
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) red[wave][lane * 16 + i] = dw[i];
  __syncthreads();
  const int cols = r.w_head ? hpw * a.D : a.D;
  for (int c = threadIdx.x; c < cols; c += kHrThreads) {
    const int e = c % a.D, h0 = c / a.D;
    // the lane and place of element e
    int p, half;
    if (e < a.R && !a.interleaved) {
      p = e < a.R2 ? e : e - a.R2;
      half = e < a.R2 ? 0 : 1;
    } else {
      p = e / 2;
      half = e % 2;
    }
    const HrLane o = hr_lane(a, p / 8);
    const bool split = o.turns && !a.interleaved;       // places (i, 8 + i), else (2 i, 2 i + 1)
    const int place = split ? p % 8 + 8 * half : 2 * (p % 8) + half;
    float sum = 0.f;
    const int s0 = r.w_head ? h0 : 0, s1 = r.w_head ? h0 + 1 : hpw;
    for (int q = s0; q < s1; ++q)
      for (int v = 0; v < 4; ++v) sum += red[v][(q * a.lph + p / 8) * 16 + place];
    if (r.w_head) {
      if (grp * hpw + h0 < r.H) s.part[((int64_t)slice * r.H + grp * hpw + h0) * a.D + e] = sum;
    } else {
      s.part[(int64_t)slice * a.D + e] = sum;
    }
  }
}

// dw of each set: sums over the slices, in their order: 16 columns per workgroup, 64 threads each
__global__ __launch_bounds__(1024) void head_rotate_dw_kernel(HrArgs a, int n0, int n1, int n2) {
  __shared__ float red[64][17];
  int blk = blockIdx.x, si = 0, cols = 0;
  for (; si < a.nseg; ++si) {
    const moc_head_rows& r = a.seg[si].r;
    cols = !a.seg[si].part ? 0 : r.w_head ? r.H * a.D : a.D;
    const int nb = (cols + 15) / 16;
    if (blk < nb) break;
    blk -= nb;
  }
  const HrSeg& s = a.seg[si];
  const int n = si == 0 ? n0 : si == 1 ? n1 : n2;
  const int c = 16 * blk + (threadIdx.x & 15), q = threadIdx.x >> 4;
  float sum = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int i = q; i < n; i += 64) sum += s.part[(int64_t)i * cols + c];
  }
  red[q][threadIdx.x & 15] = sum;
  __syncthreads();
  if (q == 0 && c < cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) t += red[i][threadIdx.x & 15];
    s.r.dw[c] = t;
  }
}

static int hr_check(const char* who, const moc_head_args* p, bool bwd, HrArgs* o) {
  MOC_REQUIRE(p != nullptr, MOC_ERR_ARG, "%s: no arguments", who);
  const moc_head_args& a = *p;
  MOC_REQUIRE(a.dtype == MOC_F32 || a.dtype == MOC_BF16, MOC_ERR_ARG, "%s: dtype %d", who, a.dtype);
  MOC_REQUIRE(a.nseg >= 1 && a.nseg <= 3, MOC_ERR_ARG, "%s: %d sets", who, a.nseg);
  MOC_REQUIRE(a.D >= 2 && a.D <= 512 && a.D % 2 == 0, MOC_ERR_UNSUPPORTED, "%s: head dim %d, expected even, 2 .. 512", who, a.D);
  MOC_REQUIRE(a.R >= 0 && a.R <= a.D && a.R % 2 == 0, MOC_ERR_ARG, "%s: %d rotated dims of %d", who, a.R, a.D);
  const int es = dtype_size(a.dtype);
  HrArgs& h = *o;
  h = HrArgs{};
  h.inv_freq = a.inv_freq;
  h.nseg = a.nseg; h.D = a.D; h.R = a.R; h.R2 = a.R / 2; h.interleaved = a.interleaved ? 1 : 0; h.eps = a.eps;
  h.lph = 1;
  h.form = kWide;
  while (16 * h.lph < a.D) h.lph *= 2;
  for (int i = 0; i < a.nseg; ++i) {
    const moc_head_rows& r = a.seg[i];
    MOC_REQUIRE(r.B >= 0 && r.L >= 0 && r.H > 0 && r.H <= 1 << 16, MOC_ERR_ARG, "%s: bad sizes", who);
    MOC_REQUIRE(r.B == 0 || r.L < ((int64_t)1 << 31) / r.B, MOC_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 tokens", who);
    const bool empty = r.B * r.L == 0;
    MOC_REQUIRE(r.page >= 0 && (r.page > 0 ? !bwd && r.max_pages >= 0 && r.num_pages >= 0 && (r.table || r.max_pages == 0 || empty)
                                           : !r.table),
                MOC_ERR_ARG, "%s: bad pages", who);
    const bool nowhere = r.page > 0 && (r.max_pages == 0 || r.num_pages == 0);     // (no row has a place)
    MOC_REQUIRE(empty || (bwd ? (r.dy && (r.x || !r.norm)) : (r.x && (r.y || nowhere))), MOC_ERR_ARG, "%s: null tensor", who);
    MOC_REQUIRE(!r.rotate || a.R == 0 || a.inv_freq, MOC_ERR_ARG, "%s: a rotation needs its frequencies", who);
    MOC_REQUIRE(r.norm || !r.w, MOC_ERR_ARG, "%s: a weight without a norm", who);
    HrSeg& s = h.seg[i];
    s.r = r;
    s.r.w_head = r.w && r.w_head ? 1 : 0;
    s.r.rotate = r.rotate && a.R > 0 ? 1 : 0;
    s.tokens = r.B * r.L;
    const int64_t st[] = {r.xb, r.xl, r.xh, r.yb, r.yl, r.yh};
    bool wide = a.D % 16 == 0 && a.R % 16 == 0, loose = a.D % 16 == 0 && (h.interleaved || es == 4 || a.R % 4 == 0);
    for (int64_t x : st) {
      wide = wide && x * es % 16 == 0;
      loose = loose && x * es % 4 == 0;
    }
    const void* ps[] = {r.x, r.y, r.dy, r.dx, r.w};
    for (const void* x : ps) {
      wide = wide && ((uintptr_t)x & 15) == 0;
      loose = loose && ((uintptr_t)x & 3) == 0;
    }
    const int form = wide ? kWide : loose ? kLoose : kByOne;
    if (form < h.form) h.form = form;
  }
  return MOC_OK;
}

// Tokens of a workgroup's step: their angles fit LDS, their rows (`per` of a token) keep each lane busy for about four
// rows, behind which the start of a workgroup and its angles disappear (8,192 + 12,000 rows of 12 heads of 64 in 8, 16 and
// 32 tokens: forward 17.4, 15.6, 19.0 us; 8,156 of 32 + 8 heads of 128: 31.8, 35.3, 56), and a small launch has
// workgroups on every CU.
static int hr_tokens(const HrArgs& h, const HrSeg& s, int per) {
  int64_t total = 0;
  for (int i = 0; i < h.nseg; ++i) total += h.seg[i].tokens;
  int64_t t = 4 * kHrThreads / ((int64_t)per * h.lph);
  const int64_t most = h.R2 ? kHrAngles / h.R2 : 16;
  if (t > 16) t = 16;
  if (t > most) t = most;
  if (t > total / 512) t = total / 512;
  return t < 1 ? 1 : (int)t;
}

template <typename T>
static void hr_fwd_launch(const HrArgs& a, unsigned grid, size_t lds, hipStream_t stream) {
  if (a.form == kWide)
    head_rotate_fwd_kernel<T, kWide><<<grid, kHrThreads, lds, stream>>>(a);
  else if (a.form == kLoose)
    head_rotate_fwd_kernel<T, kLoose><<<grid, kHrThreads, lds, stream>>>(a);
  else
    head_rotate_fwd_kernel<T, kByOne><<<grid, kHrThreads, lds, stream>>>(a);
}
template <typename T>
static void hr_bwd_launch(const HrArgs& a, int grid, size_t lds, const int (&wgs)[3], hipStream_t stream) {
  if (a.form == kWide)
    head_rotate_bwd_kernel<T, kWide><<<grid, kHrThreads, lds, stream>>>(a, wgs[0], wgs[1], wgs[2]);
  else if (a.form == kLoose)
    head_rotate_bwd_kernel<T, kLoose><<<grid, kHrThreads, lds, stream>>>(a, wgs[0], wgs[1], wgs[2]);
  else
    head_rotate_bwd_kernel<T, kByOne><<<grid, kHrThreads, lds, stream>>>(a, wgs[0], wgs[1], wgs[2]);
}

// Workgroups of each set's backward: up to 512 slices of its tokens, times the head groups of weights per head.
static void hr_bwd_plan(HrArgs& h, int (&slices)[3], int (&wgs)[3], size_t (&part)[3]) {
  for (int i = 0; i < 3; ++i) {
    slices[i] = wgs[i] = 0;
    part[i] = 0;
    if (i >= h.nseg) continue;
    HrSeg& s = h.seg[i];
    const int hpw = 64 / h.lph, ngrp = s.r.w_head ? (s.r.H + hpw - 1) / hpw : 1;
    s.toks = hr_tokens(h, s, s.r.w_head ? hpw : s.r.H);
    const int64_t steps = (s.tokens + s.toks - 1) / s.toks;
    int64_t n = 512 / ngrp;
    if (n < 64) n = 64;
    if (n > steps) n = steps;
    if (n < 1) n = 1;
    slices[i] = (int)n;
    wgs[i] = (int)n * ngrp;
    part[i] = s.r.w && s.r.dw ? (size_t)n * (s.r.w_head ? (size_t)s.r.H * h.D : h.D) : 0;
  }
}

}  // namespace moc

using namespace moc;

extern "C" {

int moc_head_rotate_fwd(const moc_head_args* args, hipStream_t stream) {
  HrArgs a;
  int rc = hr_check("moc_head_rotate_fwd", args, false, &a);
  if (rc != MOC_OK) return rc;
  int64_t grid = 0;
  size_t lds = 0;
  for (int i = 0; i < a.nseg; ++i) {
    HrSeg& s = a.seg[i];
    s.toks = hr_tokens(a, s, s.r.H);
    s.first = (int)grid;
    grid += (s.tokens + s.toks - 1) / s.toks;
    if (lds < (size_t)s.toks * a.R2 * 8) lds = (size_t)s.toks * a.R2 * 8;
  }
  MOC_REQUIRE(grid < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "moc_head_rotate_fwd: too many tokens");
  if (grid == 0) return MOC_OK;
  if (args->dtype == MOC_BF16)
    hr_fwd_launch<bf16>(a, (unsigned)grid, lds, stream);
  else
    hr_fwd_launch<float>(a, (unsigned)grid, lds, stream);
  return check_launch("moc_head_rotate_fwd");
}

size_t moc_head_rotate_bwd_workspace(const moc_head_args* args) {
  HrArgs a;
  if (hr_check("moc_head_rotate_bwd", args, true, &a) != MOC_OK) return 0;
  int slices[3], wgs[3];
  size_t part[3];
  hr_bwd_plan(a, slices, wgs, part);
  return 4 * (part[0] + part[1] + part[2]);
}

int moc_head_rotate_bwd(const moc_head_args* args, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  HrArgs a;
  int rc = hr_check("moc_head_rotate_bwd", args, true, &a);
  if (rc != MOC_OK) return rc;
  int slices[3], wgs[3];
  size_t part[3];
  hr_bwd_plan(a, slices, wgs, part);
  const size_t need = 4 * (part[0] + part[1] + part[2]);
  MOC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), MOC_ERR_ARG, "moc_head_rotate_bwd: workspace of %zu bytes, needs %zu",
              workspace_bytes, need);
  float* ws = (float*)workspace;
  int grid = 0, cols = 0;
  size_t lds = 0;
  for (int i = 0; i < a.nseg; ++i) {
    HrSeg& s = a.seg[i];
    s.first = grid;
    grid += wgs[i];
    if (lds < (size_t)s.toks * a.R2 * 8) lds = (size_t)s.toks * a.R2 * 8;
    s.part = part[i] ? ws : nullptr;
    ws += part[i];
    if (part[i]) cols += ((s.r.w_head ? s.r.H * a.D : a.D) + 15) / 16;
  }
  if (cols && lds < 4 * 64 * 16 * 4) lds = 4 * 64 * 16 * 4;
  if (args->dtype == MOC_BF16)
    hr_bwd_launch<bf16>(a, grid, lds, wgs, stream);
  else
    hr_bwd_launch<float>(a, grid, lds, wgs, stream);
  rc = check_launch("moc_head_rotate_bwd");
  if (rc != MOC_OK || cols == 0) return rc;
  head_rotate_dw_kernel<<<cols, 1024, 0, stream>>>(a, slices[0], slices[1], slices[2]);
  return check_launch("moc_head_rotate_bwd: weights");
}

}  // extern "C"
