// The end of a sublayer and the norm in front of the next one, in one pass over the rows:
//   u = norm(x) w1 + b1           (the norm after the block; without it u = x)
//   h = alpha r + g u             (residual stream r, gate g: none, one scalar, per channel, per row, per element)
//   n = norm(h) w2 + b2           (the next sublayer's norm; optional)
// norm(y) = (y - mu) / sqrt(mean((y - mu)^2) + eps), mu = mean(y) for LayerNorm and 0 for RMSNorm.
// Everything between the loads and the stores is f32: h and n are rounded once, n from the unrounded h.
//
// Backward, with xh, hh the standardised rows, rs their 1 / deviation, m(.) the row mean:
//   g2 = dn w2,  dH = dh + rs2 (g2 - m(g2) [LayerNorm] - hh m(g2 hh)),  dr = alpha dH
//   dg = dH u (summed over what the gate was broadcast over),  du = g dH,  g1 = du w1
//   dx = rs1 (g1 - m(g1) [LayerNorm] - xh m(g1 xh))
//   dw1 = sum_rows du xh, db1 = sum_rows du, dw2 = sum_rows dn hh, db2 = sum_rows dn
// h is formed again from x and r (not read back rounded), so the backward reads x, r, dh, dn and
// writes dx, dr.  A workgroup takes a strip of rows and keeps the column sums of its strip in
// registers; the strips' sums are added in a fixed order by a second kernel (deterministic).
//
// Bound: HBM.  A row is held by W waves (VEC elements per load, KCH loads per lane).
#include <algorithm>

#include "moc_common.h"

namespace moc {
namespace {

constexpr int kGnMaxD = 16384;

template <typename T, int VEC> struct GnVec;
template <> struct GnVec<float, 8> { typedef f32x8 type; };
template <> struct GnVec<bf16, 8> { typedef bf16x8 type; };
template <> struct GnVec<float, 1> { typedef float type; };
template <> struct GnVec<bf16, 1> { typedef bf16 type; };

template <typename T, int VEC> __device__ __forceinline__ float gn_get(const typename GnVec<T, VEC>::type& v, int e) {
  if constexpr (VEC == 1) return (float)v;
  else return (float)v[e];
}

template <typename T, int VEC>
__device__ __forceinline__ void gn_store(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f<T>(v[0]);
  } else {
    typename GnVec<T, VEC>::type o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = from_f<T>(v[e]);
    *reinterpret_cast<typename GnVec<T, VEC>::type*>(p) = o;
  }
}

// sums of N values over the W waves of a row, the same bits in every lane
template <int W, int N>
__device__ __forceinline__ void gn_row_sum(float (&v)[N], float* red, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (W > 1) {
    __syncthreads();   // the previous sums have been read
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += red[w * N + i];
      v[i] = s;
    }
  }
}

__device__ __forceinline__ float gn_gate_row(const moc_gated_norm& a, int64_t r) {
  if (a.gate_mode == MOC_GATE_SCALAR) return a.gate_dtype == MOC_F32 ? *(const float*)a.gate : (float)*(const bf16*)a.gate;
  if (a.gate_mode == MOC_GATE_TOKEN) return a.gate_dtype == MOC_F32 ? ((const float*)a.gate)[r] : (float)((const bf16*)a.gate)[r];
  return 1.f;
}

template <typename TX, typename TR, int VEC, int W, int KCH, bool FULL>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void gated_norm_fwd_kernel(moc_gated_norm a) {
  constexpr int RPB = W == 1 ? 4 : 1;   // rows of a workgroup
  __shared__ float red[W * 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = (int64_t)blockIdx.x * RPB + (W == 1 ? wave : 0);
  if (r >= a.rows) return;   // (W > 1: uniform over the workgroup)
  const int t = W == 1 ? lane : (int)threadIdx.x;
  const int d = (int)a.d, nch = d / VEC;
  const TX* xr = (const TX*)a.x + r * d;
  const TR* rr = (const TR*)a.residual + r * d;
  typename GnVec<TX, VEC>::type xv[KCH], gv[KCH];
  typename GnVec<TR, VEC>::type rv[KCH];
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    if (c < nch) {
      xv[i] = *reinterpret_cast<const typename GnVec<TX, VEC>::type*>(xr + VEC * c);
      rv[i] = *reinterpret_cast<const typename GnVec<TR, VEC>::type*>(rr + VEC * c);
      if constexpr (FULL) gv[i] = *reinterpret_cast<const typename GnVec<TX, VEC>::type*>((const TX*)a.gate + r * d + VEC * c);
    }
  }
  const float inv_d = 1.f / (float)d;
  float h[KCH][VEC];
#pragma unroll
  for (int i = 0; i < KCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[i][e] = t + 64 * W * i < nch ? gn_get<TX, VEC>(xv[i], e) : 0.f;
  float mu = 0.f, rs = 1.f;
  auto stats = [&](int norm, float eps) {
    mu = 0.f;
    if (norm == MOC_NORM_LAYERNORM) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < KCH; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0] += h[i][e];
      gn_row_sum<W, 1>(s, red, wave, lane);
      mu = s[0] * inv_d;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < KCH; ++i)
      if (t + 64 * W * i < nch) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = h[i][e] - mu;
          q[0] += v * v;
        }
      }
    gn_row_sum<W, 1>(q, red, wave, lane);
    rs = 1.f / sqrtf(q[0] * inv_d + eps);
  };
  if (a.post) {
    stats(a.norm, a.eps);
    if (a.stats && t == 0) {
      a.stats[r] = mu;
      a.stats[a.rows + r] = rs;
    }
  }
  const float grow = gn_gate_row(a, r);
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    if (c >= nch) continue;
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int j = VEC * c + e;
      float u = h[i][e];
      if (a.post) {
        u = (u - mu) * rs;
        if (a.w1) u *= a.w1[j];
        if (a.b1) u += a.b1[j];
      }
      float g = grow;
      if constexpr (FULL) g = gn_get<TX, VEC>(gv[i], e);
      else if (a.gate_mode == MOC_GATE_CHANNEL) g = ((const float*)a.gate)[j];
      o[e] = h[i][e] = a.alpha * gn_get<TR, VEC>(rv[i], e) + g * u;
    }
    gn_store<TR, VEC>((TR*)a.h + r * d + VEC * c, o);
  }
  if (!a.pre) return;
  stats(a.norm2, a.eps2);
  if (a.stats && t == 0) {
    a.stats[2 * a.rows + r] = mu;
    a.stats[3 * a.rows + r] = rs;
  }
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    if (c >= nch) continue;
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int j = VEC * c + e;
      float v = (h[i][e] - mu) * rs;
      if (a.w2) v *= a.w2[j];
      if (a.b2) v += a.b2[j];
      o[e] = v;
    }
    gn_store<TX, VEC>((TX*)a.n + r * d + VEC * c, o);
  }
}

// Column sums kept per strip: part[strip][q][d], q = dw1, db1, dw2, db2, dg (channel).  The scalar
// gate's gradient is summed per strip into scal[strip].
template <typename TX, typename TR, int VEC, int W, int KCH, bool FULL>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void gated_norm_bwd_kernel(moc_gated_norm a, moc_gated_norm_grads o,
                                                                               float* __restrict__ part,
                                                                               float* __restrict__ scal) {
  constexpr int RPB = W == 1 ? 4 : 1;
  constexpr int kQ = 5;
  __shared__ float red[W * 3];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = W == 1 ? lane : (int)threadIdx.x;
  const int d = (int)a.d, nch = d / VEC;
  const float inv_d = 1.f / (float)d;
  const bool layer = a.norm == MOC_NORM_LAYERNORM, layer2 = a.norm2 == MOC_NORM_LAYERNORM;
  float acc[kQ][KCH][VEC];
#pragma unroll
  for (int q = 0; q < kQ; ++q)
#pragma unroll
    for (int i = 0; i < KCH; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[q][i][e] = 0.f;
  float dscal = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * RPB + (W == 1 ? wave : 0); r < a.rows; r += (int64_t)gridDim.x * RPB) {
    typename GnVec<TX, VEC>::type xv[KCH], gv[KCH], nv[KCH];
    typename GnVec<TR, VEC>::type rv[KCH], hv[KCH];
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + 64 * W * i;
      if (c < nch) {
        const int64_t at = r * d + VEC * c;
        xv[i] = *reinterpret_cast<const typename GnVec<TX, VEC>::type*>((const TX*)a.x + at);
        rv[i] = *reinterpret_cast<const typename GnVec<TR, VEC>::type*>((const TR*)a.residual + at);
        if (o.dh) hv[i] = *reinterpret_cast<const typename GnVec<TR, VEC>::type*>((const TR*)o.dh + at);
        if (o.dn) nv[i] = *reinterpret_cast<const typename GnVec<TX, VEC>::type*>((const TX*)o.dn + at);
        if constexpr (FULL) gv[i] = *reinterpret_cast<const typename GnVec<TX, VEC>::type*>((const TX*)a.gate + at);
      }
    }
    const float mu1 = a.post ? a.stats[r] : 0.f, rs1 = a.post ? a.stats[a.rows + r] : 1.f;
    const float mu2 = o.dn ? a.stats[2 * a.rows + r] : 0.f, rs2 = o.dn ? a.stats[3 * a.rows + r] : 0.f;
    const float grow = gn_gate_row(a, r);
    float xh[KCH][VEC], hh[KCH][VEC], g2[KCH][VEC];
    float s[3] = {0.f, 0.f, 0.f};
    auto gate_of = [&](int i, int e, int j) {
      if constexpr (FULL) return gn_get<TX, VEC>(gv[i], e);
      else return a.gate_mode == MOC_GATE_CHANNEL ? ((const float*)a.gate)[j] : grow;
    };
    auto u_of = [&](float v, int j) {
      if (a.post) {
        if (a.w1) v *= a.w1[j];
        if (a.b1) v += a.b1[j];
      }
      return v;
    };
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + 64 * W * i;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        xh[i][e] = hh[i][e] = g2[i][e] = 0.f;
        if (c < nch) {
          const int j = VEC * c + e;
          xh[i][e] = (gn_get<TX, VEC>(xv[i], e) - mu1) * rs1;
          if (o.dn) {
            const float h = a.alpha * gn_get<TR, VEC>(rv[i], e) + gate_of(i, e, j) * u_of(xh[i][e], j);
            hh[i][e] = (h - mu2) * rs2;
            const float dn = gn_get<TX, VEC>(nv[i], e);
            acc[2][i][e] += dn * hh[i][e];
            acc[3][i][e] += dn;
            g2[i][e] = a.w2 ? dn * a.w2[j] : dn;
            s[0] += g2[i][e];
            s[1] += g2[i][e] * hh[i][e];
          }
        }
      }
    }
    if (o.dn) gn_row_sum<W, 3>(s, red, wave, lane);
    const float c0 = layer2 ? s[0] * inv_d : 0.f, c1 = s[1] * inv_d;
    float p[3] = {0.f, 0.f, 0.f};
    // g2 becomes dH, hh becomes g1 = du w1
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + 64 * W * i;
      if (c >= nch) continue;
      float dr[VEC], dg[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int j = VEC * c + e;
        float dH = rs2 * (g2[i][e] - c0 - hh[i][e] * c1);
        if (o.dh) dH += gn_get<TR, VEC>(hv[i], e);
        dr[e] = a.alpha * dH;
        const float u = u_of(xh[i][e], j);
        dg[e] = dH * u;
        p[2] += dg[e];
        const float du = gate_of(i, e, j) * dH;
        if (a.gate_mode == MOC_GATE_CHANNEL) acc[4][i][e] += dg[e];
        acc[0][i][e] += du * xh[i][e];
        acc[1][i][e] += du;
        const float g1 = a.post && a.w1 ? du * a.w1[j] : du;
        hh[i][e] = g1;
        p[0] += g1;
        p[1] += g1 * xh[i][e];
      }
      if (o.dres) gn_store<TR, VEC>((TR*)o.dres + r * d + VEC * c, dr);
      if constexpr (FULL) {
        if (o.dgate) gn_store<TX, VEC>((TX*)o.dgate + r * d + VEC * c, dg);
      }
    }
    gn_row_sum<W, 3>(p, red, wave, lane);
    if (a.gate_mode == MOC_GATE_SCALAR) dscal += p[2];
    if (a.gate_mode == MOC_GATE_TOKEN && o.dgate && t == 0) {
      if (a.gate_dtype == MOC_F32) ((float*)o.dgate)[r] = p[2];
      else ((bf16*)o.dgate)[r] = (bf16)p[2];
    }
    if (o.dx) {
      const float e0 = layer && a.post ? p[0] * inv_d : 0.f, e1 = a.post ? p[1] * inv_d : 0.f;
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        const int c = t + 64 * W * i;
        if (c >= nch) continue;
        float dx[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) dx[e] = rs1 * (hh[i][e] - e0 - xh[i][e] * e1);
        gn_store<TX, VEC>((TX*)o.dx + r * d + VEC * c, dx);
      }
    }
  }
  // the strip's column sums: W == 1 adds the four waves' sums through LDS, in wave order
  const int64_t strip = blockIdx.x;
  if constexpr (W == 1) {
    extern __shared__ float buf[];   // [d]
    for (int q = 0; q < kQ; ++q) {
      for (int w = 0; w < 4; ++w) {
        if (wave == w) {
#pragma unroll
          for (int i = 0; i < KCH; ++i) {
            const int c = lane + 64 * i;
            if (c < nch) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                const float v = acc[q][i][e];
                if (w == 0) buf[VEC * c + e] = v;
                else buf[VEC * c + e] += v;
              }
            }
          }
        }
        __syncthreads();
      }
      for (int j = threadIdx.x; j < d; j += 256) part[(strip * kQ + q) * d + j] = buf[j];
      __syncthreads();
    }
    if (a.gate_mode == MOC_GATE_SCALAR) {
      if (lane == 0) buf[wave] = dscal;
      __syncthreads();
      if (threadIdx.x == 0) scal[strip] = ((buf[0] + buf[1]) + buf[2]) + buf[3];
    }
  } else {
#pragma unroll
    for (int q = 0; q < kQ; ++q)
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        const int c = t + 64 * W * i;
        if (c < nch) gn_store<float, VEC>(part + (strip * kQ + q) * d + VEC * c, acc[q][i]);
      }
    if (a.gate_mode == MOC_GATE_SCALAR && t == 0) scal[strip] = dscal;
  }
}

// grads[q][j] = sum over the strips, in strip order within eight interleaved groups that are then added in
// order.  64 columns per workgroup.
__global__ __launch_bounds__(512) void gated_norm_cols_kernel(const float* __restrict__ part, int strips, int64_t n,
                                                              float* __restrict__ out, const float* __restrict__ scal,
                                                              float* __restrict__ dscal) {
  __shared__ float buf[8][64];
  const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (j < n)
    for (int i = grp; i < strips; i += 8) s += part[(int64_t)i * n + j];
  buf[grp][lane] = s;
  __syncthreads();
  if (grp == 0 && j < n) {
    float v = buf[0][lane];
#pragma unroll
    for (int g = 1; g < 8; ++g) v += buf[g][lane];
    out[j] = v;
  }
  if (dscal && blockIdx.x == 0 && grp == 1) {
    float v = 0.f;
    for (int i = lane; i < strips; i += 64) v += scal[i];
    v = wave_sum(v);
    if (lane == 0) *dscal = v;
  }
}

// waves per row, and the strips of the backward: 512 workgroups put two on every CU
int gn_waves(int64_t d, bool vec) { return vec ? (d <= 1024 ? 1 : d <= 8192 ? 4 : 16) : (d <= 512 ? 1 : d <= 2048 ? 4 : 16); }
int64_t gn_strips(int64_t rows, int64_t d, bool vec) {
  const int rpb = gn_waves(d, vec) == 1 ? 4 : 1;
  return std::max<int64_t>(1, std::min<int64_t>((rows + rpb - 1) / rpb, 512));
}

int gn_check(const char* who, const moc_gated_norm* a) {
  MOC_REQUIRE(a && (a->rows == 0 || (a->x && a->residual)), MOC_ERR_ARG, "%s: null pointer", who);
  MOC_REQUIRE(a->rows >= 0 && a->d > 0 && a->d <= kGnMaxD, MOC_ERR_UNSUPPORTED, "%s: rows=%lld d=%lld (d up to %d)", who,
              (long long)a->rows, (long long)a->d, kGnMaxD);
  MOC_REQUIRE(a->rows < ((int64_t)1 << 31), MOC_ERR_UNSUPPORTED, "%s: rows=%lld", who, (long long)a->rows);
  MOC_REQUIRE((a->norm == MOC_NORM_RMS || a->norm == MOC_NORM_LAYERNORM) &&
                  (a->norm2 == MOC_NORM_RMS || a->norm2 == MOC_NORM_LAYERNORM),
              MOC_ERR_ARG, "%s: norm %d, %d", who, a->norm, a->norm2);
  MOC_REQUIRE(dtype_size(a->x_dtype) && dtype_size(a->r_dtype), MOC_ERR_UNSUPPORTED, "%s: dtypes x %d residual %d", who,
              a->x_dtype, a->r_dtype);
  MOC_REQUIRE(a->gate_mode >= MOC_GATE_NONE && a->gate_mode <= MOC_GATE_FULL && (a->gate_mode == MOC_GATE_NONE || a->gate || a->rows == 0),
              MOC_ERR_ARG, "%s: gate mode %d", who, a->gate_mode);
  MOC_REQUIRE(a->gate_mode == MOC_GATE_NONE || (a->gate_mode == MOC_GATE_CHANNEL ? a->gate_dtype == MOC_F32
              : a->gate_mode == MOC_GATE_FULL ? a->gate_dtype == a->x_dtype : dtype_size(a->gate_dtype) != 0),
              MOC_ERR_UNSUPPORTED, "%s: gate dtype %d of gate mode %d", who, a->gate_dtype, a->gate_mode);
  MOC_REQUIRE(a->eps >= 0.f && a->eps2 >= 0.f, MOC_ERR_ARG, "%s: eps < 0", who);
  return MOC_OK;
}

// 16-byte (f32: 2 x 16) loads of eight elements: every row of every operand starts on 16 bytes
bool gn_vec(const moc_gated_norm& a, const moc_gated_norm_grads* g) {
  uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.h | (uintptr_t)a.n;
  if (a.gate_mode == MOC_GATE_FULL) p |= (uintptr_t)a.gate;
  if (g) {
    p |= (uintptr_t)g->dh | (uintptr_t)g->dn | (uintptr_t)g->dx | (uintptr_t)g->dres;
    if (a.gate_mode == MOC_GATE_FULL) p |= (uintptr_t)g->dgate;
  }
  return a.d % 8 == 0 && (p & 15) == 0;
}

}  // namespace
}  // namespace moc

using namespace moc;

#define GN_FULL(KERN, TX, TR, VEC, W, KCH, ...)                                \
  do {                                                                         \
    if (full) KERN(TX, TR, VEC, W, KCH, true, __VA_ARGS__);                    \
    else KERN(TX, TR, VEC, W, KCH, false, __VA_ARGS__);                        \
  } while (0)
// eight elements per load: one wave up to 1,024, four up to 8,192, sixteen up to 16,384 elements
#define GN_SHAPE(KERN, TX, TR, ...)                                            \
  do {                                                                         \
    if (vec) {                                                                 \
      if (d <= 512) GN_FULL(KERN, TX, TR, 8, 1, 1, __VA_ARGS__);               \
      else if (d <= 1024) GN_FULL(KERN, TX, TR, 8, 1, 2, __VA_ARGS__);         \
      else if (d <= 2048) GN_FULL(KERN, TX, TR, 8, 4, 1, __VA_ARGS__);         \
      else if (d <= 4096) GN_FULL(KERN, TX, TR, 8, 4, 2, __VA_ARGS__);         \
      else if (d <= 8192) GN_FULL(KERN, TX, TR, 8, 4, 4, __VA_ARGS__);         \
      else GN_FULL(KERN, TX, TR, 8, 16, 2, __VA_ARGS__);                       \
    } else {                                                                   \
      if (d <= 512) GN_FULL(KERN, TX, TR, 1, 1, 8, __VA_ARGS__);               \
      else if (d <= 2048) GN_FULL(KERN, TX, TR, 1, 4, 8, __VA_ARGS__);         \
      else if (d <= 4096) GN_FULL(KERN, TX, TR, 1, 16, 4, __VA_ARGS__);        \
      else GN_FULL(KERN, TX, TR, 1, 16, 16, __VA_ARGS__);                      \
    }                                                                          \
  } while (0)
#define GN_TYPES(KERN, ...)                                                                                \
  do {                                                                                                     \
    if (a->x_dtype == MOC_F32 && a->r_dtype == MOC_F32) GN_SHAPE(KERN, float, float, __VA_ARGS__);         \
    else if (a->x_dtype == MOC_F32) GN_SHAPE(KERN, float, bf16, __VA_ARGS__);                              \
    else if (a->r_dtype == MOC_F32) GN_SHAPE(KERN, bf16, float, __VA_ARGS__);                              \
    else GN_SHAPE(KERN, bf16, bf16, __VA_ARGS__);                                                          \
  } while (0)

extern "C" {

int moc_gated_norm_fwd(const moc_gated_norm* a, hipStream_t stream) {
  if (int rc = gn_check("moc_gated_norm_fwd", a)) return rc;
  if (a->rows == 0) return MOC_OK;
  MOC_REQUIRE(a->h && (!a->pre || a->n), MOC_ERR_ARG, "moc_gated_norm_fwd: null output");
  const bool vec = gn_vec(*a, nullptr), full = a->gate_mode == MOC_GATE_FULL;
  const int64_t d = a->d;
  const int rpb = gn_waves(d, vec) == 1 ? 4 : 1;
  const dim3 grid((unsigned)((a->rows + rpb - 1) / rpb));
#define GN_FWD(TX, TR, VEC, W, KCH, FULL, ...)                                                                 \
  hipLaunchKernelGGL((gated_norm_fwd_kernel<TX, TR, VEC, W, KCH, FULL>), grid, dim3(W == 1 ? 256 : 64 * W), 0, \
                     stream, *a)
  GN_TYPES(GN_FWD, 0);
#undef GN_FWD
  return check_launch("gated_norm_fwd_kernel");
}

size_t moc_gated_norm_bwd_workspace(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0) return 0;
  return (size_t)(std::max(gn_strips(rows, d, true), gn_strips(rows, d, false)) * (5 * d + 1)) * sizeof(float);
}

int moc_gated_norm_bwd(const moc_gated_norm* a, const moc_gated_norm_grads* g, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  if (int rc = gn_check("moc_gated_norm_bwd", a)) return rc;
  MOC_REQUIRE(g && g->dparams && (a->rows == 0 || a->stats || (!a->post && !g->dn)), MOC_ERR_ARG, "moc_gated_norm_bwd: null pointer");
  MOC_REQUIRE(!g->dn || a->pre, MOC_ERR_ARG, "moc_gated_norm_bwd: a gradient of n without the second norm");
  MOC_REQUIRE(a->rows == 0 || (workspace && workspace_bytes >= moc_gated_norm_bwd_workspace(a->rows, a->d)), MOC_ERR_ARG,
              "moc_gated_norm_bwd: workspace too small");
  const int64_t d = a->d;
  const bool vec = gn_vec(*a, g), full = a->gate_mode == MOC_GATE_FULL;
  const int64_t strips = a->rows == 0 ? 0 : gn_strips(a->rows, d, vec);
  float* part = (float*)workspace;
  float* scal = part + strips * 5 * d;
  if (strips > 0) {
    const dim3 grid((unsigned)strips);
#define GN_BWD(TX, TR, VEC, W, KCH, FULL, ...)                                                                 \
  hipLaunchKernelGGL((gated_norm_bwd_kernel<TX, TR, VEC, W, KCH, FULL>), grid, dim3(W == 1 ? 256 : 64 * W),    \
                     W == 1 ? (size_t)std::max<int64_t>(d, 4) * sizeof(float) : 0, stream, *a, *g, part, scal)
    GN_TYPES(GN_BWD, 0);
#undef GN_BWD
    if (int rc = check_launch("gated_norm_bwd_kernel")) return rc;
  }
  hipLaunchKernelGGL(gated_norm_cols_kernel, dim3((unsigned)((5 * d + 63) / 64)), dim3(512), 0, stream, part, (int)strips,
                     5 * d, g->dparams, scal, a->gate_mode == MOC_GATE_SCALAR ? g->dparams + 5 * d : nullptr);
  return check_launch("gated_norm_cols_kernel");
}

}  // extern "C"
