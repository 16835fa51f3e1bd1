// Kernels of gated_norm.hip, instantiated per pair of row types (gated_norm_<x><residual>.hip).
#pragma once

#include "moc_common.h"

namespace moc {

// launches of one pair of row types; `vec`: eight elements per load
int gn_fwd_ff(const moc_gated_norm& a, bool vec, hipStream_t stream);
int gn_fwd_fb(const moc_gated_norm& a, bool vec, hipStream_t stream);
int gn_fwd_bf(const moc_gated_norm& a, bool vec, hipStream_t stream);
int gn_fwd_bb(const moc_gated_norm& a, bool vec, hipStream_t stream);
struct GnStrips {
  int64_t n;      // workgroups
  float *part, *scal;
};
int gn_bwd_ff(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream);
int gn_bwd_fb(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream);
int gn_bwd_bf(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream);
int gn_bwd_bb(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t stream);

// column sums kept by a strip, in the order of moc_gated_norm_grads::dparams
enum { kGnDw1, kGnDb1, kGnDw2, kGnDb2, kGnDg, kGnSums };

constexpr int kGnWaves = 4;   // of a workgroup with several rows
// waves of a row and rows in parallel of the backward's workgroups: one load of eight (or four scalar ones) per lane
// and operand up to 8,192 (4,096) elements
inline int gn_bwd_waves(int64_t d, bool vec) {
  const int64_t per = vec ? 512 : 256;
  return d <= per ? 1 : d <= 2 * per ? 2 : d <= 4 * per ? 4 : d <= 8 * per ? 8 : 16;
}
inline int gn_bwd_rows(int waves) { return waves < kGnWaves ? kGnWaves / waves : 1; }

namespace gn {

template <typename T, int VEC> struct Vec;
template <> struct Vec<float, 8> { typedef f32x8 type; };
template <> struct Vec<bf16, 8> { typedef bf16x8 type; };
template <> struct Vec<float, 1> { typedef float type; };
template <> struct Vec<bf16, 1> { typedef bf16 type; };

template <typename T, int VEC> __device__ __forceinline__ typename Vec<T, VEC>::type load(const void* p, int64_t i) {
  return *reinterpret_cast<const typename Vec<T, VEC>::type*>((const T*)p + i);
}
template <typename T, int VEC> __device__ __forceinline__ float get(const typename Vec<T, VEC>::type& v, int e) {
  if constexpr (VEC == 1) return (float)v;
  else return (float)v[e];
}
template <typename T, int VEC> __device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    ((T*)p)[i] = from_f<T>(v[0]);
  } else {
    typename Vec<T, VEC>::type o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = from_f<T>(v[e]);
    *reinterpret_cast<typename Vec<T, VEC>::type*>((T*)p + i) = o;
  }
}
// a lane's values of a per-channel vector (`none` without one)
template <int VEC> __device__ __forceinline__ void load_w(const float* p, int j, bool live, float none, float (&v)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = none;
  if (p && live) {
    if constexpr (VEC == 8) {
      // (the vectors are only known to start on 4 bytes)
      typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
      const f32x4u a = *reinterpret_cast<const f32x4u*>(p + j), b = *reinterpret_cast<const f32x4u*>(p + j + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
      v[0] = p[j];
    }
  }
}

// Sum over the wave, the same bits in every lane: neighbours, pairs, quads and halves of a 16-lane row by DPP, then
// the rows by permutes; no LDS (against six rounds of ds_bpermute).
template <int kCtrl> __device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ float lanes_sum(float v) {
  v = dpp_add<0xB1>(v);    // quad_perm [1, 0, 3, 2]
  v = dpp_add<0x4E>(v);    // quad_perm [2, 3, 0, 1]
  v = dpp_add<0x141>(v);   // row_half_mirror
  v = dpp_add<0x140>(v);   // row_mirror
  return quad_sum_pl(v);
}

// sums of N values over the W waves of a row (waves w0 .. w0 + W - 1 of the workgroup), the same bits in every
// lane.  W > 1: every wave of the workgroup calls it.
template <int W, int N> __device__ __forceinline__ void row_sum(float (&v)[N], float* red, int wave) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i]);
  if constexpr (W > 1) {
    __syncthreads();   // the previous sums have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave * N + i] = v[i];
    }
    __syncthreads();
    const int w0 = wave / W * W;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += red[(w0 + w) * N + i];
      v[i] = s;
    }
  }
}

__device__ __forceinline__ float gate_row(const moc_gated_norm& a, int64_t r) {
  if (a.gate_mode == MOC_GATE_SCALAR) return a.gate_dtype == MOC_F32 ? *(const float*)a.gate : (float)*(const bf16*)a.gate;
  if (a.gate_mode == MOC_GATE_TOKEN) return a.gate_dtype == MOC_F32 ? ((const float*)a.gate)[r] : (float)((const bf16*)a.gate)[r];
  return 1.f;
}

// Forward: W waves per row, W == 1 four rows per workgroup.  Every load of a row is issued before its first use.
template <typename TX, typename TR, int VEC, int W, int KCH, bool FULL>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void gated_norm_fwd_kernel(moc_gated_norm a) {
  constexpr int RPB = W == 1 ? 4 : 1;   // rows of a workgroup
  __shared__ float red[W];
  const int wave = threadIdx.x >> 6;
  const int64_t r = (int64_t)blockIdx.x * RPB + (W == 1 ? wave : 0);
  if (r >= a.rows) return;   // (W > 1: uniform over the workgroup)
  const int t = W == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const int d = (int)a.d, nch = d / VEC;
  typename Vec<TX, VEC>::type xv[KCH], gv[KCH];
  typename Vec<TR, VEC>::type rv[KCH];
  float w1[KCH][VEC], b1[KCH][VEC], w2[KCH][VEC], b2[KCH][VEC], gc[KCH][VEC];
  const float grow = gate_row(a, r);
  const bool chan = !FULL && a.gate_mode == MOC_GATE_CHANNEL;
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    if (c < nch) {
      xv[i] = load<TX, VEC>(a.x, r * d + VEC * c);
      rv[i] = load<TR, VEC>(a.residual, r * d + VEC * c);
      if constexpr (FULL) gv[i] = load<TX, VEC>(a.gate, r * d + VEC * c);
    }
  }
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    load_w<VEC>(a.w1, VEC * c, c < nch, 1.f, w1[i]);
    load_w<VEC>(a.b1, VEC * c, c < nch, 0.f, b1[i]);
    if constexpr (!FULL) load_w<VEC>(chan ? (const float*)a.gate : nullptr, VEC * c, c < nch, grow, gc[i]);
    load_w<VEC>(a.w2, VEC * c, c < nch, 1.f, w2[i]);
    load_w<VEC>(a.b2, VEC * c, c < nch, 0.f, b2[i]);
  }
  const float inv_d = 1.f / (float)d;
  float h[KCH][VEC];
#pragma unroll
  for (int i = 0; i < KCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[i][e] = t + 64 * W * i < nch ? get<TX, VEC>(xv[i], e) : 0.f;
  float mu = 0.f, rs = 1.f;
  auto stats = [&](int norm, float eps) {
    mu = 0.f;
    if (norm == MOC_NORM_LAYERNORM) {
      float s[1] = {0.f};
#pragma unroll
      for (int i = 0; i < KCH; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0] += h[i][e];
      row_sum<W, 1>(s, red, wave);
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
    row_sum<W, 1>(q, red, wave);
    rs = 1.f / sqrtf(q[0] * inv_d + eps);
  };
  if (a.post) {
    stats(a.norm, a.eps);
    if (a.stats && t == 0) {
      a.stats[r] = mu;
      a.stats[a.rows + r] = rs;
    }
  }
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    if (c >= nch) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float u = (h[i][e] - mu) * rs;   // (without the first norm: 0, 1, and weights of 1 and 0)
      u = u * w1[i][e] + b1[i][e];
      float g;
      if constexpr (FULL) g = get<TX, VEC>(gv[i], e);
      else g = gc[i][e];
      h[i][e] = a.alpha * get<TR, VEC>(rv[i], e) + g * u;
    }
    store<TR, VEC>(a.h, r * d + VEC * c, h[i]);
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
    for (int e = 0; e < VEC; ++e) o[e] = (h[i][e] - mu) * rs * w2[i][e] + b2[i][e];
    store<TX, VEC>(a.n, r * d + VEC * c, o);
  }
}

// Backward of a strip of rows: RPB rows at a time, W waves each.  The channels' weights and the strip's column sums stay
// in registers (BIAS: of the biases too; GATE: the channel gate's).  part[strip][q][d], scal[strip].
// Bound: HBM, and the two sums over a row that the next row's loads have to cover (issued a row ahead; two rows ahead
// gained nothing).  8,192 x 768, f32 stream: 113 MB in 24 us, 4.7 TB/s; 6,123 x 4,096 bf16: 301 MB in 68 us, 4.4 TB/s.
enum { kGateRow, kGateChannel, kGateFull };

template <typename TX, typename TR, int VEC, int W, int RPB, int KCH, int GATE, bool BIAS>
__global__ __launch_bounds__(64 * W * RPB) void gated_norm_bwd_kernel(moc_gated_norm a, moc_gated_norm_grads o,
                                                                      float* __restrict__ part, float* __restrict__ scal) {
  constexpr bool FULL = GATE == kGateFull, CHAN = GATE == kGateChannel;
  __shared__ float red[W * RPB * 3];
  extern __shared__ float buf[];   // [d]
  const int wave = threadIdx.x >> 6, grp = wave / W;
  const int t = (int)threadIdx.x - 64 * W * grp;
  const int d = (int)a.d, nch = d / VEC;
  const float inv_d = 1.f / (float)d;
  const bool layer = a.norm == MOC_NORM_LAYERNORM, layer2 = a.norm2 == MOC_NORM_LAYERNORM;
  const bool chan = CHAN && a.gate_mode == MOC_GATE_CHANNEL;
  const bool has_dn = o.dn != nullptr;
  float w1[KCH][VEC], b1[KCH][VEC], w2[KCH][VEC], gc[KCH][VEC];
  float dw1[KCH][VEC], db1[KCH][VEC], dw2[KCH][VEC], db2[KCH][VEC], dgc[KCH][VEC];
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    const int c = t + 64 * W * i;
    load_w<VEC>(a.w1, VEC * c, c < nch, 1.f, w1[i]);
    load_w<VEC>(BIAS ? a.b1 : nullptr, VEC * c, c < nch, 0.f, b1[i]);
    load_w<VEC>(a.w2, VEC * c, c < nch, 1.f, w2[i]);
    load_w<VEC>(chan ? (const float*)a.gate : nullptr, VEC * c, c < nch, 1.f, gc[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw1[i][e] = db1[i][e] = dw2[i][e] = db2[i][e] = dgc[i][e] = 0.f;
  }
  float dscal = 0.f;
  // a row's operands, loaded one round ahead (raw: nothing here waits for a load)
  struct Row {
    typename Vec<TX, VEC>::type xv[KCH], gv[KCH], nv[KCH];
    typename Vec<TR, VEC>::type rv[KCH], hv[KCH];
    float mu1, rs1, mu2, rs2;
    uint32_t gate;
  };
  auto fetch = [&](Row& n, int64_t r) {
    n.mu1 = n.mu2 = n.rs2 = 0.f;
    n.rs1 = 1.f;
    n.gate = 0;
    if (r >= a.rows) return;
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + 64 * W * i;
      if (c < nch) {
        const int64_t at = r * d + VEC * c;
        n.xv[i] = load<TX, VEC>(a.x, at);
        if (has_dn) {
          n.rv[i] = load<TR, VEC>(a.residual, at);
          n.nv[i] = load<TX, VEC>(o.dn, at);
        }
        if (o.dh) n.hv[i] = load<TR, VEC>(o.dh, at);
        if constexpr (FULL) n.gv[i] = load<TX, VEC>(a.gate, at);
      }
    }
    if (a.post) {
      n.mu1 = a.stats[r];
      n.rs1 = a.stats[a.rows + r];
    }
    if (has_dn) {
      n.mu2 = a.stats[2 * a.rows + r];
      n.rs2 = a.stats[3 * a.rows + r];
    }
    if (!FULL && (a.gate_mode == MOC_GATE_SCALAR || a.gate_mode == MOC_GATE_TOKEN)) {
      const int64_t at = a.gate_mode == MOC_GATE_TOKEN ? r : 0;
      if (a.gate_dtype == MOC_F32) n.gate = ((const uint32_t*)a.gate)[at];
      else n.gate = ((const uint16_t*)a.gate)[at];
    }
  };
  // (every wave takes part in every round: the sums of a row over its waves synchronise the workgroup)
  auto process = [&](const Row& cur, int64_t r) {
    const bool live = r < a.rows;
    const float mu1 = cur.mu1, rs1 = cur.rs1, mu2 = cur.mu2, rs2 = cur.rs2;
    float grow = 1.f;   // (a bf16's bits are the upper half of the float's)
    if (!FULL && (a.gate_mode == MOC_GATE_SCALAR || a.gate_mode == MOC_GATE_TOKEN))
      grow = __uint_as_float(a.gate_dtype == MOC_F32 ? cur.gate : cur.gate << 16);
    auto gate_of = [&](int i, int e) {
      if constexpr (FULL) return get<TX, VEC>(cur.gv[i], e);
      else if constexpr (CHAN) return gc[i][e] * grow;   // (one of the two is 1)
      else return grow;
    };
    float xh[KCH][VEC], hh[KCH][VEC], g2[KCH][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) xh[i][e] = hh[i][e] = g2[i][e] = 0.f;
      if (t + 64 * W * i < nch && live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) xh[i][e] = (get<TX, VEC>(cur.xv[i], e) - mu1) * rs1;
        if (has_dn) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float u = xh[i][e] * w1[i][e] + b1[i][e];
            const float h = a.alpha * get<TR, VEC>(cur.rv[i], e) + gate_of(i, e) * u;
            hh[i][e] = (h - mu2) * rs2;
            const float dn = get<TX, VEC>(cur.nv[i], e);
            dw2[i][e] += dn * hh[i][e];
            if constexpr (BIAS) db2[i][e] += dn;
            g2[i][e] = dn * w2[i][e];
            s[0] += g2[i][e];
            s[1] += g2[i][e] * hh[i][e];
          }
        }
      }
    }
    if (has_dn) row_sum<W, 2>(s, red, wave);
    const float c0 = layer2 ? s[0] * inv_d : 0.f, c1 = s[1] * inv_d;
    float p[3] = {0.f, 0.f, 0.f};
    // g2 becomes dH, hh becomes g1 = du w1
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      const int c = t + 64 * W * i;
      if (c >= nch || !live) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e) g2[i][e] = rs2 * (g2[i][e] - c0 - hh[i][e] * c1);
      if (o.dh) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) g2[i][e] += get<TR, VEC>(cur.hv[i], e);
      }
      if (o.dres) {
        float dr[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) dr[e] = a.alpha * g2[i][e];
        store<TR, VEC>(o.dres, r * d + VEC * c, dr);
      }
      float dg[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        dg[e] = g2[i][e] * (xh[i][e] * w1[i][e] + b1[i][e]);
        p[2] += dg[e];
        const float du = gate_of(i, e) * g2[i][e];
        if constexpr (CHAN) dgc[i][e] += dg[e];
        dw1[i][e] += du * xh[i][e];
        if constexpr (BIAS) db1[i][e] += du;
        hh[i][e] = du * w1[i][e];
        p[0] += hh[i][e];
        p[1] += hh[i][e] * xh[i][e];
      }
      if constexpr (FULL) {
        if (o.dgate) store<TX, VEC>(o.dgate, r * d + VEC * c, dg);
      }
    }
    row_sum<W, 3>(p, red, wave);
    if (a.gate_mode == MOC_GATE_SCALAR) dscal += p[2];
    if (a.gate_mode == MOC_GATE_TOKEN && o.dgate && t == 0 && live) {
      if (a.gate_dtype == MOC_F32) ((float*)o.dgate)[r] = p[2];
      else ((bf16*)o.dgate)[r] = (bf16)p[2];
    }
    if (o.dx) {
      const float e0 = layer && a.post ? p[0] * inv_d : 0.f, e1 = a.post ? p[1] * inv_d : 0.f;
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        const int c = t + 64 * W * i;
        if (c >= nch || !live) continue;
        float dx[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) dx[e] = rs1 * (hh[i][e] - e0 - xh[i][e] * e1);
        store<TX, VEC>(o.dx, r * d + VEC * c, dx);
      }
    }
  };
  // two rows' operands in turn: a copy from one to the other would wait for the loads
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t r0 = (int64_t)blockIdx.x * RPB;
  Row even, odd;
  fetch(even, r0 + grp);
  while (r0 < a.rows) {
    fetch(odd, r0 + step + grp);
    process(even, r0 + grp);
    r0 += step;
    if (r0 >= a.rows) break;
    fetch(even, r0 + step + grp);
    process(odd, r0 + grp);
    r0 += step;
  }
  // the strip's column sums; several row groups add theirs through LDS, in order
  const int64_t strip = blockIdx.x;
  auto put = [&](int q, float (&v)[KCH][VEC]) {
    float* dst = part + (strip * kGnSums + q) * d;
    if constexpr (RPB > 1) {
      for (int w = 0; w < RPB; ++w) {
        if (grp == w) {
#pragma unroll
          for (int i = 0; i < KCH; ++i) {
            const int c = t + 64 * W * i;
            if (c < nch) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                if (w > 0) v[i][e] += buf[VEC * c + e];
                if (w < RPB - 1) buf[VEC * c + e] = v[i][e];
              }
              if (w == RPB - 1) store<float, VEC>(dst, VEC * c, v[i]);
            }
          }
        }
        __syncthreads();
      }
    } else {
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        const int c = t + 64 * W * i;
        if (c < nch) store<float, VEC>(dst, VEC * c, v[i]);
      }
    }
  };
  if (a.w1) put(kGnDw1, dw1);
  if (BIAS && a.b1) put(kGnDb1, db1);
  if (a.w2 && has_dn) put(kGnDw2, dw2);
  if (BIAS && a.b2 && has_dn) put(kGnDb2, db2);
  if (chan) put(kGnDg, dgc);
  if (a.gate_mode == MOC_GATE_SCALAR) {
    __syncthreads();
    if (t == 0) red[grp] = dscal;
    __syncthreads();
    if (threadIdx.x == 0) {
      float v = red[0];
      for (int w = 1; w < RPB; ++w) v += red[w];
      scal[strip] = v;
    }
  }
}

// Shapes.  Forward, eight per load: one wave up to 512 elements, two up to 1,024 (8,192 x 768: 15.8 us, one wave with two
// loads per lane 18.3), four up to 4,096 (6,123 x 4,096 with two loads per lane: 38.5 us, eight waves 41.9).  Bound: HBM;
// 75 MB (bf16 rows into an f32 stream) at 4.8 TB/s, 201 MB (bf16) at 5.2, the rate of a large copy.
template <typename TX, typename TR, int VEC, int W, int KCH> int fwd_shape(const moc_gated_norm& a, hipStream_t stream) {
  const dim3 grid((unsigned)(W == 1 ? (a.rows + 3) / 4 : a.rows)), block(W == 1 ? 256 : 64 * W);
  if (a.gate_mode == MOC_GATE_FULL)
    hipLaunchKernelGGL((gated_norm_fwd_kernel<TX, TR, VEC, W, KCH, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((gated_norm_fwd_kernel<TX, TR, VEC, W, KCH, false>), grid, block, 0, stream, a);
  return check_launch("gated_norm_fwd_kernel");
}
template <typename TX, typename TR> int fwd_types(const moc_gated_norm& a, bool vec, hipStream_t s) {
  const int64_t d = a.d;
  if (vec) {
    if (d <= 512) return fwd_shape<TX, TR, 8, 1, 1>(a, s);
    if (d <= 1024) return fwd_shape<TX, TR, 8, 2, 1>(a, s);
    if (d <= 2048) return fwd_shape<TX, TR, 8, 4, 1>(a, s);
    if (d <= 4096) return fwd_shape<TX, TR, 8, 4, 2>(a, s);
    if (d <= 8192) return fwd_shape<TX, TR, 8, 16, 1>(a, s);
    return fwd_shape<TX, TR, 8, 16, 2>(a, s);
  }
  if (d <= 256) return fwd_shape<TX, TR, 1, 1, 4>(a, s);
  if (d <= 2048) return fwd_shape<TX, TR, 1, 4, 8>(a, s);
  if (d <= 4096) return fwd_shape<TX, TR, 1, 16, 4>(a, s);
  return fwd_shape<TX, TR, 1, 16, 16>(a, s);
}

template <typename TX, typename TR, int VEC, int W, int RPB, int KCH>
int bwd_shape(const moc_gated_norm& a, const moc_gated_norm_grads& g, const GnStrips& s, hipStream_t stream) {
  const dim3 grid((unsigned)s.n), block(64 * W * RPB);
  const size_t lds = RPB > 1 ? (size_t)a.d * 4 : 0;
  const bool bias = a.b1 || a.b2;
#define GN_BWD(GATE, BIAS) \
  hipLaunchKernelGGL((gated_norm_bwd_kernel<TX, TR, VEC, W, RPB, KCH, GATE, BIAS>), grid, block, lds, stream, a, g, s.part, s.scal)
  if (a.gate_mode == MOC_GATE_FULL) {
    if (bias) GN_BWD(kGateFull, true);
    else GN_BWD(kGateFull, false);
  } else if (a.gate_mode == MOC_GATE_CHANNEL || VEC == 1) {
    if (bias) GN_BWD(kGateChannel, true);
    else GN_BWD(kGateChannel, false);
  } else if constexpr (VEC > 1) {
    if (bias) GN_BWD(kGateRow, true);
    else GN_BWD(kGateRow, false);
  }
#undef GN_BWD
  return check_launch("gated_norm_bwd_kernel");
}
template <typename TX, typename TR>
int bwd_types(const moc_gated_norm& a, const moc_gated_norm_grads& g, bool vec, const GnStrips& s, hipStream_t st) {
  const int w = gn_bwd_waves(a.d, vec);
  if (vec) {
    if (w == 1) return bwd_shape<TX, TR, 8, 1, kGnWaves, 1>(a, g, s, st);
    if (w == 2) return bwd_shape<TX, TR, 8, 2, kGnWaves / 2, 1>(a, g, s, st);
    if (w == 4) return bwd_shape<TX, TR, 8, 4, kGnWaves / 4, 1>(a, g, s, st);
    if (w == 8) return bwd_shape<TX, TR, 8, 8, 1, 1>(a, g, s, st);
    if (a.d <= 8192) return bwd_shape<TX, TR, 8, 16, 1, 1>(a, g, s, st);
    return bwd_shape<TX, TR, 8, 16, 1, 2>(a, g, s, st);
  }
  if (w == 1) return bwd_shape<TX, TR, 1, 1, kGnWaves, 4>(a, g, s, st);
  if (w == 2) return bwd_shape<TX, TR, 1, 2, kGnWaves / 2, 4>(a, g, s, st);
  if (w == 4) return bwd_shape<TX, TR, 1, 4, kGnWaves / 4, 4>(a, g, s, st);
  if (w == 8) return bwd_shape<TX, TR, 1, 8, 1, 4>(a, g, s, st);
  if (a.d <= 4096) return bwd_shape<TX, TR, 1, 16, 1, 4>(a, g, s, st);
  return bwd_shape<TX, TR, 1, 16, 1, 16>(a, g, s, st);
}

}  // namespace gn
}  // namespace moc
