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
// Bound: HBM.  A row is held by W waves (VEC elements per load, KCH loads per lane); the kernels are in gated_norm.h.
#include <algorithm>

#include "gated_norm.h"

namespace moc {
namespace {

constexpr int kGnMaxD = 16384;

// grads[q][j] = sum over the strips: eight lanes of four columns each, 128 groups of strips, added in a fixed order.
// Bound: latency; the sums of 256 to 512 strips come from the caches (768 channels 6 us, 4,096 with biases 7.5).
__global__ __launch_bounds__(1024) void gated_norm_cols_kernel(const float* __restrict__ part, int strips, int d, unsigned live,
                                                               float* __restrict__ out, const float* __restrict__ scal) {
  constexpr int kGrp = 128;
  __shared__ float buf[kGrp][33];
  const int q = blockIdx.y;
  if (q == kGnSums) {   // the scalar gate's
    if (!(live >> q & 1) || blockIdx.x > 0 || threadIdx.x >= 64) return;
    float v = 0.f;
    for (int i = threadIdx.x; i < strips; i += 64) v += scal[i];
    v = wave_sum(v);
    if (threadIdx.x == 0) out[kGnSums * (int64_t)d] = v;
    return;
  }
  if (!(live >> q & 1)) return;
  const int lane = threadIdx.x & 7, grp = threadIdx.x >> 3;
  const int j = blockIdx.x * 32 + 4 * lane;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const float* src = part + (int64_t)q * d + j;
  for (int i = grp; i < strips; i += kGrp) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += j + e < d ? src[(int64_t)i * kGnSums * d + e] : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) buf[grp][4 * lane + e] = s[e];
  __syncthreads();
  for (int n = kGrp / 2; n >= 1; n >>= 1) {
    for (int i = threadIdx.x; i < n * 32; i += 1024) buf[i >> 5][i & 31] += buf[(i >> 5) + n][i & 31];
    __syncthreads();
  }
  const int c = blockIdx.x * 32 + (int)threadIdx.x;
  if (threadIdx.x < 32 && c < d) out[(int64_t)q * d + c] = buf[0][threadIdx.x];
}

// Strips (workgroups) of the backward: two waves on every SIMD, which is what its registers allow.
int64_t gn_strips(int64_t rows, int64_t d, bool vec) {
  const int waves = gn_bwd_waves(d, vec), rpb = gn_bwd_rows(waves);
  return std::max<int64_t>(1, std::min<int64_t>((rows + rpb - 1) / rpb, 2048 / (waves * rpb)));
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

extern "C" {

int moc_gated_norm_fwd(const moc_gated_norm* a, hipStream_t stream) {
  if (int rc = gn_check("moc_gated_norm_fwd", a)) return rc;
  if (a->rows == 0) return MOC_OK;
  MOC_REQUIRE(a->h && (!a->pre || a->n), MOC_ERR_ARG, "moc_gated_norm_fwd: null output");
  const bool vec = gn_vec(*a, nullptr), xf = a->x_dtype == MOC_F32, rf = a->r_dtype == MOC_F32;
  return (xf ? rf ? gn_fwd_ff : gn_fwd_fb : rf ? gn_fwd_bf : gn_fwd_bb)(*a, vec, stream);
}

size_t moc_gated_norm_bwd_workspace(int64_t rows, int64_t d) {
  if (rows <= 0 || d <= 0) return 0;
  return (size_t)(std::max(gn_strips(rows, d, true), gn_strips(rows, d, false)) * (kGnSums * d + 1)) * sizeof(float);
}

int moc_gated_norm_bwd(const moc_gated_norm* a, const moc_gated_norm_grads* g, void* workspace, size_t workspace_bytes,
                       hipStream_t stream) {
  if (int rc = gn_check("moc_gated_norm_bwd", a)) return rc;
  MOC_REQUIRE(g && g->dparams && (a->rows == 0 || a->stats || (!a->post && !g->dn)), MOC_ERR_ARG,
              "moc_gated_norm_bwd: null pointer");
  MOC_REQUIRE(!g->dn || a->pre, MOC_ERR_ARG, "moc_gated_norm_bwd: a gradient of n without the second norm");
  MOC_REQUIRE(a->rows == 0 || (workspace && workspace_bytes >= moc_gated_norm_bwd_workspace(a->rows, a->d)), MOC_ERR_ARG,
              "moc_gated_norm_bwd: workspace too small");
  const int64_t d = a->d;
  const bool vec = gn_vec(*a, g), xf = a->x_dtype == MOC_F32, rf = a->r_dtype == MOC_F32;
  GnStrips s{a->rows == 0 ? 0 : gn_strips(a->rows, d, vec), (float*)workspace, nullptr};
  s.scal = s.part + s.n * kGnSums * d;
  if (s.n > 0)
    if (int rc = (xf ? rf ? gn_bwd_ff : gn_bwd_fb : rf ? gn_bwd_bf : gn_bwd_bb)(*a, *g, vec, s, stream)) return rc;
  unsigned live = 0;
  if (a->w1) live |= 1u << kGnDw1;
  if (a->b1) live |= 1u << kGnDb1;
  if (a->w2 && g->dn) live |= 1u << kGnDw2;
  if (a->b2 && g->dn) live |= 1u << kGnDb2;
  if (a->gate_mode == MOC_GATE_CHANNEL) live |= 1u << kGnDg;
  if (a->gate_mode == MOC_GATE_SCALAR) live |= 1u << kGnSums;
  if (!live) return MOC_OK;
  hipLaunchKernelGGL(gated_norm_cols_kernel, dim3((unsigned)((d + 31) / 32), kGnSums + 1), dim3(1024), 0, stream, s.part, (int)s.n,
                     (int)d, live, g->dparams, s.scal);
  return check_launch("gated_norm_cols_kernel");
}

}  // extern "C"
