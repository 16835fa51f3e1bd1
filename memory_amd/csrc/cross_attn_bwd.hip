// Attention over keys and values of another length, backward (notation of cross_attn.h).
//   P_ij = 2^(scale log2(e) q_i . k_j - m_i) / l_i,  delta_i = dO_i . o_i,  dS_ij = P_ij (dO_i . v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i P_ij dO_i
// delta takes the result before its rounding (out + out_low): where few keys share a row's weight, dO . v_j and delta
// nearly cancel, and out's 2^-9 alone made dq and dk twice as inexact as everything else.
// i over the rows (all queries of the G heads) of j's kv head.  dq runs over the keys of a block of rows and leaves
// -delta behind; dk and dv run over the rows of a block of keys, so nothing is summed by atomics and every result has
// one order.  P and dS enter their products rounded to the operands' type; sums, P itself and delta are f32.
//
// Measured (dq; dk and dv): 68 and 94 us for 8 x 1,024 rows of 12 heads of 64 over 1,500 ragged keys (650, 630 TFLOP/s),
// 596 and 881 us for 4 x 2,048 of 32 heads of 128 over 4,097 masked ones (990 and 890 of the live keys, of 1,247 in a
// large product).  One over l as a number of its own (see ca_stat) costs dk and dv a product per probability: 867 -> 881 us
// and 88 -> 94; dq, whose rows take it at the end, 1 %.
#include "cross_attn.h"

namespace moc {

// dq (bound as the forward is): one workgroup = 128 rows of one (sequence, kv head) as in the forward, K and V tiles
// double-buffered; K^T for dS K is read from the K tile with the transposing LDS read.  A tile's 64 keys go in two halves,
// which halves the score registers.  With SPLIT each of nsplit workgroups takes a share of the keys and writes f32 rows.
template <typename T, int D, bool SPLIT, bool FEW>
__global__ __launch_bounds__(kCaThreads) void cross_dq_kernel(CaArgs a) {
  typedef typename Frag<T>::type F8;
  using Stage = CaStage<T, D, kCaKeys, 4>;
  constexpr int KS = D / 32, DB = D / 16, TB = kCaKeys * D * (int)sizeof(T);
  constexpr bool TWO = FEW && sizeof(T) == 2;
  // dP - delta: from -delta as the product's start, which saves a subtraction, or, where exact, from the whole dP
  constexpr bool kSub = TWO || sizeof(T) == 4;
  __shared__ __attribute__((aligned(16))) char sK[2][TB];
  __shared__ __attribute__((aligned(16))) char sV[2][TB];
  __shared__ __attribute__((aligned(16))) float sB[2][kCaKeys];
  const int nrb = a.Lp / kCaRows;
  const int nsp = SPLIT ? a.nsplit : 1;
  const int64_t t0 = xcd_tile((int64_t)a.B * a.HK * nsp * nrb);
  if (t0 < 0) return;
  int b, hk;
  ca_pair(a, t0 / ((int64_t)nsp * nrb), b, hk);
  const int sp = SPLIT ? (int)((t0 / nrb) % nsp) : 0;
  const int r0 = (int)(t0 % nrb) * kCaRows;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c16 = lane & 15;

  const CaKeys keys{a.words ? a.words + (size_t)b * a.nt : nullptr, ca_keys_end(a, b)};
  const int nt = (keys.n + kCaKeys - 1) / kCaKeys;
  const int t_begin = SPLIT ? (int)((int64_t)nt * sp / nsp) : 0;
  const int t_end = SPLIT ? (int)((int64_t)nt * (sp + 1) / nsp) : nt;

  F8 qf[2][KS], dof[2][KS];
  float ref[2], dl[2];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int r = r0 + 32 * wave + 16 * qb + c16;
    const bool ok = r < a.rows;
    const int64_t l = r / a.G, h = hk * a.G + r % a.G;
    const T* qp = (const T*)a.q + b * a.qb + l * a.ql + h * a.qh;
    const T* dp = (const T*)a.dout + b * a.db + l * a.dl + h * a.dh;
    const size_t oat = (((size_t)b * a.L + l) * a.H + h) * D;
    // delta is formed as dP is, by the matrix cores and in their order: the diagonal of dO o^T.  With kSub a row that one
    // key takes whole (o = v) then has dP = delta to the bit, and no gradient; where dP's sum starts from -delta it is left
    // with that sum's roundings, some 2^-24 |dO| |v|.
    f32x4 dd = f32x4{0.f, 0.f, 0.f, 0.f}, dlow = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[qb][ks] = ok ? Load8<T, T>::run(qp + 32 * ks + 8 * g) : zero_frag<T>();
      dof[qb][ks] = ok ? Load8<T, T>::run(dp + 32 * ks + 8 * g) : zero_frag<T>();
      const F8 of = ok ? Load8<T, T>::run((const T*)a.out + oat + 32 * ks + 8 * g) : zero_frag<T>();
      mma(dd, of, dof[qb][ks]);
      if (a.out_low) {
        const F8 ol = ok ? Load8<T, T>::run((const T*)a.out_low + oat + 32 * ks + 8 * g) : zero_frag<T>();
        mma(dlow, ol, dof[qb][ks]);
      }
    }
    // the lane of group c16 / 4 holds row c16 of column c16
    dd += dlow;
    const float mine = (c16 & 2) ? ((c16 & 1) ? dd[3] : dd[2]) : ((c16 & 1) ? dd[1] : dd[0]);
    const float del = __shfl(mine, 16 * (c16 >> 2) + c16, 64);
    const size_t at = ((size_t)b * a.HK + hk) * a.Lp + r;
    dl[qb] = del;
    ref[qb] = ok ? a.stats[ca_stat((size_t)b * a.HK + hk, a.Lp, r)] : INFINITY;
    if (g == 0 && sp == 0) a.ndelta[at] = -dl[qb];
  }
  if (!a.dq) return;     // (the queries are not trained: -delta is all that dk needs)
  f32x4 acc[2][DB];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb)
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[qb][db] = f32x4{0.f, 0.f, 0.f, 0.f};

  const T* kbase = (const T*)a.k + b * a.kb + hk * a.kh;
  const T* vbase = (const T*)a.v + b * a.vb + hk * a.vh;
  auto fetch = [&](int t, uint64_t word, int buf) {
    const int left = keys.n - kCaKeys * t, rows = left < kCaKeys ? left : kCaKeys;
    const Buf kb = ca_buf(kbase + (int64_t)kCaKeys * t * a.kn, (uint32_t)(((rows - 1) * a.kn + D) * sizeof(T)));
    const Buf vb = ca_buf(vbase + (int64_t)kCaKeys * t * a.vn, (uint32_t)(((rows - 1) * a.vn + D) * sizeof(T)));
    if (wave == 0) ca_bias_put(sB[buf], word, lane);
    const uint32_t live = (uint32_t)(word >> (16 * wave));
#pragma unroll
    for (int i = 0; i < Stage::IPW; ++i) {
      const int row = Stage::row(i, lane);
      const uint32_t ch = Stage::chunk(i, lane), r = 16 * wave + row;
      uint32_t ko = r * (uint32_t)(a.kn * sizeof(T)) + ch, vo = r * (uint32_t)(a.vn * sizeof(T)) + ch;
      if (word != ~0ull && !((live >> row) & 1)) ko = vo = kCaOut;
      ca_dma16(kb.r, ko, sK[buf] + (TB / 4) * wave + 1024 * i);
      ca_dma16(vb.r, vo, sV[buf] + (TB / 4) * wave + 1024 * i);
    }
  };
  const f32x4 dinit[2] = {f32x4{-dl[0], -dl[0], -dl[0], -dl[0]}, f32x4{-dl[1], -dl[1], -dl[1], -dl[1]}};
  const float c = a.scale_log2;
  int t = t_begin;
  uint64_t word = 0;
  while (t < t_end && !(word = keys.word(t))) ++t;
  if (t < t_end) fetch(t, word, 0);
  vm_wait_all();
  __syncthreads();
  const CaFrag<T, D> fr(lane);
  const f32x4 zeros = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](auto which) {
    constexpr int buf = decltype(which)::value;
    int tn = t + 1;
    uint64_t wn = 0;
    while (tn < t_end && !(wn = keys.word(tn))) ++tn;
    if (tn < t_end) fetch(tn, wn, buf ^ 1);
    auto attend = [&] {
      const char* Ks = sK[buf];
      const char* Vs = sV[buf];
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        f32x4 st[2][2], dp[2][2];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            const F8 ak = fr.row(Ks, 32 * kh + 16 * kb, ks);
            const F8 av = fr.row(Vs, 32 * kh + 16 * kb, ks);
            const f32x4 from = *reinterpret_cast<const f32x4*>(&sB[buf][32 * kh + 16 * kb + 4 * g]);
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
              st[kb][qb] = ca_mma(ak, qf[qb][ks], ks == 0 ? from : st[kb][qb]);
              dp[kb][qb] = ca_mma(av, dof[qb][ks], ks != 0 ? dp[kb][qb] : kSub ? zeros : dinit[qb]);
            }
          }
        F8 dsf[2], dsl[2];
#pragma unroll
        for (int qb = 0; qb < 2; ++qb)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float ds = ca_exp2(ca_logit<kSub>(st[kb][qb][e], c, ref[qb])) * (kSub ? dp[kb][qb][e] - dl[qb] : dp[kb][qb][e]);
              dsf[qb][4 * kb + e] = from_f<T>(ds);
              if constexpr (TWO) dsl[qb][4 * kb + e] = ca_low<T>(ds, dsf[qb][4 * kb + e]);
            }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const F8 f = fr.col(Ks, 32 * kh, db);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            mma(acc[qb][db], dsf[qb], f);
            if constexpr (TWO) mma(acc[qb][db], dsl[qb], f);
          }
        }
      }
    };
    if constexpr (FEW) {      // (a wave without rows leaves its SIMD to the others)
      if (r0 + 32 * wave < a.rows) attend();
    } else {
      attend();
    }
    if (tn < t_end) ca_wait_all();
    t = tn;
    word = wn;
    __syncthreads();
  };
  while (t < t_end) {
    step(std::integral_constant<int, 0>());
    if (t < t_end) step(std::integral_constant<int, 1>());
  }
#pragma unroll
  for (int qb = 0; qb < 2; ++qb)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = r0 + 32 * wave + 16 * qb + 4 * g + e;
      const float inv = a.stats[ca_stat((size_t)b * a.HK + hk, a.Lp, r) + a.Lp];    // (of one over l, for the whole row)
      if constexpr (SPLIT) {
        float* dst = a.part + ((((size_t)sp * a.B + b) * a.HK + hk) * a.Lp + r) * D;
#pragma unroll
        for (int db = 0; db < DB; ++db) dst[16 * db + c16] = inv * acc[qb][db][e];
      } else if (r < a.rows) {
        T* dst = (T*)a.dq + (((size_t)b * a.L + r / a.G) * a.H + hk * a.G + r % a.G) * D;
#pragma unroll
        for (int db = 0; db < DB; ++db) dst[16 * db + c16] = from_f<T>(a.scale * inv * acc[qb][db][e]);
      }
    }
}

// dq = scale * the sum of its splits, in their order: four elements per thread
template <typename T, int D>
__device__ __forceinline__ void dq_sum(const CaArgs& a, int64_t i) {
  const int64_t row = i / (D / 4), nrow = (int64_t)a.B * a.HK * a.Lp;
  const int d0 = (int)(i % (D / 4)) * 4;
  if (row >= nrow) return;
  const int r = (int)(row % a.Lp);
  if (r >= a.rows) return;
  const int64_t bh = row / a.Lp;
  const int b = (int)(bh / a.HK), hk = (int)(bh % a.HK);
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) acc += *reinterpret_cast<const f32x4*>(a.part + (s * nrow + row) * D + d0);
  ca_store4<T>((T*)a.dq + (((size_t)b * a.L + r / a.G) * a.H + hk * a.G + r % a.G) * D + d0, nullptr, acc * a.scale);
}

// dk, dv: one workgroup = 4 waves x 16 KB keys of one (sequence, kv head), whose K and V rows stay in registers as
// matrix operands; the rows' Q and dO tiles of QS rows are double-buffered in LDS and shared by the waves, and read
// from there both as they are and transposed.
// Bound at 128 dims by LDS: 44 KB are read per wave and 32 rows, 1,375 cycles of the CU per workgroup beside 1,024
// cycles of products and 480 of vector instructions on each SIMD; at 64 dims by the latter two.  A wave's 32 keys set
// what is read (with 16, 1,196 us; with 64 the sums alone fill the registers).  VL: V stays in LDS, each wave reading
// its own rows, where with it the registers of two waves per SIMD do not hold (one wave per SIMD: 1,280 us; spilled:
// 1,330; now 881).
template <typename T, int D> struct DkvShape;
template <> struct DkvShape<bf16, 64> { static constexpr int KB = 2, QS = 128, VL = 0, WAVES = 2; };
template <> struct DkvShape<bf16, 128> { static constexpr int KB = 2, QS = 32, VL = 1, WAVES = 2; };
template <> struct DkvShape<float, 64> { static constexpr int KB = 2, QS = 32, VL = 0, WAVES = 1; };
template <> struct DkvShape<float, 128> { static constexpr int KB = 1, QS = 32, VL = 0, WAVES = 1; };

template <typename T, int D, bool SPLIT, bool FEW>
__global__ __launch_bounds__(kCaThreads, (DkvShape<T, D>::WAVES)) void cross_dkv_kernel(CaArgs a) {
  typedef typename Frag<T>::type F8;
  constexpr int KB = DkvShape<T, D>::KB, QS = DkvShape<T, D>::QS, KEYS = 64 * KB;
  using Stage = CaStage<T, D, QS, 4>;
  constexpr int KS = D / 32, DB = D / 16, TB = QS * D * (int)sizeof(T);
  constexpr bool TWO = FEW && sizeof(T) == 2;
  constexpr bool kSub = TWO || sizeof(T) == 4;   // as in dq
  constexpr bool kVL = DkvShape<T, D>::VL;
  using StageV = CaStage<T, D, KEYS, 4>;
  constexpr int VB = kVL ? KEYS * D * (int)sizeof(T) : 16;
  __shared__ __attribute__((aligned(16))) char sQ[2][TB], sD[2][TB], sV[VB];
  __shared__ __attribute__((aligned(16))) float sM[2][QS], sI[2][QS], sDl[2][QS];
  // what a lane's DMAs of a step need: offsets of its rows in Q and dO, and the rows' heads (out of registers meanwhile)
  __shared__ uint32_t sAt[3 * Stage::IPW][kCaThreads];
  const int nkb = (a.N + KEYS - 1) / KEYS;
  const int nsp = SPLIT ? a.nsplit : 1;
  const int64_t t0 = xcd_tile((int64_t)a.B * a.HK * nsp * nkb);
  if (t0 < 0) return;
  int b, hk;
  ca_pair(a, t0 / ((int64_t)nsp * nkb), b, hk);
  const int64_t bh = (int64_t)b * a.HK + hk;
  const int sp = SPLIT ? (int)((t0 / nkb) % nsp) : 0;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c16 = lane & 15;
  const int k0 = (int)(t0 % nkb) * KEYS, kw = k0 + 16 * KB * wave;   // the workgroup's and the wave's first key

  const CaKeys keys{a.words ? a.words + (size_t)b * a.nt : nullptr, ca_keys_end(a, b)};
  uint64_t any = keys.word(k0 / kCaKeys);
  if (KB == 2 && k0 + kCaKeys < a.N) any |= keys.word(k0 / kCaKeys + 1);
  // bits of this wave's keys
  const uint32_t live = kw < a.N ? (uint32_t)(keys.word(kw / kCaKeys) >> (kw % kCaKeys)) : 0u;

  F8 kf[KB][KS], vf[kVL ? 1 : KB][KS];
  {
    // bounded by the tensor's last row; what lies in keys that do not count stays in their own sums
    const int left = a.N - kw;
    const int rows = left < 0 ? 0 : left < 16 * KB ? left : 16 * KB;
    const int64_t at = rows ? kw : 0;
    const Buf kb = ca_buf((const T*)a.k + b * a.kb + hk * a.kh + at * a.kn,
                          rows ? (uint32_t)(((rows - 1) * a.kn + D) * sizeof(T)) : 0u);
    const Buf vb = ca_buf((const T*)a.v + b * a.vb + hk * a.vh + at * a.vn,
                          rows ? (uint32_t)(((rows - 1) * a.vn + D) * sizeof(T)) : 0u);
#pragma unroll
    for (int kb2 = 0; kb2 < KB; ++kb2)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t e = (32 * ks + 8 * g) * (uint32_t)sizeof(T), r = 16 * kb2 + c16;
        const uint32_t ko = r * (uint32_t)(a.kn * sizeof(T)) + e, vo = r * (uint32_t)(a.vn * sizeof(T)) + e;
        if constexpr (sizeof(T) == 2) {
          kf[kb2][ks] = __builtin_bit_cast(F8, kb.load16(ko, 0));
          if constexpr (!kVL) vf[kb2][ks] = __builtin_bit_cast(F8, vb.load16(vo, 0));
        } else {
          const V16 w2[2] = {kb.load16(ko, 0), kb.load16(ko + 16, 0)}, x2[2] = {vb.load16(vo, 0), vb.load16(vo + 16, 0)};
          kf[kb2][ks] = __builtin_bit_cast(F8, w2);
          vf[kb2][ks] = __builtin_bit_cast(F8, x2);
        }
      }
    if constexpr (kVL) {
#pragma unroll
      for (int i = 0; i < StageV::IPW; ++i)
        ca_dma16(vb.r, (uint32_t)StageV::row(i, lane) * (uint32_t)(a.vn * sizeof(T)) + StageV::chunk(i, lane),
                 sV + (VB / 4) * wave + 1024 * i);
    }
  }
  f32x4 dk[KB][DB], dv[KB][DB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      dk[kb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
      dv[kb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

  const int nstep = (a.rows + QS - 1) / QS;
  const int s_begin = SPLIT ? (int)((int64_t)nstep * sp / nsp) : 0;
  const int s_end = any == 0 ? s_begin : SPLIT ? (int)((int64_t)nstep * (sp + 1) / nsp) : nstep;
  const float* stats = a.stats + ca_stat(bh, a.Lp, 0);
  const float* ndelta = a.ndelta + bh * a.Lp;
  // Rows of step s: row QS s + r is query l0 + (q0 + r) / G, head (q0 + r) % G of the group, with r = lr G + hr a
  // constant of the lane; so its offset from query l0 is that of (lr, hr), q0 heads on, and a query on where q0 + hr
  // passes G.  (The buffers' bases are 64-bit, a step spans at most QS queries.)
#pragma unroll
  for (int i = 0; i < Stage::IPW; ++i) {
    const int r = Stage::RPW * wave + Stage::row(i, lane), lr = r / a.G, hr = r - lr * a.G;
    sAt[3 * i][tid] = (uint32_t)(lr * (uint32_t)a.ql + hr * (uint32_t)a.qh) * (uint32_t)sizeof(T) + Stage::chunk(i, lane);
    sAt[3 * i + 1][tid] = (uint32_t)(lr * (uint32_t)a.dl + hr * (uint32_t)a.dh) * (uint32_t)sizeof(T) + Stage::chunk(i, lane);
    sAt[3 * i + 2][tid] = (uint32_t)hr;
  }
  const uint32_t q_on = (uint32_t)((a.ql - a.G * a.qh) * (int64_t)sizeof(T)), d_on = (uint32_t)((a.dl - a.G * a.dh) * (int64_t)sizeof(T));
  const int l_step = QS / a.G, q_step = QS - l_step * a.G;
  int l0 = (int)((int64_t)QS * s_begin / a.G), q0 = QS * s_begin - l0 * a.G;   // of the step to be fetched next
  auto fetch = [&](int s, int buf) {
    const int r0 = QS * s, rows = a.rows - r0 < QS ? a.rows - r0 : QS;
    const int span = (q0 + rows - 1) / a.G;          // queries after the first
    const Buf qb = ca_buf((const T*)a.q + b * a.qb + (int64_t)hk * a.G * a.qh + l0 * a.ql,
                          (uint32_t)((span * a.ql + (a.G - 1) * a.qh + D) * sizeof(T)));
    const Buf db = ca_buf((const T*)a.dout + b * a.db + (int64_t)hk * a.G * a.dh + l0 * a.dl,
                          (uint32_t)((span * a.dl + (a.G - 1) * a.dh + D) * sizeof(T)));
    const uint32_t qs = q0 * (uint32_t)(a.qh * sizeof(T)), ds = q0 * (uint32_t)(a.dh * sizeof(T));
#pragma unroll
    for (int i = 0; i < Stage::IPW; ++i) {
      const int r = Stage::RPW * wave + Stage::row(i, lane);
      const bool on = q0 + (int)sAt[3 * i + 2][tid] >= a.G;
      uint32_t qo = sAt[3 * i][tid] + qs + (on ? q_on : 0u), od = sAt[3 * i + 1][tid] + ds + (on ? d_on : 0u);
      if (r >= rows) qo = od = kCaOut;
      ca_dma16(qb.r, qo, sQ[buf] + (TB / 4) * wave + 1024 * i);
      ca_dma16(db.r, od, sD[buf] + (TB / 4) * wave + 1024 * i);
    }
    l0 += l_step;
    q0 += q_step;
    if (q0 >= a.G) {
      q0 -= a.G;
      ++l0;
    }
    // reference, factor and -delta of the rows, padded to Lp, a multiple of QS, with +inf, 0 and 0
    if (64 * wave < QS) {
      const bool in = 64 * wave + lane < QS;
      const uint32_t o = in ? 4u * (64 * wave + lane) : kCaOut;
      const Buf mb = ca_buf(stats + r0, 4 * QS), ib = ca_buf(stats + a.Lp + r0, 4 * QS), eb = ca_buf(ndelta + r0, 4 * QS);
      if (in) {
        ca_dma4(mb.r, o, &sM[buf][64 * wave]);
        ca_dma4(ib.r, o, &sI[buf][64 * wave]);
        ca_dma4(eb.r, o, &sDl[buf][64 * wave]);
      }
    }
  };
  const float c = a.scale_log2;
  const CaFrag<T, D> fr(lane);
  const f32x4 zeros = f32x4{0.f, 0.f, 0.f, 0.f};
  const char* Vw = sV + 16 * KB * wave * D * (int)sizeof(T);
  if (s_begin < s_end) fetch(s_begin, 0);
  ca_wait_all();
  __syncthreads();
  // A step goes in halves of 32 rows, a half's logits in two blocks of 16: the products over the rows take 32, the
  // scores of 16 are all that is held at a time.
  auto step = [&](const int s, auto which, auto works) {
    constexpr int buf = decltype(which)::value;
    if (s + 1 < s_end) fetch(s + 1, buf ^ 1);
    const char* Qs = sQ[buf];
    const char* Ds = sD[buf];
    if constexpr (decltype(works)::value) {
#pragma unroll
      for (int half = 0; half < QS / 32; ++half) {
        const int r0 = 32 * half;
        if constexpr (FEW)
          if (QS * s + r0 >= a.rows) break;      // (no rows there)
        F8 pa[KB], sa[KB], pb[KB], sb[KB];
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const f32x4 ms = *reinterpret_cast<const f32x4*>(&sM[buf][r0 + 16 * qb + 4 * g]);
          const f32x4 nd = *reinterpret_cast<const f32x4*>(&sDl[buf][r0 + 16 * qb + 4 * g]);
          f32x4 st[KB], dp[KB];
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const F8 qa = fr.row(Qs, r0 + 16 * qb, ks), da = fr.row(Ds, r0 + 16 * qb, ks);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              st[kb] = ca_mma(qa, kf[kb][ks], ks == 0 ? zeros : st[kb]);
              const f32x4 d0 = ks != 0 ? dp[kb] : kSub ? zeros : nd;
              if constexpr (kVL)
                dp[kb] = ca_mma(da, fr.row(Vw, 16 * kb, ks), d0);
              else
                dp[kb] = ca_mma(da, vf[kb][ks], d0);
            }
          }
          // (read this late the factors take no registers from the products, which FEW does not have to spare: 49 spilled
          // at 128 dims; the others have, and wait less if the compiler reads them early: 881 us, late 985)
          if constexpr (FEW) asm volatile("" ::: "memory");
          const f32x4 is = *reinterpret_cast<const f32x4*>(&sI[buf][r0 + 16 * qb + 4 * g]);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float pt = ca_exp2(ca_logit<kSub>(st[kb][e], c, ms[e])) * is[e];
              const float ds = pt * (kSub ? dp[kb][e] + nd[e] : dp[kb][e]);
              pa[kb][4 * qb + e] = from_f<T>(pt);
              sa[kb][4 * qb + e] = from_f<T>(ds);
              if constexpr (TWO) {
                pb[kb][4 * qb + e] = ca_low<T>(pt, pa[kb][4 * qb + e]);
                sb[kb][4 * qb + e] = ca_low<T>(ds, sa[kb][4 * qb + e]);
              }
            }
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const F8 fq = fr.col(Qs, r0, db), fd = fr.col(Ds, r0, db);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            mma(dv[kb][db], pa[kb], fd);
            mma(dk[kb][db], sa[kb], fq);
            if constexpr (TWO) {
              mma(dv[kb][db], pb[kb], fd);
              mma(dk[kb][db], sb[kb], fq);
            }
          }
        }
      }
    }
    ca_wait_all();   // the next step's rows landed
    __syncthreads();
  };
  auto walk = [&](auto works) {
    for (int s = s_begin; s < s_end; s += 2) {
      step(s, std::integral_constant<int, 0>(), works);
      if (s + 1 < s_end) step(s + 1, std::integral_constant<int, 1>(), works);
    }
  };
  // (a wave none of whose keys counts fetches with the others and leaves its SIMD to them)
  if (live)
    walk(std::true_type());
  else
    walk(std::false_type());
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = kw + 16 * kb + 4 * g + e;
      if (key >= a.N) continue;
      const bool on = (live >> (16 * kb + 4 * g + e)) & 1;
      const size_t row = ((size_t)b * a.N + key) * a.HK + hk;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const float x = on ? a.scale * dk[kb][db][e] : 0.f, y = on ? dv[kb][db][e] : 0.f;
        if constexpr (SPLIT) {
          float* dst = a.part + ((size_t)sp * a.B * a.N * a.HK + row) * (2 * D) + 16 * db + c16;
          dst[0] = x;
          dst[D] = y;
        } else {
          ((T*)a.dk)[row * D + 16 * db + c16] = from_f<T>(x);
          ((T*)a.dv)[row * D + 16 * db + c16] = from_f<T>(y);
        }
      }
    }
}

// dk, dv = the sums of their splits, in their order
template <typename T, int D>
__device__ __forceinline__ void dkv_sum(const CaArgs& a, int64_t i) {
  const int64_t nrow = (int64_t)a.B * a.N * a.HK, row = i / (D / 2);
  const int d0 = (int)(i % (D / 2)) * 4;                  // of the 2 D columns dk | dv
  if (row >= nrow) return;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) acc += *reinterpret_cast<const f32x4*>(a.part + (s * nrow + row) * (2 * D) + d0);
  ca_store4<T>(d0 < D ? (T*)a.dk + row * D + d0 : (T*)a.dv + row * D + d0 - D, nullptr, acc);
}

// The sums of the splits, where there are any: the first `dq_blocks` workgroups dq's, the others dk's and dv's
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_bwd_sum_kernel(CaArgs dq, CaArgs dkv, int64_t dq_blocks) {
  if (blockIdx.x < dq_blocks)
    dq_sum<T, D>(dq, (int64_t)blockIdx.x * 256 + threadIdx.x);
  else
    dkv_sum<T, D>(dkv, ((int64_t)blockIdx.x - dq_blocks) * 256 + threadIdx.x);
}

constexpr int64_t kCaBwdWgs = 512;   // workgroups to aim at (two per CU)

struct BwdPlan {
  int dq_splits, dkv_splits;
  size_t delta, dq_part, dkv_part;   // floats
  size_t bytes() const { return 4 * (delta + dq_part + dkv_part); }
};

// Splits where there are few workgroups: of the keys for dq, of the rows for dk and dv.
BwdPlan bwd_plan(int64_t B, int64_t L, int64_t N, int H, int HK, int D, int dtype) {
  BwdPlan p = {};
  const int64_t rows = L * (H / HK), Lp = (rows + kCaRows - 1) / kCaRows * kCaRows;
  auto splits = [](int64_t wgs, int64_t steps) {
    if (wgs >= kCaBwdWgs / 2) return 1;
    int64_t s = kCaBwdWgs / (wgs < 1 ? 1 : wgs);
    if (s > steps / 2) s = steps / 2;
    return s < 1 ? 1 : s > 128 ? 128 : (int)s;
  };
  int KEYS = 0, QS = 0;
  auto shape = [&](auto s) {
    KEYS = 64 * decltype(s)::KB;
    QS = decltype(s)::QS;
  };
  if (dtype == MOC_BF16)
    D == 64 ? shape(DkvShape<bf16, 64>()) : shape(DkvShape<bf16, 128>());
  else
    D == 64 ? shape(DkvShape<float, 64>()) : shape(DkvShape<float, 128>());
  p.dq_splits = splits(B * HK * (Lp / kCaRows), (N + kCaKeys - 1) / kCaKeys);
  p.dkv_splits = splits(B * HK * ((N + KEYS - 1) / KEYS), (rows + QS - 1) / QS);
  p.delta = (size_t)B * HK * Lp;
  p.dq_part = p.dq_splits > 1 ? (size_t)p.dq_splits * B * HK * Lp * D : 0;
  p.dkv_part = p.dkv_splits > 1 ? (size_t)p.dkv_splits * B * N * HK * 2 * D : 0;
  return p;
}

template <typename T, int D>
static int bwd_launch(CaArgs& a, const BwdPlan& p, hipStream_t stream) {
  const char* who = "moc_cross_bwd";
  constexpr int KEYS = 64 * DkvShape<T, D>::KB;
  const bool few = ca_few(a);
  CaArgs q = a, kv = a;
  q.nsplit = a.dq ? p.dq_splits : 1;
  kv.nsplit = p.dkv_splits;
  kv.part = a.part + p.dq_part;
  const int64_t tiles = (int64_t)a.B * a.HK * q.nsplit * (a.Lp / kCaRows);
  const int64_t blocks = (int64_t)a.B * a.HK * kv.nsplit * ((a.N + KEYS - 1) / KEYS);
  MOC_REQUIRE(tiles < (int64_t)1 << 31 && blocks < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "%s: too many row or key blocks", who);
  // (dq comes first: it leaves -delta behind)
  if (q.nsplit > 1)
    few ? cross_dq_kernel<T, D, true, true><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(q)
        : cross_dq_kernel<T, D, true, false><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(q);
  else
    few ? cross_dq_kernel<T, D, false, true><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(q)
        : cross_dq_kernel<T, D, false, false><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(q);
  int rc = check_launch("moc_cross_bwd: dq");
  if (rc != MOC_OK) return rc;
  if (a.dk) {
    if (kv.nsplit > 1)
      few ? cross_dkv_kernel<T, D, true, true><<<xcd_grid(blocks), kCaThreads, 0, stream>>>(kv)
          : cross_dkv_kernel<T, D, true, false><<<xcd_grid(blocks), kCaThreads, 0, stream>>>(kv);
    else
      few ? cross_dkv_kernel<T, D, false, true><<<xcd_grid(blocks), kCaThreads, 0, stream>>>(kv)
          : cross_dkv_kernel<T, D, false, false><<<xcd_grid(blocks), kCaThreads, 0, stream>>>(kv);
    rc = check_launch("moc_cross_bwd: dk, dv");
    if (rc != MOC_OK) return rc;
  }
  const int64_t nq = q.nsplit > 1 ? ((int64_t)a.B * a.HK * a.Lp * (D / 4) + 255) / 256 : 0;
  const int64_t nk = a.dk && kv.nsplit > 1 ? ((int64_t)a.B * a.N * a.HK * (D / 2) + 255) / 256 : 0;
  if (nq + nk == 0) return MOC_OK;
  MOC_REQUIRE(nq + nk < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "%s: too many rows to sum", who);
  cross_bwd_sum_kernel<T, D><<<(unsigned)(nq + nk), 256, 0, stream>>>(q, kv, nq);
  return check_launch("moc_cross_bwd: sums");
}

}  // namespace moc

using namespace moc;

extern "C" {

size_t moc_cross_bwd_workspace(int64_t B, int64_t L, int64_t N, int H, int HK, int D, int dtype) {
  return HK <= 0 ? 0 : bwd_plan(B, L, N, H, HK, D, dtype).bytes();
}

int moc_cross_bwd(const moc_cross_args* args, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const char* who = "moc_cross_bwd";
  CaArgs a;
  int rc = ca_check(who, args, &a);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(a.q && a.k && a.v && a.out && a.dout && a.stats && (a.dq || a.dk), MOC_ERR_ARG, "%s: null tensor", who);
  MOC_REQUIRE(!a.dk == !a.dv, MOC_ERR_ARG, "%s: dk and dv together or neither", who);
  // the rows of a step of dk, dv are read through one bounded buffer with 32-bit offsets
  const int64_t es = dtype_size(args->dtype);
  const int64_t far = 128 * (a.ql > a.dl ? a.ql : a.dl) + (int64_t)a.G * (a.qh > a.dh ? a.qh : a.dh) + args->D;
  MOC_REQUIRE(far * es < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "%s: rows of Q and dO lie too far apart", who);
  const BwdPlan p = bwd_plan(args->B, args->L, args->N, args->H, args->HK, args->D, args->dtype);
  MOC_REQUIRE(workspace && workspace_bytes >= p.bytes(), MOC_ERR_ARG, "%s: workspace of %zu bytes, needs %zu", who,
              workspace_bytes, p.bytes());
  a.ndelta = (float*)workspace;
  a.part = a.ndelta + p.delta;
  if (args->dtype == MOC_BF16)
    return args->D == 64 ? bwd_launch<bf16, 64>(a, p, stream) : bwd_launch<bf16, 128>(a, p, stream);
  return args->D == 64 ? bwd_launch<float, 64>(a, p, stream) : bwd_launch<float, 128>(a, p, stream);
}

}  // extern "C"
