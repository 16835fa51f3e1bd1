// Attention over keys and values of another length, forward (see cross_attn.h).
//
// One workgroup = 128 rows of one (sequence, kv head), four waves of 32; K and V tiles of 64 keys are
// double-buffered in LDS, fetched by DMA.  Each wave computes S^T = K Q^T (a lane holds one row's logits of
// 16 keys), keeps the running maximum, and accumulates O^T = V^T P^T, whose accumulator layout is again one
// row per lane, so rescaling moves no data; the row sums come from a product with ones, so they are those of
// the rounded P.  Keys that do not count are fetched as zeros (whatever their memory holds) and their logits
// start from -inf; tiles without live keys are passed over.  Few workgroups split the keys between them.
//
// Bound by products and vector instructions: of 2 x 64 keys x 32 rows of 128 dims a wave issues 68 products (1,088
// cycles), 32 exponentials (512) and some 330 cycles of other vector instructions, one after the other; LDS is busy for
// 1,024 cycles per workgroup beside that.  A SIMD has two waves, of two workgroups (three at 64 dims), which fill each
// other's gaps only in part: counted over 4 x 2,048 rows of 32 heads of 128 over 4,097 masked keys, the matrix cores are
// busy for 43 % of all cycles and vector instructions other than products issue in 31 % (dq: 49 and 24 %, dk and dv: 41 and
// 19 %).  Measured: 56 us for 8 x 1,024 rows of 12 heads of 64 over 1,500 ragged keys (530 TFLOP/s; its workgroups are one
// round of the card, as long as the longest sequence), 458 us for those of 128 dims above (850 TFLOP/s of the live keys, of
// 1,247 in a large product), 84 + 7 us for one prompt of 509 rows, 16 heads on 4, over 16,001 keys (790).  Not kept: the
// next tile's scores formed beside this one's exponentials (507 us, with the two interleaved by hand 486: 32 registers
// more), waves without rows skipping the work (703: the loop no longer runs on scalars).
#include "cross_attn.h"

namespace moc {

// A row's reference maximum moves only when a tile's exceeds it by more than this (log2 units): most tiles skip
// the rescale, and P stays <= 2^8.
constexpr float kCaSlack = 8.f;

// FEW (see kCaFew): bf16 probabilities in two pieces, and waves without rows leave their SIMD to the others.
template <typename T, int D, bool SPLIT, bool FEW>
__global__ __launch_bounds__(kCaThreads) void cross_fwd_kernel(CaArgs a) {
  typedef typename Frag<T>::type F8;
  using Stage = CaStage<T, D, kCaKeys, 4>;
  constexpr int KS = D / 32, DB = D / 16, TB = kCaKeys * D * (int)sizeof(T);
  constexpr bool TWO = FEW && sizeof(T) == 2;
  __shared__ __attribute__((aligned(16))) char sK[2][TB];
  __shared__ __attribute__((aligned(16))) char sV[2][TB];
  __shared__ __attribute__((aligned(16))) float sB[2][kCaKeys];

  // (sequence, kv head) major, row block minor: blocks that read the same keys share an XCD's L2
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

  F8 qf[2][KS];
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const int r = r0 + 32 * wave + 16 * qb + c16;
    const T* qp = (const T*)a.q + b * a.qb + (int64_t)(r / a.G) * a.ql + (int64_t)(hk * a.G + r % a.G) * a.qh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[qb][ks] = r < a.rows ? Load8<T, T>::run(qp + 32 * ks + 8 * g) : zero_frag<T>();
  }

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

  float m[2] = {-INFINITY, -INFINITY}, lsum[2] = {0.f, 0.f};
  F8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = from_f<T>(1.f);
  f32x4 o[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) o[db][qb] = f32x4{0.f, 0.f, 0.f, 0.f};
  const float c = a.scale_log2;

  int t = t_begin;
  uint64_t word = 0;
  while (t < t_end && !(word = keys.word(t))) ++t;
  if (t < t_end) fetch(t, word, 0);
  vm_wait_all();
  __syncthreads();
  const CaFrag<T, D> fr(lane);
  const f32x4 zeros = ca_zeros();
  auto step = [&](auto which) {
    constexpr int buf = decltype(which)::value;
    int tn = t + 1;
    uint64_t wn = 0;
    while (tn < t_end && !(wn = keys.word(tn))) ++tn;
    // (buffer buf ^ 1 was last read a tile ago, which every wave has finished)
    if (tn < t_end) fetch(tn, wn, buf ^ 1);
    auto attend = [&] {
      const char* Ks = sK[buf];
      const char* Vs = sV[buf];
      f32x4 st[4][2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const F8 f = fr.row(Ks, 16 * kb, ks);
          const f32x4 from = *reinterpret_cast<const f32x4*>(&sB[buf][16 * kb + 4 * g]);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) st[kb][qb] = ca_mma(f, qf[qb][ks], ks == 0 ? from : st[kb][qb]);
        }
      float cm[2];
      bool grow = false;
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        float mx = ca_max3(st[0][qb][0], st[0][qb][1], st[0][qb][2]);
        mx = ca_max3(mx, st[0][qb][3], st[1][qb][0]);
        mx = ca_max3(mx, st[1][qb][1], st[1][qb][2]);
        mx = ca_max3(mx, st[1][qb][3], st[2][qb][0]);
        mx = ca_max3(mx, st[2][qb][1], st[2][qb][2]);
        mx = ca_max3(mx, st[2][qb][3], st[3][qb][0]);
        mx = ca_max3(mx, st[3][qb][1], st[3][qb][2]);
        cm[qb] = quad_max_pl(fmax_fast(mx, st[3][qb][3])) * c;
        grow |= cm[qb] > m[qb] + kCaSlack;
      }
      if (__any(grow)) {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
          const float mn = cm[qb] > m[qb] + kCaSlack ? cm[qb] : m[qb];
          const float alpha = m[qb] == mn ? 1.f : ca_exp2(m[qb] - mn);
          m[qb] = mn;
          lsum[qb] *= alpha;
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db][qb] *= alpha;
        }
      }
      F8 pf[2][2], pl[2][2];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
        const float off = m[qb] == -INFINITY ? 0.f : m[qb];   // (a row whose logits so far are all -inf)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float p = ca_exp2(ca_logit<TWO || sizeof(T) == 4>(st[2 * h + (x >> 2)][qb][x & 3], c, off));
            pf[qb][h][x] = from_f<T>(p);
            if constexpr (TWO) pl[qb][h][x] = ca_low<T>(p, pf[qb][h][x]);
          }
      }
      f32x4 ls[2];
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ls[qb] = ca_mma(ones, pf[qb][h], h == 0 ? zeros : ls[qb]);
          if constexpr (TWO) mma(ls[qb], ones, pl[qb][h]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const F8 f = fr.col(Vs, 32 * h, db);
#pragma unroll
          for (int qb = 0; qb < 2; ++qb) {
            mma(o[db][qb], f, pf[qb][h]);
            if constexpr (TWO) mma(o[db][qb], f, pl[qb][h]);
          }
        }
#pragma unroll
      for (int qb = 0; qb < 2; ++qb) lsum[qb] += ls[qb][0];
    };
    if constexpr (FEW) {
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

  // rows without live keys: 0, and +inf as the backward's reference (its probabilities are 0 then), as in the padding
  // rows up to Lp
#pragma unroll
  for (int qb = 0; qb < 2; ++qb) {
    const float l = lsum[qb];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int r = r0 + 32 * wave + 16 * qb + c16;
    if constexpr (SPLIT) {
      const size_t row = (((size_t)sp * a.B + b) * a.HK + hk) * a.Lp + r;
      float* pp = a.part + row * D + 4 * g;
#pragma unroll
      for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(pp + 16 * db) = o[db][qb];
      if (g == 0) {
        a.part_m[row] = m[qb];
        a.part_l[row] = l;
      }
    } else {
      if (r < a.rows) {
        const size_t at = (((size_t)b * a.L + r / a.G) * a.H + hk * a.G + r % a.G) * D + 4 * g;
        T* op = (T*)a.out + at;
        T* lp = a.out_low ? (T*)a.out_low + at : nullptr;
#pragma unroll
        for (int db = 0; db < DB; ++db) ca_store4<T>(op + 16 * db, lp ? lp + 16 * db : nullptr, o[db][qb] * inv);
      }
      if (a.stats && g == 0) {
        const bool none = r >= a.rows || l == 0.f;
        float* st = a.stats + ca_stat((size_t)b * a.HK + hk, a.Lp, r);
        st[0] = none ? INFINITY : m[qb];
        st[a.Lp] = none ? 0.f : inv;
      }
    }
  }
}

// out = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i over the splits of a row, and its stats: D / 4 lanes of four
// dims in each of 1024 / D groups.  With few rows all groups of a workgroup share one, each taking every so many
// splits, joined in LDS: a chain of two loads whatever the number of splits (32 of them one after the other took 7 us,
// this 3).  With many rows (ALONE) each group has its own, which keeps more loads in flight.
template <typename T, int D, bool ALONE>
__global__ __launch_bounds__(256) void cross_merge_kernel(CaArgs a, int64_t nrow) {
  constexpr int LPR = D / 4, GR = 256 / LPR;
  __shared__ float sM[GR], sS[GR];
  __shared__ __attribute__((aligned(16))) float sO[ALONE ? 1 : GR][D];
  const int ch = threadIdx.x % LPR, gr = threadIdx.x / LPR;
  const int64_t row = ALONE ? (int64_t)blockIdx.x * GR + gr : blockIdx.x;   // (b, hk, r)
  if (row >= nrow) return;
  const int r = (int)((uint32_t)row % (uint32_t)a.Lp);
  const uint32_t bh = (uint32_t)row / (uint32_t)a.Lp, b = bh / (uint32_t)a.HK, hk = bh - b * a.HK;
  float* st = a.stats && ch == 0 ? a.stats + ca_stat(bh, a.Lp, r) : nullptr;
  if (r >= a.rows) {
    if (st && (ALONE || gr == 0)) {
      st[0] = INFINITY;
      st[a.Lp] = 0.f;
    }
    return;
  }
  float M = -INFINITY, den = 0.f;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  auto take = [&](float d, const f32x4& o, float s) {
    // (a split without live keys has sums of 0, one of NaN logits alone NaN: both go through with the weight 1)
    const float m = fmax_fast(M, d);
    const float w = d == -INFINITY ? 1.f : ca_exp2(d - m), f = M == -INFINITY ? 1.f : ca_exp2(M - m);
    acc = acc * f + o * w;
    den = den * f + s * w;
    M = m;
  };
#pragma unroll 4
  for (int s = ALONE ? 0 : gr; s < a.nsplit; s += ALONE ? 1 : GR)
    take(a.part_m[s * nrow + row], *reinterpret_cast<const f32x4*>(a.part + (s * nrow + row) * D + 4 * ch),
         a.part_l[s * nrow + row]);
  if constexpr (!ALONE) {
    if (ch == 0) {
      sM[gr] = M;
      sS[gr] = den;
    }
    *reinterpret_cast<f32x4*>(&sO[gr][4 * ch]) = acc;
    __syncthreads();
    if (gr != 0) return;
    const int used = a.nsplit < GR ? a.nsplit : GR;
    for (int q = 1; q < used; ++q) take(sM[q], *reinterpret_cast<const f32x4*>(&sO[q][4 * ch]), sS[q]);
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  const size_t at = (((size_t)b * a.L + r / a.G) * a.H + hk * a.G + r % a.G) * D + 4 * ch;
  ca_store4<T>((T*)a.out + at, a.out_low ? (T*)a.out_low + at : nullptr, acc * inv);
  if (st) {
    st[0] = den == 0.f ? INFINITY : M;
    st[a.Lp] = inv;
  }
}

// words[b][t]: the live keys of tile t, from one byte per key and the sequence's length; a wave per word
__global__ __launch_bounds__(256) void key_words_kernel(const uint8_t* __restrict__ mask, int64_t mb, int64_t mn,
                                                        const int32_t* __restrict__ lengths, int64_t B, int N, int nt,
                                                        uint64_t* __restrict__ words) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= B * nt) return;
  const int64_t b = w / nt;
  const int key = kCaKeys * (int)(w % nt) + (threadIdx.x & 63);
  const bool live = key < N && (!lengths || key < lengths[b]) && mask[b * mb + key * mn] != 0;
  const uint64_t bits = __ballot(live);
  if ((threadIdx.x & 63) == 0) words[w] = bits;
}

// Workgroups of the forward from which on splitting the keys no longer pays (two to three per CU).
constexpr int64_t kCaWgs = 512;

// Splits of the keys: enough workgroups to fill the card, each with a few tiles (float32: one; a tile costs a workgroup
// on its own about 5 us there and 1.2 in bf16, the join 4).
int ca_fwd_splits(int64_t wgs, int64_t nt, int dtype) {
  if (wgs >= kCaWgs / 2) return 1;
  int64_t s = kCaWgs / (wgs < 1 ? 1 : wgs);
  const int64_t most = dtype == MOC_F32 ? nt : nt / 4;
  if (s > most) s = most;
  return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}

int ca_check(const char* who, const moc_cross_args* p, CaArgs* c) {
  MOC_REQUIRE(p != nullptr, MOC_ERR_ARG, "%s: no arguments", who);
  const moc_cross_args& a = *p;
  MOC_REQUIRE(a.dtype == MOC_F32 || a.dtype == MOC_BF16, MOC_ERR_ARG, "%s: dtype %d", who, a.dtype);
  MOC_REQUIRE(a.D == 64 || a.D == 128, MOC_ERR_UNSUPPORTED, "%s: head dim %d, expected 64 or 128", who, a.D);
  MOC_REQUIRE(a.H > 0 && a.HK > 0 && a.H % a.HK == 0, MOC_ERR_ARG, "%s: %d query heads on %d kv heads", who, a.H, a.HK);
  MOC_REQUIRE(a.B > 0 && a.L > 0 && a.N > 0, MOC_ERR_ARG, "%s: empty sizes", who);
  const int64_t G = a.H / a.HK, es = dtype_size(a.dtype);
  MOC_REQUIRE(a.L * G < (int64_t)1 << 30 && a.N < (int64_t)1 << 30 && a.B < (int64_t)1 << 24, MOC_ERR_UNSUPPORTED,
              "%s: sizes B=%lld L=%lld N=%lld", who, (long long)a.B, (long long)a.L, (long long)a.N);
  // (scale log2(e) is finite then: a logit of 0 stays 0)
  MOC_REQUIRE(a.scale > 0.f && a.scale < 0x1p127f, MOC_ERR_ARG, "%s: scale must be positive and less than 2^127", who);
  const int64_t st[] = {a.qb, a.ql, a.qh, a.kb, a.kn, a.kh, a.vb, a.vn, a.vh, a.db, a.dl, a.dh};
  for (int64_t s : st)
    MOC_REQUIRE(s >= 0 && s * es % 16 == 0, MOC_ERR_ARG, "%s: strides must be multiples of 16 bytes", who);
  const void* ptrs[] = {a.q, a.k, a.v, a.out, a.out_low, a.dout, a.dq, a.dk, a.dv};
  for (const void* x : ptrs)
    MOC_REQUIRE(((uintptr_t)x & 15) == 0, MOC_ERR_ARG, "%s: tensors must be 16-byte aligned", who);
  // a tile's rows are read through one bounded buffer with 32-bit offsets (the top bit marks keys left out)
  MOC_REQUIRE((a.kn * es) < ((int64_t)1 << 24) && (a.vn * es) < ((int64_t)1 << 24), MOC_ERR_UNSUPPORTED,
              "%s: rows of K and V must lie less than 16 MiB apart", who);
  MOC_REQUIRE(a.N == 1 || (a.kn >= a.D && a.vn >= a.D), MOC_ERR_ARG, "%s: rows of K or V overlap", who);
  CaArgs& o = *c;
  o = CaArgs{};
  o.q = a.q; o.k = a.k; o.v = a.v; o.out = a.out; o.out_low = a.dtype == MOC_BF16 ? a.out_low : nullptr; o.dout = a.dout;
  o.dq = a.dq; o.dk = a.dk; o.dv = a.dv; o.stats = a.lse; o.lengths = a.lengths; o.words = a.words;
  o.qb = a.qb; o.ql = a.ql; o.qh = a.qh; o.kb = a.kb; o.kn = a.kn; o.kh = a.kh; o.vb = a.vb; o.vn = a.vn; o.vh = a.vh;
  o.db = a.db; o.dl = a.dl; o.dh = a.dh;
  o.B = (int)a.B; o.L = (int)a.L; o.N = (int)a.N; o.H = a.H; o.HK = a.HK; o.G = (int)G;
  o.rows = (int)(a.L * G);
  o.Lp = (o.rows + kCaRows - 1) / kCaRows * kCaRows;
  o.nt = (o.N + kCaKeys - 1) / kCaKeys;
  o.nsplit = 1;
  o.scale = a.scale;
  o.scale_log2 = a.scale * 1.4426950408889634f;
  return MOC_OK;
}

template <typename T, int D>
static int fwd_launch(CaArgs& a, hipStream_t stream) {
  const int64_t tiles = (int64_t)a.B * a.HK * a.nsplit * (a.Lp / kCaRows);
  MOC_REQUIRE(tiles < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "moc_cross_fwd: too many row blocks");
  const bool few = ca_few(a);
  if (a.nsplit == 1) {
    few ? cross_fwd_kernel<T, D, false, true><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(a)
        : cross_fwd_kernel<T, D, false, false><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(a);
    return check_launch("moc_cross_fwd");
  }
  few ? cross_fwd_kernel<T, D, true, true><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(a)
      : cross_fwd_kernel<T, D, true, false><<<xcd_grid(tiles), kCaThreads, 0, stream>>>(a);
  int rc = check_launch("moc_cross_fwd");
  if (rc != MOC_OK) return rc;
  return ca_merge(sizeof(T) == 2 ? MOC_BF16 : MOC_F32, D, a, stream);
}

template <typename T, int D>
static void merge_launch(const CaArgs& a, int64_t rows, hipStream_t stream) {
  constexpr int GR = 1024 / D;
  if (rows >= 2048)
    cross_merge_kernel<T, D, true><<<(unsigned)((rows + GR - 1) / GR), 256, 0, stream>>>(a, rows);
  else
    cross_merge_kernel<T, D, false><<<(unsigned)rows, 256, 0, stream>>>(a, rows);
}

int ca_merge(int dtype, int D, const CaArgs& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.B * a.HK * a.Lp;
  MOC_REQUIRE(rows < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "attention merge: too many rows");
  if (dtype == MOC_BF16)
    D == 64 ? merge_launch<bf16, 64>(a, rows, stream) : merge_launch<bf16, 128>(a, rows, stream);
  else
    D == 64 ? merge_launch<float, 64>(a, rows, stream) : merge_launch<float, 128>(a, rows, stream);
  return check_launch("attention merge");
}

}  // namespace moc

using namespace moc;

extern "C" {

int64_t moc_cross_rows(int64_t L, int H, int HK) {
  if (HK <= 0 || L <= 0) return 0;
  return 2 * ((L * (H / HK) + kCaRows - 1) / kCaRows * kCaRows);
}

size_t moc_cross_fwd_workspace(int64_t B, int64_t L, int64_t N, int H, int HK, int D, int dtype) {
  const int64_t Lp = moc_cross_rows(L, H, HK) / 2;
  const int s = ca_fwd_splits(B * HK * (Lp / kCaRows), (N + kCaKeys - 1) / kCaKeys, dtype);
  return s == 1 ? 0 : (size_t)s * B * HK * Lp * (D + 2) * 4;
}

int moc_cross_fwd(const moc_cross_args* args, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  CaArgs a;
  int rc = ca_check("moc_cross_fwd", args, &a);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(a.q && a.k && a.v && a.out, MOC_ERR_ARG, "moc_cross_fwd: null tensor");
  const int64_t bhl = (int64_t)a.B * a.HK * a.Lp;
  a.nsplit = ca_fwd_splits((int64_t)a.B * a.HK * (a.Lp / kCaRows), a.nt, args->dtype);
  const size_t need = moc_cross_fwd_workspace(args->B, args->L, args->N, args->H, args->HK, args->D, args->dtype);
  MOC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), MOC_ERR_ARG, "moc_cross_fwd: workspace of %zu bytes, needs %zu",
              workspace_bytes, need);
  a.part = (float*)workspace;
  a.part_m = a.part + (size_t)a.nsplit * bhl * args->D;
  a.part_l = a.part_m + (size_t)a.nsplit * bhl;
  if (args->dtype == MOC_BF16) return args->D == 64 ? fwd_launch<bf16, 64>(a, stream) : fwd_launch<bf16, 128>(a, stream);
  return args->D == 64 ? fwd_launch<float, 64>(a, stream) : fwd_launch<float, 128>(a, stream);
}

int moc_key_words(const void* mask, int64_t mb, int64_t mn, const int32_t* lengths, int64_t B, int64_t N, uint64_t* words,
                  hipStream_t stream) {
  MOC_REQUIRE(mask && words && B > 0 && N > 0 && N < (int64_t)1 << 30, MOC_ERR_ARG, "moc_key_words: bad arguments");
  const int64_t nt = (N + kCaKeys - 1) / kCaKeys;
  MOC_REQUIRE(B * nt < (int64_t)1 << 32, MOC_ERR_UNSUPPORTED, "moc_key_words: too many keys");
  key_words_kernel<<<(unsigned)((B * nt + 3) / 4), 256, 0, stream>>>((const uint8_t*)mask, mb, mn, lengths, B, (int)N,
                                                                    (int)nt, words);
  return check_launch("moc_key_words");
}

}  // extern "C"
