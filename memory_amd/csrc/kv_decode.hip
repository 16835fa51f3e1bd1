// Attention of few queries per sequence over their keys and values, strided or in pages: bound by HBM, each key
// and value is read once.
//
// A unit is one (sequence, kv head, 16 RB rows) with r = l G + g as in cross_attn.h; its tiles of 64 keys are split
// over nsplit workgroups and there over four waves, each with a running maximum of its own, joined in LDS and
// (nsplit > 1) by a second launch.  K goes straight to registers as the matrix operand, V through a tile of the
// wave's own in LDS, from which it is read transposed.  A tile is four blocks of 16 keys, each within one page.
//
// Measured: 123 us for 64 sequences of up to 4,096 keys, 12 heads of 64 (608 MB: 4.9 TB/s, a copy runs at 5.2), 111 + 4
// for 37 of up to 5,001 keys, 8 kv heads of 128 in pages of 16 (575 MB: 5.0), 9 + 3 for one of 8,191 keys (34 MB), where
// the chain length -> page -> keys -> products -> join of a few loads each is what is left.
#include "cross_attn.h"

namespace moc {

constexpr int kKdWaves = 4;

struct KdArgs {
  CaArgs c;
  const int32_t* table;
  int64_t kp, vp, tb, num_pages, max_pages;
  int page, causal, nrb;
};

// RB: row blocks of 16 that a unit's keys and values are read for once (two where there are more than 16 rows).
template <typename T, int D, int RB, bool PAGED, bool SPLIT>
__global__ __launch_bounds__(64 * kKdWaves) void kv_decode_kernel(KdArgs p) {
  typedef typename Frag<T>::type F8;
  using Tile = SwzTile<T, D>;
  using Stage = CaStage<T, D, 16, 1>;            // a block of 16 keys, by one wave
  constexpr int KS = D / 32, DB = D / 16, TB = kCaKeys * D * (int)sizeof(T);
  constexpr bool kTwo = sizeof(T) == 2;
  constexpr int ROWS = 16 * RB;
  static_assert(TB >= 16 * D * 4, "a wave's V tile holds 16 of its result rows");
  __shared__ __attribute__((aligned(16))) char sV[kKdWaves][TB];
  __shared__ float sM[kKdWaves][ROWS], sL[kKdWaves][ROWS];
  const CaArgs& a = p.c;
  const int nsp = SPLIT ? a.nsplit : 1;
  const int64_t u = blockIdx.x;                  // ((b, hk), row block, split)
  const int sp = (int)(u % nsp), rb = (int)(u / nsp % p.nrb);
  const int64_t bh = u / nsp / p.nrb;
  const int b = (int)(bh / a.HK), hk = (int)(bh % a.HK);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c16 = lane & 15;

  // tokens of the sequence, and those of them that have a place (the first n): what a causal row sees is counted from
  // the former, since the tokens of the call are the sequence's last ones whether they found a place or not
  int len = a.lengths ? ca_scalar(a.lengths + b) : a.N;
  len = len < 0 ? 0 : len;
  const int n = len < a.N ? len : a.N;
  const CaKeys keys{!PAGED && a.words ? a.words + (size_t)b * a.nt : nullptr, n};
  const int nt = (n + kCaKeys - 1) / kCaKeys;
  const int t_begin = (int)((int64_t)nt * sp / nsp), t_end = (int)((int64_t)nt * (sp + 1) / nsp);

  // keys that this lane's rows see, and those that every row does
  int limit[RB];
  const int all_see = p.causal && len - (a.L - 1) < n ? len - (a.L - 1) : n;
  F8 qf[RB][KS];
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    const int r = ROWS * rb + 16 * x + c16, l = r / a.G, h = hk * a.G + r % a.G;
    const bool ok = r < a.rows;
    const int see = len - (ok ? a.L - l - 1 : 0);       // (never past len, which may be 2^31 - 1)
    limit[x] = !ok ? 0 : p.causal && see < n ? see : n;
    const T* qp = (const T*)a.q + b * a.qb + (int64_t)l * a.ql + (int64_t)h * a.qh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[x][ks] = ok ? Load8<T, T>::run(qp + 32 * ks + 8 * g) : zero_frag<T>();
  }

  const T* kbase = (const T*)a.k + (PAGED ? 0 : b * a.kb) + hk * a.kh;
  const T* vbase = (const T*)a.v + (PAGED ? 0 : b * a.vb) + hk * a.vh;
  char* Vs = sV[wave];
  F8 kf[4][KS];
  uint64_t word = 0;
  // requests a tile: K into kf, V into Vs; keys that do not count come as zeros
  auto fetch = [&](int t) {
    word = keys.word(t);
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      const int pos = kCaKeys * t + 16 * kb;
      int rows = n - pos;
      rows = rows < 0 ? 0 : rows < 16 ? rows : 16;
      int64_t ko = (int64_t)pos * a.kn, vo = (int64_t)pos * a.vn;
      if constexpr (PAGED) {
        const int pg = rows > 0 ? ca_scalar(p.table + b * p.tb + pos / p.page) : -1;
        if (pg < 0 || pg >= p.num_pages) {
          rows = 0;
          word &= ~(0xffffull << (16 * kb));
        }
        ko = (int64_t)pg * p.kp + (int64_t)(pos % p.page) * a.kn;
        vo = (int64_t)pg * p.vp + (int64_t)(pos % p.page) * a.vn;
      }
      // (without rows the base stays within the tensor and the bound is 0)
      const Buf kbuf = ca_buf(kbase + (rows ? ko : 0), rows ? (uint32_t)(((rows - 1) * a.kn + D) * sizeof(T)) : 0u);
      const Buf vbuf = ca_buf(vbase + (rows ? vo : 0), rows ? (uint32_t)(((rows - 1) * a.vn + D) * sizeof(T)) : 0u);
      const uint32_t live = (uint32_t)(word >> (16 * kb));
#pragma unroll
      for (int i = 0; i < Stage::IPW; ++i) {
        const int row = Stage::row(i, lane);
        uint32_t off = (uint32_t)row * (uint32_t)(a.vn * sizeof(T)) + Stage::chunk(i, lane);
        if (!((live >> row) & 1)) off = kCaOut;
        ca_dma16(vbuf.r, off, Vs + (TB / 4) * kb + 1024 * i);
      }
      const uint32_t ro = (live >> c16) & 1 ? (uint32_t)c16 * (uint32_t)(a.kn * sizeof(T)) : kCaOut;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t off = ro + (32 * ks + 8 * g) * (int)sizeof(T);
        if constexpr (sizeof(T) == 2) {
          kf[kb][ks] = __builtin_bit_cast(F8, kbuf.load16(off, 0));
        } else {
          const V16 w2[2] = {kbuf.load16(off, 0), kbuf.load16(off + 16, 0)};
          kf[kb][ks] = __builtin_bit_cast(F8, w2);
        }
      }
    }
  };

  float m[RB], lsum[RB];
  f32x4 o[RB][DB];
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    m[x] = -INFINITY;
    lsum[x] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[x][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float c = a.scale_log2;
  const CaFrag<T, D> fr(lane);

  for (int t = t_begin + wave; t < t_end; t += kKdWaves) {
    fetch(t);
    f32x4 st[RB][4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int x = 0; x < RB; ++x) {
        st[x][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) mma(st[x][kb], kf[kb][ks], qf[x][ks]);
      }
    if (word != ~0ull || kCaKeys * (t + 1) > all_see) {
      const uint32_t w[2] = {(uint32_t)word >> (4 * g), (uint32_t)(word >> 32) >> (4 * g)};
#pragma unroll
      for (int x = 0; x < RB; ++x) {
        const int left = limit[x] - kCaKeys * t - 4 * g;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((w[kb >> 1] >> (16 * (kb & 1) + e)) & 1) || 16 * kb + e >= left) st[x][kb][e] = -INFINITY;
      }
    }
    // the sums: a lane's 16 keys here, the four lanes of the row at the end.  In bf16 the probabilities enter their
    // product in two pieces, 16 bits of them: the second product costs nothing under the loads, and one piece alone would
    // make the result's error 1.35 times that of its rounding (1,000 keys).
    F8 pf[RB][2], pl[RB][2];
#pragma unroll
    for (int x = 0; x < RB; ++x) {
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        mx = ca_max3(mx, st[x][kb][0], st[x][kb][1]);
        mx = ca_max3(mx, st[x][kb][2], st[x][kb][3]);
      }
      const float cm = quad_max_pl(mx) * c;
      if (__any(cm > m[x])) {
        const float mn = cm > m[x] ? cm : m[x];
        const float alpha = m[x] == mn ? 1.f : ca_exp2(m[x] - mn);
        m[x] = mn;
        lsum[x] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[x][db] *= alpha;
      }
      const float off = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float pr = ca_exp2(ca_logit<true>(st[x][2 * hh + (y >> 2)][y & 3], c, off));
          lsum[x] += pr;
          pf[x][hh][y] = from_f<T>(pr);
          if constexpr (kTwo) pl[x][hh][y] = ca_low<T>(pr, pf[x][hh][y]);
        }
    }
    ca_wait_all();   // V landed
    wave_lds_sync();
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const F8 f = fr.col(Vs, 32 * hh, db);
#pragma unroll
        for (int x = 0; x < RB; ++x) {
          mma(o[x][db], f, pf[x][hh]);
          if constexpr (kTwo) mma(o[x][db], f, pl[x][hh]);
        }
      }
    wave_lds_sync();   // the next tile's V overwrites this one once it has been read
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  // the waves' results in units of their common maximum, sixteen rows at a time
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    lsum[x] = quad_sum(lsum[x]);
    if (g == 0) {
      sM[wave][16 * x + c16] = m[x];
      sL[wave][16 * x + c16] = lsum[x];
    }
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < RB; ++x) {
    float M = sM[0][16 * x + c16];
#pragma unroll
    for (int w = 1; w < kKdWaves; ++w) M = fmax_fast(M, sM[w][16 * x + c16]);
    const float f = m[x] == -INFINITY ? 1.f : ca_exp2(m[x] - M);   // (a wave without live keys: its sums are 0 or NaN)
    float* res = reinterpret_cast<float*>(Vs);                    // [16 rows][D]
    if (x > 0) __syncthreads();
#pragma unroll
    for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(res + c16 * D + 16 * db + 4 * g) = o[x][db] * f;
    __syncthreads();
#pragma unroll
    for (int i = tid; i < 16 * D / 4; i += 64 * kKdWaves) {
      const int row = i / (D / 4), d0 = i % (D / 4) * 4, rx = 16 * x + row, rr = ROWS * rb + rx;
      float Mr = sM[0][rx], den = 0.f;
#pragma unroll
      for (int w = 1; w < kKdWaves; ++w) Mr = fmax_fast(Mr, sM[w][rx]);
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kKdWaves; ++w) {
        acc += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(sV[w]) + row * D + d0);
        den += sM[w][rx] == -INFINITY ? sL[w][rx] : sL[w][rx] * ca_exp2(sM[w][rx] - Mr);
      }
      const float inv = den == 0.f ? 0.f : 1.f / den;
      if (rr >= a.rows) continue;
      if constexpr (SPLIT) {
        const size_t at = (((size_t)sp * a.B + b) * a.HK + hk) * a.Lp + rr;
        *reinterpret_cast<f32x4*>(a.part + at * D + d0) = acc;
        if (d0 == 0) {
          a.part_m[at] = Mr;
          a.part_l[at] = den;
        }
      } else {
        T* op = (T*)a.out + (((size_t)b * a.L + rr / a.G) * a.H + hk * a.G + rr % a.G) * D + d0;
        ca_store4<T>(op, nullptr, acc * inv);
      }
    }
  }
}

// Splits of the keys, each with a tile per wave at least.  A card holds 1,024 workgroups of 64 dims in bf16 (33 KB of
// LDS) and half or a quarter as many of wider tiles.  With most of that taken there is no split (64 sequences of 12
// heads of 64: 128 us, two splits 133, four 135); with less, three rounds of workgroups (37 sequences of 8 heads of 128
// in 1, 2, 5 and 10 splits of ragged lengths: -, 153, 124, 137 us).
int kd_splits(int64_t units, int64_t n_max, int row_bytes) {
  const int64_t most = ((n_max + kCaKeys - 1) / kCaKeys + kKdWaves - 1) / kKdWaves;
  const int64_t slots = 1024 * 128 / row_bytes;
  if (units < 1) units = 1;
  int64_t s = 10 * units >= 7 * slots ? 1 : (3 * slots + units / 2) / units;
  if (s > most) s = most;
  return s < 1 ? 1 : s > 128 ? 128 : (int)s;
}

// Row blocks of a unit: two where there is more than one and the registers hold them
int kd_row_blocks(int64_t rows, int D, int dtype) { return rows > 16 && !(dtype == MOC_F32 && D == 128) ? 2 : 1; }

template <typename T, int D, int RB>
static int kd_launch_rows(KdArgs& p, bool paged, hipStream_t stream) {
  const int64_t grid = (int64_t)p.c.B * p.c.HK * p.nrb * p.c.nsplit;
  MOC_REQUIRE(grid < (int64_t)1 << 31, MOC_ERR_UNSUPPORTED, "moc_kv_decode: too many rows");
  const bool split = p.c.nsplit > 1;
  const dim3 gr((unsigned)grid), bl(64 * kKdWaves);
  if (paged)
    split ? kv_decode_kernel<T, D, RB, true, true><<<gr, bl, 0, stream>>>(p)
          : kv_decode_kernel<T, D, RB, true, false><<<gr, bl, 0, stream>>>(p);
  else
    split ? kv_decode_kernel<T, D, RB, false, true><<<gr, bl, 0, stream>>>(p)
          : kv_decode_kernel<T, D, RB, false, false><<<gr, bl, 0, stream>>>(p);
  int rc = check_launch("moc_kv_decode");
  if (rc != MOC_OK || !split) return rc;
  return ca_merge(sizeof(T) == 2 ? MOC_BF16 : MOC_F32, D, p.c, stream);
}

template <typename T, int D>
static int kd_launch(KdArgs& p, bool paged, int rb, hipStream_t stream) {
  if constexpr (!(sizeof(T) == 4 && D == 128))
    if (rb == 2) return kd_launch_rows<T, D, 2>(p, paged, stream);
  return kd_launch_rows<T, D, 1>(p, paged, stream);
}

}  // namespace moc

using namespace moc;

extern "C" {

size_t moc_kv_decode_workspace(int64_t B, int64_t L, int64_t n_max, int H, int HK, int D, int dtype) {
  if (HK <= 0) return 0;
  const int64_t rows = L * (H / HK), per = 16 * kd_row_blocks(rows, D, dtype), nrb = (rows + per - 1) / per;
  const int s = kd_splits(B * HK * nrb, n_max, D * dtype_size(dtype));
  return s == 1 ? 0 : (size_t)s * B * HK * rows * (D + 2) * 4;
}

int moc_kv_decode(const moc_kv_decode_args* d, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const char* who = "moc_kv_decode";
  MOC_REQUIRE(d != nullptr, MOC_ERR_ARG, "%s: no arguments", who);
  const bool paged = d->table != nullptr;
  moc_cross_args x = {};
  x.q = d->q; x.k = d->k; x.v = d->v; x.out = d->out; x.lengths = d->lengths; x.words = d->words;
  x.qb = d->qb; x.ql = d->ql; x.qh = d->qh;
  x.kb = paged ? d->kp : d->kb; x.kn = d->kn; x.kh = d->kh;
  x.vb = paged ? d->vp : d->vb; x.vn = d->vn; x.vh = d->vh;
  x.B = d->B; x.L = d->L; x.H = d->H; x.HK = d->HK; x.D = d->D; x.dtype = d->dtype; x.scale = d->scale;
  x.N = paged ? (d->max_pages > 0 && d->page > 0 ? d->max_pages * d->page : 0) : d->N;
  KdArgs p = {};
  int rc = ca_check(who, &x, &p.c);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(d->q && d->k && d->v && d->out, MOC_ERR_ARG, "%s: null tensor", who);
  if (paged) {
    MOC_REQUIRE(d->lengths && !d->words, MOC_ERR_ARG, "%s: pages need lengths and take no key mask", who);
    MOC_REQUIRE(d->page > 0 && d->page % 16 == 0, MOC_ERR_UNSUPPORTED, "%s: pages of %d tokens, expected a multiple of 16", who,
                d->page);
    MOC_REQUIRE(d->num_pages >= 0 && d->num_pages < (int64_t)1 << 31 && d->tb >= 0, MOC_ERR_ARG, "%s: bad page table", who);
    p.table = d->table; p.kp = d->kp; p.vp = d->vp; p.tb = d->tb;
    p.num_pages = d->num_pages; p.max_pages = d->max_pages; p.page = d->page;
  }
  p.causal = d->causal ? 1 : 0;
  const int rb = kd_row_blocks(p.c.rows, x.D, x.dtype);
  p.nrb = (p.c.rows + 16 * rb - 1) / (16 * rb);
  p.c.Lp = p.c.rows;     // (of the partial results)
  p.c.stats = nullptr;
  p.c.nsplit = kd_splits((int64_t)p.c.B * p.c.HK * p.nrb, p.c.N, x.D * dtype_size(x.dtype));
  const size_t need = moc_kv_decode_workspace(x.B, x.L, x.N, x.H, x.HK, x.D, x.dtype);
  MOC_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), MOC_ERR_ARG, "%s: workspace of %zu bytes, needs %zu", who,
              workspace_bytes, need);
  p.c.part = (float*)workspace;
  p.c.part_m = p.c.part + (size_t)p.c.nsplit * p.c.B * p.c.HK * p.c.Lp * x.D;
  p.c.part_l = p.c.part_m + (size_t)p.c.nsplit * p.c.B * p.c.HK * p.c.Lp;
  if (x.dtype == MOC_BF16)
    return x.D == 64 ? kd_launch<bf16, 64>(p, paged, rb, stream) : kd_launch<bf16, 128>(p, paged, rb, stream);
  return x.D == 64 ? kd_launch<float, 64>(p, paged, rb, stream) : kd_launch<float, 128>(p, paged, rb, stream);
}

}  // extern "C"
