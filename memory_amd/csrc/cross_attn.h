// Shared parts of the attention over keys and values of another length (cross_attn_fwd.hip,
// cross_attn_bwd.hip, kv_decode.hip):
//   s_ij = scale q_i . k_j,   o_i = sum_j softmax_j(s_ij) v_j      over the live keys j of i's sequence.
//
// Rows: query l of head h = hk G + g is row r = l G + g of kv head hk, so the G heads that share a kv
// head fill one block of rows whatever L is (a block of few queries would leave the matrix cores idle,
// and heads of one query lie side by side in memory).  Keys come in tiles of 64; the live keys of a tile
// are the bits of a 64-bit word, worked out from the sequence's length or read from packed mask words.
#pragma once

#include "moc_common.h"

namespace moc {

constexpr int kCaThreads = 256;
constexpr int kCaRows = 128;     // rows of a workgroup (4 waves x 32)
constexpr int kCaKeys = 64;      // keys of a tile
constexpr uint32_t kCaOut = 0x80000000u;   // an offset behind every bounded buffer: reads as zeros

typedef __attribute__((address_space(3))) void* ca_lds_ptr_t;
// One 16-byte-per-lane LDS DMA: lane l's 16 bytes at voff of the buffer land at LDS address lds + 16 l;
// offsets past the buffer's bound write zeros.  The wait is an explicit vmcnt(0).
__device__ __forceinline__ void ca_dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, const char* lds) {
  const uint32_t m0 = (uint32_t)(uintptr_t)(ca_lds_ptr_t)lds;
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(m0) : "memory");
}
// The same with 4 bytes per lane
__device__ __forceinline__ void ca_dma4(__amdgpu_buffer_rsrc_t r, uint32_t voff, const void* lds) {
  const uint32_t m0 = (uint32_t)(uintptr_t)(ca_lds_ptr_t)lds;
  asm volatile("buffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(r), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void ca_wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ float ca_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float ca_max3(float a, float b, float c) { return fmax_fast(fmax_fast(a, b), c); }

// Four zeros that the compiler takes for unknown, so that a product that starts from them reads these registers instead
// of having its own cleared first (the row sums of the forward: 57.6 -> 55.3 us at 64 dims).
__device__ __forceinline__ f32x4 ca_zeros() {
  f32x4 z = f32x4{0.f, 0.f, 0.f, 0.f};
  asm volatile("" : "+v"(z));
  return z;
}
// a b + c as a new accumulator
__device__ __forceinline__ f32x4 ca_mma(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 ca_mma(const f32x8& a, const f32x8& b, const f32x4& c) {
  f32x4 x = c;
  mma(x, a, b);
  return x;
}

// s c - off; EXACT rounds the product by itself, so that a row's largest logit has exactly 2^0.  Fused, half a step of the
// logit is left in the exponent, the same of a key forward and backward, so that it cancels against the row's sum.
template <bool EXACT>
__device__ __forceinline__ float ca_logit(float s, float c, float off) {
  if constexpr (EXACT) {
#pragma clang fp contract(off)
    const float x = s * c;
    return x - off;
  } else {
    return __builtin_fmaf(s, c, -off);
  }
}

// Rows of D elements, ROWS of them, moved global -> LDS (SwzTile<T, D>) by WAVES waves: an instruction
// fills RPI rows of CH 16-byte chunks, wave w issues the IPW instructions from row (ROWS / WAVES) w.
template <typename T, int D, int ROWS, int WAVES>
struct CaStage {
  static constexpr int CH = D * (int)sizeof(T) / 16;
  static constexpr int RPI = 64 / CH;
  static constexpr int RPW = ROWS / WAVES;       // rows per wave
  static constexpr int IPW = RPW / RPI;
  static_assert(CH >= 8 && 64 % CH == 0 && RPW % 8 == 0 && IPW * RPI == RPW, "staging geometry");
  // row of the wave's block and byte offset in it that this lane moves with instruction i
  static __device__ __forceinline__ int row(int i, int lane) { return RPI * i + lane / CH; }
  static __device__ __forceinline__ uint32_t chunk(int i, int lane) {
    return (uint32_t)(((lane % CH) ^ (row(i, lane) & 7)) * 16);
  }
};

// The operand reads of a lane from SwzTile<T, D> tiles, with what a lane adds to their addresses worked out once (bf16:
// two registers for rows as they are, four for rows transposed; a row block, a further 64 dims and the tile itself are
// constants in the instructions).  R, rb: first row, multiples of 16 and of 32.
template <typename T, int D>
struct CaFrag {
  using Tile = SwzTile<T, D>;
  typedef typename Frag<T>::type F8;
  int lane;
  uint32_t s[2], t[4];
  __device__ __forceinline__ explicit CaFrag(int ln) : lane(ln) {
    if constexpr (sizeof(T) == 2) {
      const int g = ln >> 4, q = ln & 15, row = 4 * g + (q >> 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = (uint32_t)(q * 2 * D + (((4 * i + g) ^ (q & 7)) << 4));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t[i] = (uint32_t)(row * 2 * D + (((2 * i + ((q & 3) >> 1)) ^ (row & 7)) << 4) + 8 * (q & 1));
    }
  }
  // rows R + c16, dims 32 ks + 8 g ..
  __device__ __forceinline__ F8 row(const char* tile, int R, int ks) const {
    if constexpr (sizeof(T) == 2)
      return *reinterpret_cast<const bf16x8*>(tile + s[ks & 1] + (R * 2 * D + 128 * (ks >> 1)));
    else
      return Tile::frag(tile, R + (lane & 15), 32 * ks + 8 * (lane >> 4));
  }
  // dim 16 db + c16 of rows rb + 4 g + e and rb + 16 + 4 g + e
  __device__ __forceinline__ F8 col(const char* tile, int rb, int db) const {
    if constexpr (sizeof(T) == 2) {
      typedef short v4s __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) v4s* lds_v4s;
      const char* p = tile + t[db & 3] + (rb * 2 * D + 128 * (db >> 2));
      const v4s v[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)p),
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(p + 16 * 2 * D))};
      return __builtin_bit_cast(F8, v);
    } else {
      return mk_frag<Tile, T>(tile, rb, 16 * db, lane);
    }
  }
};

// A load from an address that is one for the whole wave, through the scalar cache: it does not queue behind the
// DMAs in flight, as a vector load's wait would.  Nothing in the launch writes there.
template <typename T>
__device__ __forceinline__ T ca_scalar(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}

// A bounded buffer at an address that is one for the whole wave but may stand in vector registers
__device__ __forceinline__ Buf ca_buf(const void* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return Buf((const void*)(uintptr_t)((uint64_t)hi << 32 | lo), __builtin_amdgcn_readfirstlane(bytes));
}

// Live keys of a sequence's tile
struct CaKeys {
  const uint64_t* words;   // of the sequence, or null
  int n;                   // keys before the sequence's end
  __device__ __forceinline__ uint64_t word(int t) const {
    if (words) return ca_scalar(words + t);
    const int left = n - kCaKeys * t;
    return left >= kCaKeys ? ~0ull : left <= 0 ? 0ull : ~0ull >> (kCaKeys - left);
  }
};

// bf16 probabilities and logit gradients enter their products rounded to 8 bits.  That takes the error of a result from
// that of its own rounding alone to 1.05 (2 keys) to 1.35 (1,000 keys) times it, of a gradient to 1.4 times at any number.
// In calls of up to this many keys, or rows of a kv head, they go in two pieces, 16 bits, at half as many products again,
// and results have their own rounding's error alone: those calls are launches and loads, so the products cost them nothing.
// (It is the call's number of keys that counts, with those that lengths and masks leave out.)  In either type the kernels of such calls pass over blocks of rows that are
// empty, which would cost the others the schedule of their loops (11 sequences of one token of 16 heads of 64 over 4 kv
// heads and 10,813 keys: forward 45 -> 37 us and backward 117 -> 91 in bf16, 152 -> 92 and 326 -> 252 in float32).
constexpr int kCaFew = 128;

// Of each row the backward takes the reference of its logits (log2 units: their maximum, or less by up to kCaSlack) and
// one over the sum of 2^(logit - reference).  In one number, reference + log2(sum), the logarithm's lower bits are lost
// under a large logit, and where one key takes a row so is what the fused product leaves of it: dv was off by 8e-5 at
// logits of 4,096 (float32), by 0.005 at 2^18 and by 0.4 at 2^24.  Partial results keep the two apart as well.
// stats: [B][HK][2][Lp], the references (+inf in rows without keys, and behind the last) and the factors (0 there).
__device__ __forceinline__ size_t ca_stat(size_t bh, int Lp, int r) { return 2 * bh * Lp + r; }

// What a launch works on (moc_cross_args with the derived sizes)
struct CaArgs {
  const void *q, *k, *v, *dout;
  void *out, *out_low, *dq, *dk, *dv;
  float *stats, *ndelta, *part, *part_m, *part_l;
  const int32_t* lengths;
  const uint64_t* words;
  int64_t qb, ql, qh, kb, kn, kh, vb, vn, vh, db, dl, dh;   // element strides
  int B, L, N, H, HK, G, rows, Lp, nt, nsplit;
  float scale, scale_log2;
};

// Pair i of a launch's (sequence, kv head) pairs, the sequences innermost: the eight XCDs each take a run of pairs,
// and with ragged sequences those of one head are as much work as those of another.
__device__ __forceinline__ void ca_pair(const CaArgs& a, int64_t i, int& b, int& hk) {
  b = (int)((uint32_t)i % (uint32_t)a.B);
  hk = (int)((uint32_t)i / (uint32_t)a.B);
}

__device__ __forceinline__ int ca_keys_end(const CaArgs& a, int b) {
  if (!a.lengths) return a.N;
  const int n = ca_scalar(a.lengths + b);
  return n < 0 ? 0 : n < a.N ? n : a.N;
}

// What a tile's logits start from: 0, or -inf for keys that do not count (whose rows of K are fetched as zeros), as the
// first operand of their product.  Written with the tile by one wave; lane (g, c16) reads keys 16 kb + 4 g + e.  (Setting
// the logits afterwards took two vector instructions for each of them.)
__device__ __forceinline__ void ca_bias_put(float* bias, uint64_t word, int lane) {
  bias[lane] = (word >> lane) & 1 ? 0.f : -INFINITY;
}

// Stores 4 consecutive results, and with `low` what their rounding left over
template <typename T> struct Vec4;
template <> struct Vec4<bf16> { typedef bf16x4 type; };
template <> struct Vec4<float> { typedef f32x4 type; };
template <typename T>
__device__ __forceinline__ void ca_store4(T* out, T* low, const f32x4& x) {
  typename Vec4<T>::type y, z;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = from_f<T>(x[e]);
    z[e] = from_f<T>(x[e] - to_f(y[e]));
  }
  *reinterpret_cast<typename Vec4<T>::type*>(out) = y;
  if (low) *reinterpret_cast<typename Vec4<T>::type*>(low) = z;
}

// The piece of x that its rounding to T leaves over
template <typename T>
__device__ __forceinline__ T ca_low(float x, T rounded) { return from_f<T>(x - to_f(rounded)); }

inline bool ca_few(const CaArgs& a) { return a.N <= kCaFew || a.rows <= kCaFew; }

int ca_check(const char* who, const moc_cross_args* a, CaArgs* c);
// out (and stats) of a.nsplit partial results over rows [B][HK][Lp]: sums a.part, references a.part_m, row sums a.part_l
int ca_merge(int dtype, int D, const CaArgs& a, hipStream_t stream);

}  // namespace moc
