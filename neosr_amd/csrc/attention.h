// attention.h — tiles, fragments and arguments shared by attention_fwd.hip and attention_bwd.hip (internal).
//
// Every product of the three kernels is v_mfma_f32_32x32x16_bf16 on operands held as NP bf16 pieces: bf16 tensors are one
// piece, fp32 tensors three (bf16x3.h: a product from the six leading cross terms is as good as an fp32 one, at 6 x 32 cycles
// per 16 reduction indices against 8 x 64 of the fp32 MFMA).  bf16 P and dS are rounded once, to nearest, when they become
// operands of the second product (the backward's short calls keep a second piece: attention_bwd.hip): half a bf16 step of each, which
// over independent keys adds up to as much as the output's own rounding, 2.3e-3 of its norm together instead of 1.7e-3.  A second
// piece of P in the forward as well would cost a third (4 x 4096 of 8 / 2 heads x 64: 195 -> 260 us) and make NaN of an infinite
// v times a remainder of 0.  Running maxima, sums, accumulators and the row statistics stay fp32.
//
// The score tile is formed transposed wherever the softmax row is the COLUMN of the accumulator: a lane then owns one row
// (query) and 16 of every 32 keys, the row statistics are per-lane scalars with one cross-half exchange, and the accumulator
// registers are, in order, the B operand of the next product — with the reduction index permuted to
//   slot (half h, e) of chunk c  <->  index 16 c + 4 h + (e & 3) + 8 (e >> 2)
// so the A operand reads the same indices: two ds_read_b64_tr_b16 (4 rows x 16 columns, transposed on the way) from the
// row-major tile.  One row-major copy in LDS serves both products; nothing is transposed by hand and no P goes through LDS.
#pragma once
#include "bf16x3.h"
#include "../../include/neosr_amd.h"

#include "lds_swizzle.h"

namespace attn {

struct Tensor4 {          // (B, L, heads, D), unit channel stride
  const char* p;
  int64_t sb, sl, sh;     // element strides
};

struct Args {
  Tensor4 q, k, v, o, dout;
  char *out, *rest, *dq, *dk, *dv;   // dense (B, L, heads, D); rest: bf16, out before its rounding less out (or null)
  float* lse;                    // (B, Hk, R) base-2 log of the row sums (scaled scores); +inf for an empty row
  float* delta;                  // (B, Hk, R)
  float* part;                   // split partials
  float* part_lse;
  char *kv_img, *row_img;        // packed tiles of (K, V) and of (Q, dO): [batch, key head][tile]
  unsigned long long* words;         // one truth bit for each key of a tile, [batch][tile]
  int kv_tiles, row_tiles;
  const unsigned char* mask;     // (B, Lk) truth values or null
  int64_t mask_sb, mask_sl;
  int B, Lq, Lk, H, Hk, G, D, R; // R = Lq * G rows of a (batch, key head): r = position * G + group
  int causal, off;               // off = Lk - Lq
  float scale, cs;               // cs = scale * log2 e
  int nblk, nsplit;              // blocks of the outer index, splits of the inner one
  int vec;                       // widest access every row allows: 2 = 16 bytes, 1 = two elements, 0 = one
};

template <typename E> struct Pieces;
template <> struct Pieces<float> { static constexpr int n = 3; };
template <> struct Pieces<__bf16> { static constexpr int n = 1; };

// 8 consecutive channels of one row as they come from memory
template <typename E> struct Raw8;
template <> struct Raw8<float> { f32x4 a, b; };
template <> struct Raw8<__bf16> { u32x4 a; };

__device__ __forceinline__ void zero(Raw8<float>& r) { r.a = r.b = (f32x4){0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ void zero(Raw8<__bf16>& r) { r.a = (u32x4){0u, 0u, 0u, 0u}; }

// channels d .. d + 7 of a row of D (zeros behind D).  `vec` is uniform over the launch.
__device__ __forceinline__ Raw8<float> load8(const float* row, int d, int D, int vec) {
  Raw8<float> r;
  zero(r);
  if (vec == 2) {            // D % 4 == 0
    if (d < D) r.a = *reinterpret_cast<const f32x4*>(row + d);
    if (d + 4 < D) r.b = *reinterpret_cast<const f32x4*>(row + d + 4);
  } else if (vec == 1) {     // D % 2 == 0
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (d + 2 * i < D) {
        const float2 t = *reinterpret_cast<const float2*>(row + d + 2 * i);
        if (i < 2) { r.a[2 * i] = t.x; r.a[2 * i + 1] = t.y; }
        else { r.b[2 * i - 4] = t.x; r.b[2 * i - 3] = t.y; }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d + i < D) { if (i < 4) r.a[i] = row[d + i]; else r.b[i - 4] = row[d + i]; }
  }
  return r;
}
__device__ __forceinline__ Raw8<__bf16> load8(const __bf16* row, int d, int D, int vec) {
  Raw8<__bf16> r;
  zero(r);
  if (vec == 2) {            // D % 8 == 0
    if (d < D) r.a = *reinterpret_cast<const u32x4*>(row + d);
  } else if (vec == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + 2 * i < D) r.a[i] = *reinterpret_cast<const unsigned*>(row + d + 2 * i);
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned lo = 0, hi = 0;
      if (d + 2 * i < D) lo = s[d + 2 * i];
      if (d + 2 * i + 1 < D) hi = s[d + 2 * i + 1];
      r.a[i] = lo | hi << 16;
    }
  }
  return r;
}

__device__ __forceinline__ void pieces(const Raw8<float>& r, bf16x8 (&P)[3]) {
  const float x[8] = {r.a[0], r.a[1], r.a[2], r.a[3], r.b[0], r.b[1], r.b[2], r.b[3]};
  split3r(x, P);
}
// Operands may be any fp32 number.  From 0x1.FFp127 on the nearest bf16 is an infinity, whose remainder is none: finite numbers
// there take the largest bf16 as their first piece.  An infinity is (+-1, 0, +-infinity): of the six terms only those of the third
// piece with the other factor's first are infinite, so its products are infinities of the right sign (and NaN with a zero).
constexpr float BEYOND = 0x1.FFp127f;
__device__ __forceinline__ float largest(const Raw8<float>& r, float top) {
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(fmaxf(top, fabsf(r.a[i])), fabsf(r.b[i]));
  return top;
}
__device__ __forceinline__ void pieces_beyond(const Raw8<float>& r, bf16x8 (&P)[3]) {
  pieces(r, P);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = i < 4 ? r.a[i & 3] : r.b[i & 3];
    const bool inf = fabsf(x) == INFINITY, big = fabsf(x) >= BEYOND;
    const float p0 = copysignf(inf ? 1.f : 0x1.FEp127f, x), p1 = inf ? 0.f : (float)(__bf16)(x - p0), p2 = inf ? x : x - p0 - p1;
    P[0][i] = big ? __builtin_bit_cast(short, (__bf16)p0) : P[0][i];
    P[1][i] = big ? __builtin_bit_cast(short, (__bf16)p1) : P[1][i];
    P[2][i] = big ? __builtin_bit_cast(short, (__bf16)p2) : P[2][i];
  }
}
__device__ __forceinline__ void pieces(const Raw8<__bf16>& r, bf16x8 (&P)[1]) { P[0] = __builtin_bit_cast(bf16x8, r.a); }
__device__ __forceinline__ float largest(const Raw8<__bf16>&, float) { return 0.f; }
__device__ __forceinline__ void pieces_beyond(const Raw8<__bf16>& r, bf16x8 (&P)[1]) { pieces(r, P); }
// pieces of operands as they come from memory; the rare numbers are seen to afterwards, by a branch of the whole wave, so that each
// load is split as it arrives
template <typename E, int NP, int N>
__device__ __forceinline__ void operands(const Raw8<E> (&r)[N], bf16x8 (&P)[N][NP]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    pieces(r[i], P[i]);
    top = largest(r[i], top);
  }
  if (__any(top >= BEYOND)) {
#pragma unroll
    for (int i = 0; i < N; ++i) pieces_beyond(r[i], P[i]);
  }
}

// 8 fp32 accumulator values -> operand pieces
__device__ __forceinline__ void pieces_of(const float (&x)[8], bf16x8 (&P)[3]) { split3r(x, P); }
__device__ __forceinline__ void pieces_of(const float (&x)[8], bf16x8 (&P)[1]) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  b8 t;
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = (__bf16)x[i];
  P[0] = __builtin_bit_cast(bf16x8, t);
}

__device__ __forceinline__ f32x16 mac(const bf16x8 (&A)[3], const bf16x8 (&B)[3], f32x16 c) { return mac6(A, B, c); }
__device__ __forceinline__ f32x16 mac(const bf16x8 (&A)[1], const bf16x8 (&B)[1], f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[0], c, 0, 0, 0);
}

// lo + c += A B, the leading terms alone in c: an MFMA rounds its accumulator, and over 16384 keys the six roundings of every 16
// are 2.2e-6 of the output, one of them 0.9e-6.
__device__ __forceinline__ void mac_lo(const bf16x8 (&A)[3], const bf16x8 (&B)[3], f32x16& lo, f32x16& c) {
  constexpr int ia[5] = {2, 0, 1, 1, 0}, ib[5] = {0, 2, 1, 0, 1};
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[0], c, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < 5; ++k) lo = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[ia[k]], B[ib[k]], lo, 0, 0, 0);
}
// two products with one B operand, their dependent MFMAs interleaved (one chain issues every 64 cycles, two every 40)
__device__ __forceinline__ void mac2(const bf16x8 (&A0)[3], const bf16x8 (&A1)[3], const bf16x8 (&B)[3], f32x16& c0, f32x16& c1) {
  constexpr int ia[6] = {2, 0, 1, 1, 0, 0}, ib[6] = {0, 2, 1, 0, 1, 0};    // smallest terms first
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    c0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A0[ia[k]], B[ib[k]], c0, 0, 0, 0);
    c1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A1[ia[k]], B[ib[k]], c1, 0, 0, 0);
  }
}

__device__ __forceinline__ float dot8(const Raw8<float>& x, const Raw8<float>& y) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(x.a[i], y.a[i], s);
#pragma unroll
  for (int i = 0; i < 4; ++i) s = fmaf(x.b[i], y.b[i], s);
  return s;
}
__device__ __forceinline__ float dot8(const Raw8<__bf16>& x, const Raw8<__bf16>& y) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(__uint_as_float(x.a[i] << 16), __uint_as_float(y.a[i] << 16), s);
    s = fmaf(__uint_as_float(x.a[i] & 0xffff0000u), __uint_as_float(y.a[i] & 0xffff0000u), s);
  }
  return s;
}

// A row-major tile of ROWS x DP channels, NP planes, without padding — one run of bytes, in LDS and in the packed image that an
// LDS-DMA copies.  A row's 16-byte units are permuted by u ^ unit_swizzle(row).
template <int NP, int DP, int ROWS>
struct Tile {
  static constexpr int PLANE = ROWS * DP;
  static constexpr int ELEMS = NP * PLANE;
  static constexpr int UPR = DP / 8;

  __device__ __forceinline__ static int at(int row, int unit) { return row * DP + ((unit ^ unit_swizzle<UPR>(row)) << 3); }

  __device__ __forceinline__ static void put(short* t, int row, int unit, const bf16x8 (&P)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(t + p * PLANE + at(row, unit)) = P[p];
  }
  // A operand, reduction over channels 16 c .. 16 c + 15: lane = row (lane & 31) of the 32-row block `r0`
  __device__ __forceinline__ static void rows(const short* t, int r0, int c, int lane, bf16x8 (&P)[NP]) {
    const short* s = t + r0 * DP + at(lane & 31, 2 * c + (lane >> 5));     // (the swizzle has period 16)
#pragma unroll
    for (int p = 0; p < NP; ++p) P[p] = *reinterpret_cast<const bf16x8*>(s + p * PLANE);
  }
  // A operand, reduction over rows r0 .. r0 + 15 (permuted as above): lane = channel d0 + (lane & 31)
  __device__ __forceinline__ static void cols(const short* t, int r0, int d0, int lane, bf16x8 (&P)[NP]) {
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), unit = d0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const short* lo_p = t + r0 * DP + at(row, unit) + 4 * (lane & 1);      // (r0 is a multiple of 16)
    const short* hi_p = t + r0 * DP + at(row + 8, unit) + 4 * (lane & 1);
    typedef const __attribute__((address_space(3))) short* lds_t;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_t)(lo_p + p * PLANE));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_t)(hi_p + p * PLANE));
      P[p] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Rows of a staged tile and its size in bytes: two tensors (K and V, or Q and dO) side by side.  64 rows; 32 where three pieces
// of wide heads would leave room for one workgroup's buffers only.
template <int NP, int DP> constexpr int tile_rows() { return NP == 3 && DP >= 64 ? 32 : 64; }
template <int NP, int DP> constexpr int tile_bytes() { return 2 * NP * tile_rows<NP, DP>() * DP * 2; }

// One LDS-DMA instruction: 64 lanes x 16 bytes -> 1 KB at LDS byte address `at` (wave-uniform).  As inline assembly because
// hipcc waits for every LDS-DMA it knows of in front of any ds_read of the same array, i.e. for the next tile before this one
// is computed.  It has no register output; the waits are dma_wait()'s.
__device__ __forceinline__ void dma16(const char* src, unsigned at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ unsigned lds_address(const short* p) {
  return (unsigned)(unsigned long long)(const __attribute__((address_space(3))) short*)p;
}

// the BYTES of a packed tile -> LDS, by all waves of the workgroup together; `src` and `at` include lane * 16 and wave * 1024
template <int BYTES, int NW>
__device__ __forceinline__ void dma_tile(const char* src, unsigned at) {
  static_assert(BYTES % (1024 * NW) == 0, "whole waves");
#pragma unroll
  for (int i = 0; i < BYTES / (1024 * NW); ++i) dma16(src + i * 1024 * NW, at + i * 1024 * NW);
}

// (r[0] holds the lower half's values in both halves, r[1] the upper half's: one VALU instruction instead of a trip through LDS)
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int acc_row(int i) { return 8 * (i >> 2) + (i & 3); }   // + 4 * half

// truth value of key `j` of sample b (out of range: false)
__device__ __forceinline__ bool key_ok(const Args& a, int b, int j) {
  if (j >= a.Lk) return false;
  return !a.mask || a.mask[(int64_t)b * a.mask_sb + (int64_t)j * a.mask_sl] != 0;
}

// The part of the inner range [beg, end) that split `s` of `n` takes, beg and all parts in multiples of 64 (whole tiles).  Of what
// the workgroup has to do, not of the whole length: in causal order every split has an equal share of the triangle.
struct Range { int beg, end; };
__device__ __forceinline__ Range share(int beg, int end, int s, int n) {
  const int len = ((max(0, end - beg) + n - 1) / n + 63) / 64 * 64;
  const int b = min(end, beg + s * len);
  return {b, min(end, b + len)};
}

// consecutive work on one XCD: workgroups are dealt round-robin to the 8 XCDs, so give each of them one contiguous run —
// the row blocks of a head then share that XCD's L2 copy of K and V
__device__ __forceinline__ int64_t xcd_order(int64_t bid, int64_t n) {
  const int64_t per = n / 8;
  return bid < per * 8 ? (bid % 8) * per + bid / 8 : bid;
}

// four consecutive channels d .. d + 3 of a dense row, element type E
template <typename E>
__device__ __forceinline__ void store4(E* row, int d, int D, const float (&x)[4]) {
  if (D % 4 == 0) {
    if (d < D) {
      if constexpr (sizeof(E) == 4) {
        *reinterpret_cast<f32x4*>(row + d) = (f32x4){x[0], x[1], x[2], x[3]};
      } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<b4*>(row + d) = (b4){(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) row[d + i] = (E)x[i];
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
// out (and rest) of four channels
template <typename E>
__device__ __forceinline__ void store_out(const Args& a, int64_t at, int d, const float (&x)[4]) {
  store4(reinterpret_cast<E*>(a.out) + at, d, a.D, x);
  if constexpr (sizeof(E) == 2) {
    if (a.rest) {
      float r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = x[i] - (float)(E)x[i];
      store4(reinterpret_cast<E*>(a.rest) + at, d, a.D, r);
    }
  }
}

constexpr int64_t MAX_GRID = 0xffffffffll / 256;   // workgroups of 256: a launch holds less than 2^32 threads

// How a pass is laid out over the chip: `packed` tiles and four waves of 32 outer indices, or single waves of 32.
struct Plan { bool packed; int nblk, nsplit; };

inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
inline int tile_rows_of(int dtype, int D) { return dtype == NEOSR_DT_F32 && D > 32 ? 32 : 64; }
inline int padded(int D) { return D <= 32 ? 32 : (D <= 64 ? 64 : 128); }
// bytes of one (batch, key head)'s packed image of L rows, two tensors
inline int64_t image_bytes(int dtype, int D, int64_t L) {
  const int kt = tile_rows_of(dtype, D);
  return (L + kt - 1) / kt * 2 * (dtype == NEOSR_DT_F32 ? 3 : 1) * kt * padded(D) * 2;
}

int check(const neosr_attention_desc* d, bool backward, const char* who);
void fill(const neosr_attention_desc* d, Args& a);
Plan plan(int64_t bh, int64_t outer, int64_t inner, int D);
int64_t words_bytes(const neosr_attention_desc* d);
// K, V tiles and the truth words; Q, dO tiles and delta (one launch)
int pack(const neosr_attention_desc* d, const Args& a, bool kv, bool rows, hipStream_t st);
}  // namespace attn
