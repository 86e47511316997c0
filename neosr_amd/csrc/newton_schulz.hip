// newton_schulz.hip — orthogonalised updates for a whole list of matrices (the `muon` optimizer):
//   X_0 = G / (|G|_F + eps),   X <- (a I + b A + c A A) X,  A = X X^T   (rows <= columns; A = X^T X, X <- X (...) otherwise).
//
// All matrices of a list advance together: one launch per product and step over the tiles of every matrix, so a network's
// 200 small products are 3 launches a step and not 600.  Matrices of equal shape form a class with a regular workspace
// layout; the class table travels as a kernel argument (nothing is copied to the device, captured graphs replay as they are).
//
// Products are six-term bf16x3 (bf16x3.h), fp32-faithful: rounding errors of early steps are amplified by up to a^steps = 485
// along the small singular directions, so plain bf16 products would not do for fp32 weights.  X, A and the polynomial
// Q = a I + b A + c A A are KEPT as their three bf16 planes: an element is split once, by the epilogue that writes it,
// instead of by every tile that reads it.  A, A A and Q are symmetric: only the tiles on and above the diagonal are computed
// and written twice.  Both orientations run on X as the caller stores it: the products that reduce over rows take their
// operands through ds_read_b64_tr_b16 (transposed on the way from a row-major LDS tile), nothing is transposed in memory.
//
// Measured: the 223 matrices of swinir_medium in 581 us (5 steps: 39 us for A, 25 for Q, 62 for X, whose planes are 70 MB read and
// written; matrix pipe 26 %); 2048^2, 1024 x 4096 and 2304 x 1024 in bf16 1.13 ms; one 180 x 180 matrix 114 us, 18 launches of 4 to 7
// us that each wait for one trip to memory.  Large products: 0.65 us per 32-wide step of a 128-wide tile; matrix pipe 54 % with
// 128-wide tiles, 35 % with the 208 workgroups of the symmetric products in 64-wide ones.
#include "bf16x3.h"
#include "../../include/neosr_amd.h"
#include "prof.h"
#include <math.h>

#include "lds_swizzle.h"

namespace ns {

constexpr int MAXCLS = 32, MAXITEM = 40;
constexpr int TURN = 512;                   // units of 8 elements per workgroup of the element-wise passes

struct Cls {
  int rows, cols, rp, cp, m, tall, count;   // padded to multiples of 32; m = padded smaller side
  int nb;                                   // norm partials per matrix
  int64_t base;                             // first matrix, in shorts
  int64_t per;                              // one matrix, in shorts: X | X' | A | Q planes
  int64_t part;                             // first norm partial, in doubles
};
struct Classes {
  Cls c[MAXCLS];
  int n;
};

// what the product kernels need of the classes (kernel arguments stay under 4 KB)
struct TCls {
  int64_t base, per;
  int rp, cp, m, tall;
};
struct Table {
  TCls c[MAXCLS];
  int tiles[MAXCLS + 1];                    // prefix: workgroups of the classes before
  int ncls;
};

// what the element-wise passes need of the items
struct Item {
  char* p;                                  // the caller's matrices
  int64_t sb, sr;
  int64_t base, per, part;                  // the item's first matrix
  int rows, cols, rp, cp, nb, blocks;       // blocks: prefix of workgroups
};
struct Items {
  Item it[MAXITEM];
  int n;
};
static_assert(sizeof(Table) < 3800 && sizeof(Items) < 3800, "kernel arguments");

// ---- pieces ----------------------------------------------------------------------------------------------------------------------
// fp32 matrices: three pieces, six terms.  bf16 matrices: two pieces rounded to nearest (2^-18 of the value), three terms — the
// result is rounded to 2^-9 at the end, and 2^-18 amplified over five steps stays below that (measured against 64 bits: 2e-4
// against the rounding's 1.7e-3), at half the matrix work and two thirds of the traffic.
template <typename E> struct Pieces;
template <> struct Pieces<float> { static constexpr int n = 3; };
template <> struct Pieces<__bf16> { static constexpr int n = 2; };

__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&P)[3]) { split3r(x, P); }
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&P)[2]) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  b8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi[i] = (__bf16)x[i];
    lo[i] = (__bf16)(x[i] - (float)hi[i]);
  }
  P[0] = __builtin_bit_cast(bf16x8, hi);
  P[1] = __builtin_bit_cast(bf16x8, lo);
}
__device__ __forceinline__ float piece(short p) { return __uint_as_float((unsigned)(unsigned short)p << 16); }
__device__ __forceinline__ float join(const short (&p)[3]) { return (piece(p[2]) + piece(p[1])) + piece(p[0]); }
__device__ __forceinline__ float join(const short (&p)[2]) { return piece(p[1]) + piece(p[0]); }
// acc[0] + acc[1] + acc[2] += A B, the terms of a size together: every MFMA rounds its accumulator, and the sum of the leading
// terms is rounded once per 16 indices this way instead of six times (a Gram matrix of 1620 columns: 101 roundings, all of one
// sign's sums).  Three chains as well: dependent MFMAs issue every 64 cycles, independent ones every 40.
constexpr int CHAINS = 3;
__device__ __forceinline__ void mac(const bf16x8 (&A)[3], const bf16x8 (&B)[3], f32x16 (&acc)[CHAINS]) {
  acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[2], B[0], acc[2], 0, 0, 0);
  acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[0], acc[1], 0, 0, 0);
  acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[2], acc[2], 0, 0, 0);
  acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[1], acc[1], 0, 0, 0);
  acc[2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[1], acc[2], 0, 0, 0);
  acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[0], acc[0], 0, 0, 0);
}
__device__ __forceinline__ void mac(const bf16x8 (&A)[2], const bf16x8 (&B)[2], f32x16 (&acc)[CHAINS]) {
  acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[1], B[0], acc[1], 0, 0, 0);
  acc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[0], acc[0], 0, 0, 0);
  acc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(A[0], B[1], acc[1], 0, 0, 0);
}

// Where an element of a plane lies: columns in panels of 32, each panel all rows of 64 bytes.  The 64- or 128-row slice that a
// product step reads along rows is one run then, and the slice it reads across rows is runs of 2 KB; plain rows gave 64-byte
// pieces — half an L2 line each — at a stride that for 2048 columns kept them in one L2 channel.
__device__ __forceinline__ int64_t element(int rows, int row, int col) {
  return ((int64_t)(col >> 5) * rows + row) * 32 + (col & 31);
}

// ---- norm, pack, unpack ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

__device__ __forceinline__ const Item& find_item(const Items& a, int& blk) {
  int i = 0;
  while (i + 1 < a.n && blk >= a.it[i + 1].blocks) ++i;
  blk -= a.it[i].blocks;
  return a.it[i];
}

// elements col .. col + 7 of a row that ends at `cols`; `vec`: the row's address and stride allow 16-byte accesses
__device__ __forceinline__ void get8(const float* row, int col, int cols, int vec, float (&v)[8]) {
  if (vec && col + 8 <= cols) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(row + col), b = *reinterpret_cast<const f32x4*>(row + col + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? row[col + i] : 0.f;
  }
}
__device__ __forceinline__ void get8(const __bf16* row, int col, int cols, int vec, float (&v)[8]) {
  typedef __bf16 b8 __attribute__((ext_vector_type(8)));
  if (vec && col + 8 <= cols) {
    const b8 a = *reinterpret_cast<const b8*>(row + col);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? (float)row[col + i] : 0.f;
  }
}
__device__ __forceinline__ int vector_rows(const Item& it, int esz) {
  return (((uint64_t)(uintptr_t)it.p | (uint64_t)(it.sb * esz) | (uint64_t)(it.sr * esz)) & 15) == 0;
}

// Sums of squares in 64 bits, and the norm and its reciprocal too (pack_kernel): no matrix that fits fp32 overflows or vanishes in
// its norm.  The item's `nb` workgroups of a matrix take its units of 8 columns in turn.
template <typename E>
__global__ __launch_bounds__(256) void sumsq_kernel(const Items a, double* part) {
  __shared__ double red[4];
  int blk = blockIdx.x;
  const Item& it = find_item(a, blk);
  const int mat = blk / it.nb, b = blk - mat * it.nb, vec = vector_rows(it, sizeof(E));
  const int upr = (it.cols + 7) / 8;
  const int64_t units = (int64_t)it.rows * upr;
  const E* src = reinterpret_cast<const E*>(it.p) + mat * it.sb;
  double s = 0.0;
  for (int64_t u = (int64_t)b * 256 + threadIdx.x; u < units; u += (int64_t)it.nb * 256) {
    const unsigned r = (unsigned)u / (unsigned)upr, col = ((unsigned)u - r * upr) * 8;
    float v[8];
    get8(src + r * it.sr, (int)col, it.cols, vec, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += (double)v[i] * (double)v[i];
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) part[it.part + (int64_t)mat * it.nb + b] = s;
}

// X_0 = G / (norm + eps) as planes, zeros in the padding.  One unit of 8 columns per thread and turn.
template <typename E>
__global__ __launch_bounds__(256) void pack_kernel(const Items a, const double* part, short* ws, float eps) {
  constexpr int NP = Pieces<E>::n;
  __shared__ double red[4];
  int blk = blockIdx.x;
  const Item& it = find_item(a, blk);
  const unsigned upr = it.cp / 8, units = it.rp * upr, bpm = (units + TURN - 1) / TURN;
  const int mat = blk / bpm, vec = vector_rows(it, sizeof(E));
  const unsigned first = (blk - mat * bpm) * TURN;
  double s = 0.0;
  for (int i = threadIdx.x; i < it.nb; i += 256) s += part[it.part + (int64_t)mat * it.nb + i];
  s = block_sum(s, red);
  // (the reciprocal of a norm above 8.5e37 or below 2.9e-39 is no normal fp32 number; X_0 is one rounding of the 64-bit product)
  const double inv = 1.0 / (sqrt(s) + (double)eps);
  const E* src = reinterpret_cast<const E*>(it.p) + mat * it.sb;
  short* x = ws + it.base + mat * it.per;
  const int64_t plane = (int64_t)it.rp * it.cp;
  for (unsigned u = first + threadIdx.x; u < min(units, first + TURN); u += 256) {
    const unsigned r = u / upr, col = (u - r * upr) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if ((int)r < it.rows) get8(src + r * it.sr, (int)col, it.cols, vec, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)((double)v[i] * inv);
    if ((int)r >= it.rows || (int)col + 8 > it.cols) {      // the padding is 0 even when inv is not a number
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((int)r >= it.rows || (int)col + i >= it.cols) v[i] = 0.f;
    }
    bf16x8 P[NP];
    split(v, P);
#pragma unroll
    for (int p = 0; p < NP; ++p) *reinterpret_cast<bf16x8*>(x + p * plane + element(it.rp, r, col)) = P[p];
  }
}

template <typename E>
__global__ __launch_bounds__(256) void unpack_kernel(const Items a, const short* ws, int which) {
  constexpr int NP = Pieces<E>::n;
  int blk = blockIdx.x;
  const Item& it = find_item(a, blk);
  const unsigned upr = it.cp / 8, units = it.rp * upr, bpm = (units + TURN - 1) / TURN;
  const int mat = blk / bpm, vec = vector_rows(it, sizeof(E));
  const unsigned first = (blk - mat * bpm) * TURN;
  const int64_t plane = (int64_t)it.rp * it.cp;
  const short* x = ws + it.base + mat * it.per + which * NP * plane;
  E* dst = reinterpret_cast<E*>(it.p) + mat * it.sb;
  for (unsigned u = first + threadIdx.x; u < min(units, first + TURN); u += 256) {
    const int r = (int)(u / upr), col = (int)(u - r * upr) * 8;
    if (r >= it.rows || col >= it.cols) continue;
    bf16x8 P[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) P[p] = *reinterpret_cast<const bf16x8*>(x + p * plane + element(it.rp, r, col));
    E v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      short q[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) q[p] = P[p][i];
      v[i] = (E)join(q);
    }
    E* out = dst + r * it.sr + col;
    if (vec && col + 8 <= it.cols) {
      typedef E ev __attribute__((ext_vector_type(16 / sizeof(E))));
#pragma unroll
      for (int i = 0; i < (int)(sizeof(E) / 2); ++i) {
        ev t;
#pragma unroll
        for (int e = 0; e < (int)(16 / sizeof(E)); ++e) t[e] = v[i * (16 / sizeof(E)) + e];
        *reinterpret_cast<ev*>(out + i * (16 / sizeof(E))) = t;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < it.cols) out[i] = v[i];
    }
  }
}

// ---- the products --------------------------------------------------------------------------------------------------------------
enum { GRAM = 0, POLY = 1, APPLY = 2 };
constexpr int BK = 32;

struct Operand {
  const short* p;      // plane 0
  int64_t plane;
  int rows, limit;     // limit: rows (row form) or columns (column form) that exist, a multiple of 32
};

typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 resource(const short* p) {
  const unsigned long long a = (unsigned long long)p;
  return (i32x4){(int)__builtin_amdgcn_readfirstlane((unsigned)a), (int)__builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffff), -1,
                 0x00020000};
}
// 64 lanes x 16 bytes -> 1 KB of LDS, as inline assembly because hipcc would wait for it in front of the next ds_read of any
// stage.  No register output; the counted waits are in tile_product.
// `at`: its byte address in LDS, wave-uniform.
__device__ __forceinline__ void dma16(i32x4 rsrc, unsigned at, int voff, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(at), "v"(voff), "s"(rsrc), "s"(soff)
               : "memory", "m0");
}

// LDS image of one operand's BM x 32 slice: NP planes, row form [BM][32] or column form [32][BM], the 16-byte units of a row
// permuted (lds_swizzle.h) so that neither form's fragment reads meet in a bank.  Filled by LDS-DMA straight
// from the planes, the permutation is on the source side.
template <int NP, int BM, int NW, bool COL>
struct Slice {
  static constexpr int LD = COL ? BM : BK, ROWS = COL ? BK : BM, UPR = LD / 8;
  static constexpr int PLANE = BM * BK;
  static constexpr int DMAS = PLANE * 2 / 1024 / NW;      // instructions per wave and plane
  static_assert(DMAS >= 1, "tile too small");

  __device__ __forceinline__ static int swz(int row) { return unit_swizzle<UPR>(row); }

  // byte offsets of the lane's units at k = 0.  Rows behind the limit repeat the last one: blocks that hold them are not stored.
  __device__ __forceinline__ static void offsets(const Operand& o, int i0, int wave, int lane, int (&off)[DMAS]) {
#pragma unroll
    for (int u = 0; u < DMAS; ++u) {
      const int idx = (u * NW + wave) * 64 + lane, row = idx / UPR, unit = (idx % UPR) ^ swz(row);
      const int gr = COL ? row : min(i0 + row, o.limit - 1), gc = COL ? min(i0 + unit * 8, o.limit - 8) : unit * 8;
      off[u] = (int)element(o.rows, gr, gc) * 2;
    }
  }
  __device__ __forceinline__ static int step_bytes(const Operand& o) { return COL ? BK * 64 : o.rows * 64; }
  __device__ __forceinline__ static void issue(const i32x4 (&rsrc)[NP], const int (&off)[DMAS], int soff, unsigned at) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int u = 0; u < DMAS; ++u) dma16(rsrc[p], at + p * PLANE * 2 + u * NW * 1024, off[u], soff);
  }
  // MFMA operand: index i0 + (lane & 31), reduction 16 c + 8 (lane >> 5) + 0..7
  __device__ __forceinline__ static void frag(const short* lds, int i0, int c, int lane, bf16x8 (&P)[NP]) {
    if constexpr (!COL) {
      const int row = i0 + (lane & 31);
      const short* s = lds + row * LD + (((2 * c + (lane >> 5)) ^ swz(row)) << 3);
#pragma unroll
      for (int p = 0; p < NP; ++p) P[p] = *reinterpret_cast<const bf16x8*>(s + p * PLANE);
    } else {
      const int row = 16 * c + 8 * (lane >> 5) + ((lane & 15) >> 2), unit = i0 / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      const short* s0 = lds + row * LD + ((unit ^ swz(row)) << 3) + 4 * (lane & 1);
      const short* s1 = lds + (row + 4) * LD + ((unit ^ swz(row + 4)) << 3) + 4 * (lane & 1);
      typedef const __attribute__((address_space(3))) short* lds_t;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_t)(s0 + p * PLANE));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_t)(s1 + p * PLANE));
        P[p] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
  }
};

struct Out {
  short* p;
  int64_t plane;
  int rows, cols, mirror;
  const short* add;     // POLY: A planes (same layout)
  float a, b, c;
};

// 64-wide tiles: 2 x 2 waves of 32 x 32, three stages in LDS (48 or 72 KB: three or two workgroups per CU); 128-wide ones: 2 x 4 waves
// of 64 x 32, two stages (64 KB in bf16, two workgroups per CU; 96 KB in fp32, one).  Two waves per SIMD or more either way, so
// that one's LDS reads and DMA issue run under another's MFMAs; the barriers too, but for 128-wide fp32 tiles.
template <int BM> struct Shape { static constexpr int waves = BM == 64 ? 4 : 8, wi = BM == 64 ? 1 : 2, stages = BM == 64 ? 3 : 2; };

template <int NP, int BM, bool CA, bool CB>
__device__ __forceinline__ void tile_product(const Operand& A, const Operand& B, int K, const Out& o, int i0, int j0, short* lds) {
  constexpr int NW = Shape<BM>::waves, W = Shape<BM>::wi, STAGES = Shape<BM>::stages;     // W: 32-row blocks of a wave
  typedef Slice<NP, BM, NW, CA> SA;
  typedef Slice<NP, BM, NW, CB> SB;
  constexpr int STAGE = 2 * NP * BM * BK, PER_STAGE = NP * (SA::DMAS + SB::DMAS);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int wi = (NW == 4 ? wave >> 1 : wave >> 2) * 32 * W, wj = (NW == 4 ? wave & 1 : wave & 3) * 32;
  i32x4 ra[NP], rb[NP];
  int oa[SA::DMAS], ob[SB::DMAS];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    ra[p] = resource(A.p + p * A.plane);
    rb[p] = resource(B.p + p * B.plane);
  }
  SA::offsets(A, i0, wave, lane, oa);
  SB::offsets(B, j0, wave, lane, ob);
  const int sa = SA::step_bytes(A), sb = SB::step_bytes(B), steps = K / BK;
  const unsigned base = (unsigned)(unsigned long long)(const __attribute__((address_space(3))) short*)lds + wave * 1024;
  int next = 0, next_a = 0, next_b = 0;      // the stage and source offsets of the next issue
  auto issue = [&]() {
    SA::issue(ra, oa, next_a, base + next * STAGE * 2);
    SB::issue(rb, ob, next_b, base + next * STAGE * 2 + NP * SA::PLANE * 2);
    next_a += sa;
    next_b += sb;
    next = next + 1 == STAGES ? 0 : next + 1;
  };
  f32x16 acc[W][CHAINS];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int k = 0; k < CHAINS; ++k)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][k][e] = 0.f;
  bf16x8 fa[2][W][NP], fb[2][NP];            // the two 16-wide halves of a step
  auto read = [&](int stage, int c) {
    const short* la = lds + stage * STAGE;
    const short* lb = la + NP * SA::PLANE;
#pragma unroll
    for (int i = 0; i < W; ++i) SA::frag(la, wi + 32 * i, c, lane, fa[c][i]);
    SB::frag(lb, wj, c, lane, fb[c]);
  };
  auto multiply = [&](int c) {               // lane = row i, registers run along j
#pragma unroll
    for (int i = 0; i < W; ++i) mac(fb[c], fa[c][i], acc[i]);
  };
  // Stage s + 1 is waited for between the two halves of step s, so the fragments of each half are read under the other half's
  // MFMAs; behind that barrier every wave has its last fragments of stage s, whose place stage s + STAGES takes.
  for (int s = 0; s < STAGES && s < steps; ++s) issue();
  if (steps >= STAGES) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((STAGES - 1) * PER_STAGE) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  __syncthreads();
  read(0, 0);
  for (int s = 0, stage = 0; s < steps; ++s) {
    read(stage, 1);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    if (s + 1 < steps) {
      if (s + STAGES <= steps) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((STAGES - 2) * PER_STAGE) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
      __syncthreads();
      if (s + STAGES < steps) issue();
      read(stage, 0);
    }
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
      const int row = i0 + wi + 32 * i + (lane & 31);
      if (i0 + wi + 32 * i >= o.rows || j0 + wj >= o.cols) continue;    // sides are multiples of 32
#pragma unroll
      for (int h = 0; h < 2; ++h) {          // two runs of 4 columns, 8 apart
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (acc[i][2][8 * h + e] + acc[i][1][8 * h + e]) + acc[i][0][8 * h + e];
        const int col = j0 + wj + 16 * h + 4 * half;
        if (o.add) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int64_t at = element(o.rows, row, col + 8 * g);
            s16x4 q[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p) q[p] = *reinterpret_cast<const s16x4*>(o.add + p * o.plane + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              short x[NP];
#pragma unroll
              for (int p = 0; p < NP; ++p) x[p] = q[p][e];
              v[4 * g + e] = fmaf(o.c, v[4 * g + e], o.b * join(x)) + (row == col + 8 * g + e ? o.a : 0.f);
            }
          }
        }
        bf16x8 P[NP];
        split(v, P);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          short* dst = o.p + p * o.plane;
          *reinterpret_cast<s16x4*>(dst + element(o.rows, row, col)) = __builtin_shufflevector(P[p], P[p], 0, 1, 2, 3);
          *reinterpret_cast<s16x4*>(dst + element(o.rows, row, col + 8)) = __builtin_shufflevector(P[p], P[p], 4, 5, 6, 7);
          if (o.mirror) {
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[element(o.rows, col + (e & 3) + 8 * (e >> 2), row)] = P[p][e];
          }
        }
      }
    }
}

template <int NP, int BM>
__global__ __launch_bounds__(64 * Shape<BM>::waves) void product_kernel(const Table t, short* ws, int op, int flip, float ca, float cb, float cc) {
  __shared__ __attribute__((aligned(1024))) short lds[Shape<BM>::stages * 2 * NP * BM * BK];
  int blk = blockIdx.x, ci = 0;
  while (ci + 1 < t.ncls && blk >= t.tiles[ci + 1]) ++ci;
  blk -= t.tiles[ci];
  // neighbouring tiles, which read the same panels, on one XCD: workgroups are dealt round-robin to the 8 XCDs, so each of them
  // gets one contiguous run of the class (of each class: the runs of a launch are equally long)
  const int per8 = (t.tiles[ci + 1] - t.tiles[ci]) / 8;
  if (blk < per8 * 8) blk = (blk % 8) * per8 + blk / 8;
  const TCls& c = t.c[ci];
  const int64_t xp = (int64_t)c.rp * c.cp, mp = (int64_t)c.m * c.m;
  int ti, tj, mat;
  if (op == APPLY) {
    const int nj = (c.cp + BM - 1) / BM, per = nj * ((c.rp + BM - 1) / BM);
    mat = blk / per;
    const int k = blk - mat * per;
    ti = k / nj;
    tj = k - ti * nj;
  } else {
    const int n = (c.m + BM - 1) / BM, per = n * (n + 1) / 2;
    mat = blk / per;
    int k = blk - mat * per;
    for (ti = 0; k >= n - ti; ++ti) k -= n - ti;
    tj = ti + k;
  }
  short* base = ws + c.base + mat * c.per;
  short *x = base + (flip ? NP * xp : 0), *y = base + (flip ? 0 : NP * xp), *am = base + 2 * NP * xp, *qm = am + NP * mp;
  const int i0 = ti * BM, j0 = tj * BM;
  if (op == GRAM) {
    const Operand X = {x, xp, c.rp, c.tall ? c.cp : c.rp};
    const Out o = {am, mp, c.m, c.m, ti != tj, nullptr, 0.f, 0.f, 0.f};
    if (c.tall) tile_product<NP, BM, true, true>(X, X, c.rp, o, i0, j0, lds);
    else tile_product<NP, BM, false, false>(X, X, c.cp, o, i0, j0, lds);
  } else if (op == POLY) {
    const Operand M = {am, mp, c.m, c.m};
    const Out o = {qm, mp, c.m, c.m, ti != tj, am, ca, cb, cc};
    tile_product<NP, BM, false, false>(M, M, c.m, o, i0, j0, lds);
  } else {
    const Operand X = {x, xp, c.rp, c.tall ? c.rp : c.cp}, M = {qm, mp, c.m, c.m};
    const Out o = {y, xp, c.rp, c.cp, 0, nullptr, 0.f, 0.f, 0.f};
    if (c.tall) tile_product<NP, BM, false, false>(X, M, c.m, o, i0, j0, lds);
    else tile_product<NP, BM, false, true>(M, X, c.m, o, i0, j0, lds);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
constexpr int64_t MAX_GRID = 0xffffffffll / 512;   // a launch holds less than 2^32 threads

static int pad32(int n) { return (n + 31) / 32 * 32; }

static int check_items(const neosr_ns_item* items, int n, int dtype, const char* who) {
  NEOSR_CHECK(n >= 0 && (items || n == 0), "%s: null items", who);
  NEOSR_CHECK(dtype == NEOSR_DT_F32 || dtype == NEOSR_DT_BF16, "%s: dtype %d", who, dtype);
  const int esz = dtype == NEOSR_DT_F32 ? 4 : 2;
  for (int i = 0; i < n; ++i) {
    const neosr_ns_item& it = items[i];
    NEOSR_CHECK(it.rows >= 1 && it.cols >= 1 && it.rows <= 32768 && it.cols <= 32768 && it.count >= 1 && it.count <= 65536,
                "%s: item %d is %d x (%d x %d) (sides 1 to 32768, 1 to 65536 matrices)", who, i, it.count, it.rows, it.cols);
    NEOSR_CHECK((int64_t)pad32(it.rows) * pad32(it.cols) <= 1 << 29, "%s: item %d of %d x %d elements is too large (2^29)", who, i, it.rows,
                it.cols);
    NEOSR_CHECK(it.in && it.out && ((uintptr_t)it.in | (uintptr_t)it.out) % esz == 0, "%s: item %d: null or misaligned pointer", who, i);
  }
  return 0;
}

// The classes of items [i0, return value): as many items as fit MAXCLS shapes.  `bytes`: the batch's workspace.
static int build(const neosr_ns_item* items, int i0, int n, int np, Classes& t, int64_t* bytes, int64_t* part_at) {
  t.n = 0;
  int i = i0;
  for (; i < n; ++i) {
    int k = 0;
    while (k < t.n && (t.c[k].rows != items[i].rows || t.c[k].cols != items[i].cols)) ++k;
    if (k == t.n) {
      if (k == MAXCLS) break;
      Cls& c = t.c[t.n++];
      c = Cls{};
      c.rows = items[i].rows;
      c.cols = items[i].cols;
      c.rp = pad32(c.rows);
      c.cp = pad32(c.cols);
      c.tall = c.rows > c.cols;
      c.m = c.tall ? c.cp : c.rp;
      const int64_t nb = ((int64_t)c.rows * ((c.cols + 7) / 8) + TURN - 1) / TURN;
      c.nb = (int)(nb < 256 ? nb : 256);
    }
    if ((int64_t)t.c[k].count + items[i].count > (1 << 20)) break;
    t.c[k].count += items[i].count;
  }
  int64_t shorts = 0, parts = 0;
  for (int k = 0; k < t.n; ++k) {
    Cls& c = t.c[k];
    c.per = 2 * np * ((int64_t)c.rp * c.cp + (int64_t)c.m * c.m);
    c.base = shorts;
    shorts += c.per * c.count;
    c.part = parts;
    parts += (int64_t)c.nb * c.count;
  }
  *part_at = shorts * 2;                    // bytes; a multiple of 16
  *bytes = shorts * 2 + parts * 8;
  return i;
}

static int tiles_of(const Cls& c, int BM, int op) {
  const int n = (c.m + BM - 1) / BM;
  return op == APPLY ? ((c.rp + BM - 1) / BM) * ((c.cp + BM - 1) / BM) : n * (n + 1) / 2;
}

static int depth(const Cls& c, int op) { return op != GRAM ? c.m : (c.tall ? c.rp : c.cp); }

// 128-wide tiles move half as much through L2 and LDS as 64-wide ones and take over from 512 of them in a launch on, two for each
// CU.  bf16: the symmetric products of 1024- to 2304-wide matrices (208 tiles of 128) were 77 us in 64-wide tiles against 87, their
// third product (656 tiles) 103 us in 128-wide tiles against 134.  Five steps by this rule / in 64-wide tiles alone / in 128-wide ones
// alone, us: bf16 16 x 768^2 707 / 700 / 730, 8 x 1024^2 738 / 778 / 783, 4 x 1536^2 1137 / 1188 / 1174, 6 x 2048^2 3275 / 4438 /
// 3266; fp32, where one of them fills a CU, 1225 / 1172 / 1366, 1284 / 1335 / 1450, 2079 / 2022 / 2278, 6390 / 7176 / 6392.  Sides
// below 512 would mostly pad them.
template <typename E>
static int products(const Classes& t, short* ws, int op, int flip, const float* k, hipStream_t st) {
  int64_t wide = 0;
  for (int i = 0; i < t.n; ++i)
    if (t.c[i].m >= 512) wide += (int64_t)tiles_of(t.c[i], 128, op) * t.c[i].count;
  // the longest reductions first: the tiles of a launch end together
  int order[MAXCLS];
  for (int i = 0; i < t.n; ++i) {
    int j = i;
    for (; j > 0 && depth(t.c[order[j - 1]], op) < depth(t.c[i], op); --j) order[j] = order[j - 1];
    order[j] = i;
  }
  for (int pass = 0; pass < 2; ++pass) {
    Table s;
    s.ncls = 0;
    int64_t total = 0;
    for (int i = 0; i < t.n; ++i) {
      const Cls& c = t.c[order[i]];
      if ((wide >= 512 && c.m >= 512) != (pass == 1)) continue;
      s.tiles[s.ncls] = (int)total;
      s.c[s.ncls++] = {c.base, c.per, c.rp, c.cp, c.m, c.tall};
      total += (int64_t)tiles_of(c, pass ? 128 : 64, op) * c.count;
      NEOSR_CHECK(total <= MAX_GRID, "neosr_newton_schulz: too many tiles");
    }
    if (s.ncls == 0) continue;
    s.tiles[s.ncls] = (int)total;
    if (pass) product_kernel<Pieces<E>::n, 128><<<(unsigned)total, 512, 0, st>>>(s, ws, op, flip, k[0], k[1], k[2]);
    else product_kernel<Pieces<E>::n, 64><<<(unsigned)total, 256, 0, st>>>(s, ws, op, flip, k[0], k[1], k[2]);
    NEOSR_LAUNCH_CHECK();
  }
  return 0;
}

enum { SUMSQ = 0, PACK = 1, UNPACK = 2 };

// the element-wise passes over items [i0, i1), MAXITEM per launch
template <typename E>
static int items_pass(int kind, const neosr_ns_item* items, int i0, int i1, const Classes& t, short* ws, double* part, float eps, int which,
                      hipStream_t st) {
  int64_t first[MAXCLS] = {};
  for (int i = i0; i < i1;) {
    Items a;
    a.n = 0;
    int64_t total = 0;
    for (; i < i1 && a.n < MAXITEM; ++i) {
      const neosr_ns_item& x = items[i];
      int k = 0;
      while (t.c[k].rows != x.rows || t.c[k].cols != x.cols) ++k;
      const Cls& c = t.c[k];
      const int64_t blocks = (int64_t)x.count * (kind == SUMSQ ? c.nb : ((int64_t)c.rp * (c.cp / 8) + TURN - 1) / TURN);
      NEOSR_CHECK(blocks <= MAX_GRID, "neosr_newton_schulz: item %d is too large", i);
      if (total + blocks > MAX_GRID) break;
      a.it[a.n++] = {kind == UNPACK ? (char*)x.out : (char*)const_cast<void*>(x.in), kind == UNPACK ? x.out_sb : x.in_sb,
                     kind == UNPACK ? x.out_sr : x.in_sr, c.base + first[k] * c.per, c.per, c.part + first[k] * c.nb, c.rows, c.cols,
                     c.rp, c.cp, c.nb, (int)total};
      first[k] += x.count;
      total += blocks;
    }
    if (kind == SUMSQ) sumsq_kernel<E><<<(unsigned)total, 256, 0, st>>>(a, part);
    else if (kind == PACK) pack_kernel<E><<<(unsigned)total, 256, 0, st>>>(a, part, ws, eps);
    else unpack_kernel<E><<<(unsigned)total, 256, 0, st>>>(a, ws, which);
    NEOSR_LAUNCH_CHECK();
  }
  return 0;
}

template <typename E>
static int run(const neosr_ns_item* items, int n, int steps, const float* coef, float eps, char* ws, hipStream_t st) {
  for (int i = 0; i < n;) {
    Classes t;
    int64_t bytes, part_at;
    const int end = build(items, i, n, Pieces<E>::n, t, &bytes, &part_at);
    short* w = (short*)ws;
    double* part = (double*)(ws + part_at);
    int rc = items_pass<E>(SUMSQ, items, i, end, t, w, part, eps, 0, st);
    if (!rc) rc = items_pass<E>(PACK, items, i, end, t, w, part, eps, 0, st);
    for (int s = 0; s < steps && !rc; ++s)
      for (int op = GRAM; op <= APPLY && !rc; ++op) rc = products<E>(t, w, op, s & 1, coef + 3 * s, st);
    if (!rc) rc = items_pass<E>(UNPACK, items, i, end, t, w, part, eps, steps & 1, st);
    if (rc) return rc;
    i = end;
  }
  return 0;
}

static int64_t workspace(const neosr_ns_item* items, int n, int dtype) {
  const int np = dtype == NEOSR_DT_F32 ? Pieces<float>::n : Pieces<__bf16>::n;
  int64_t most = 0;
  for (int i = 0; i < n;) {
    Classes t;
    int64_t bytes, part_at;
    i = build(items, i, n, np, t, &bytes, &part_at);
    if (bytes > most) most = bytes;
  }
  return most;
}

}  // namespace ns

extern "C" int64_t neosr_newton_schulz_workspace_bytes(const neosr_ns_item* items, int32_t n, int32_t dtype) {
  if (ns::check_items(items, n, dtype, "neosr_newton_schulz_workspace_bytes")) return -1;
  return ns::workspace(items, n, dtype);
}

extern "C" int neosr_newton_schulz(const neosr_ns_item* items, int32_t n, int32_t dtype, int32_t steps, const float* coefficients, float eps,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  if (ns::check_items(items, n, dtype, "neosr_newton_schulz")) return 1;
  NEOSR_CHECK(steps >= 1 && steps <= 64 && coefficients, "neosr_newton_schulz: %d steps (1 to 64)", steps);
  NEOSR_CHECK(eps >= 0.f && eps < HUGE_VALF, "neosr_newton_schulz: eps must be finite and not negative");
  if (n == 0) return 0;
  const int64_t need = ns::workspace(items, n, dtype);
  NEOSR_CHECK(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need,
              "neosr_newton_schulz: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)workspace_bytes, (long long)need);
  return dtype == NEOSR_DT_F32 ? ns::run<float>(items, n, steps, coefficients, eps, (char*)workspace, (hipStream_t)stream)
                               : ns::run<__bf16>(items, n, steps, coefficients, eps, (char*)workspace, (hipStream_t)stream);
}
