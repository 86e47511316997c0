// attention_pack.hip — what the packed forms of attention_fwd.hip / attention_bwd.hip read: K and V (or Q and dO) as bf16
// pieces in the byte order of their LDS tiles (attention.h: Tile), masked keys as zeros, and one truth word for each tile.
//
// A K / V tile is staged by every row block of its head (32 of them at 4096 rows), so what staging costs beyond a copy —
// strides, head sizes that are no vector, masks, and for fp32 the split into three pieces, 5.5 vector instructions an element —
// is paid once here and the product kernels stage with LDS-DMA alone, without a register or a vector instruction.
// Bound by HBM / L2: reads each tensor once, writes 2 or 6 bytes an element (84 MB of Q, dO, O in 19 us).
#include <math.h>
#include "attention.h"

namespace attn {

// one 8-channel unit per thread; a tile's rows are covered by ROWS * DP / 8 consecutive threads
template <typename E, int DP>
__device__ __forceinline__ void pack_kv_block(const Args& a, unsigned block) {
  constexpr int NP = Pieces<E>::n, KT = tile_rows<NP, DP>(), UPR = DP / 8, UNITS = KT * UPR;
  typedef Tile<NP, DP, KT> T;
  constexpr int WGS = 2 * UNITS / 256;      // workgroups of a tile
  static_assert(UNITS % 256 == 0, "whole workgroups");
  const int64_t tile = block / WGS;
  const int idx = (int)(block % WGS) * 256 + threadIdx.x, which = idx / UNITS, u = idx % UNITS, row = u / UPR, unit = u % UPR;
  const int t = (int)(tile % a.kv_tiles), bh = (int)(tile / a.kv_tiles), b = bh / a.Hk, hk = bh % a.Hk;
  const int j = t * KT + row;
  const Tensor4& x = which ? a.v : a.k;
  Raw8<E> r[1];
  zero(r[0]);
  if (key_ok(a, b, j)) r[0] = load8(reinterpret_cast<const E*>(x.p) + b * x.sb + j * x.sl + (int64_t)hk * x.sh, unit * 8, a.D, a.vec);
  bf16x8 P[1][NP];
  operands(r, P);
  if (NP == 3 && DP > a.D && which && unit == a.D / 8 && key_ok(a, b, j)) {    // V's first padding channel: P V's is the row sum of P
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i == a.D % 8) P[0][0][i] = 0x3f80;
  }
  T::put(reinterpret_cast<short*>(a.kv_img + tile * tile_bytes<NP, DP>()) + which * T::ELEMS, row, unit, P[0]);
  if (hk == 0 && block % WGS == 0 && threadIdx.x < 64) {
    const unsigned long long w = __ballot((int)threadIdx.x < KT && key_ok(a, b, t * KT + threadIdx.x));
    if (threadIdx.x == 0) a.words[(int64_t)b * a.kv_tiles + t] = w;
  }
}

template <typename E, int DP>
__device__ __forceinline__ void pack_rows_block(const Args& a, unsigned block) {
  constexpr int NP = Pieces<E>::n, KT = tile_rows<NP, DP>(), UPR = DP / 8, WGS = KT * UPR / 256;
  typedef Tile<NP, DP, KT> T;
  static_assert(KT * UPR % 256 == 0, "whole workgroups");
  const int64_t tile = block / WGS;
  const int u = (int)(block % WGS) * 256 + threadIdx.x, row = u / UPR, unit = u % UPR;
  const int t = (int)(tile % a.row_tiles), bh = (int)(tile / a.row_tiles), b = bh / a.Hk, hk = bh % a.Hk;
  const int r = t * KT + row;
  Raw8<E> qd[2], o, rest;                // Q and dO
  zero(qd[0]);
  zero(qd[1]);
  zero(o);
  zero(rest);
  // (a row without a key passes no gradient, whatever its dO holds)
  if (r < a.R && a.lse[(int64_t)bh * a.R + r] != INFINITY) {
    const int pos = r / a.G, h = hk * a.G + (r - pos * a.G);
    qd[0] = load8(reinterpret_cast<const E*>(a.q.p) + b * a.q.sb + pos * a.q.sl + (int64_t)h * a.q.sh, unit * 8, a.D, a.vec);
    qd[1] = load8(reinterpret_cast<const E*>(a.dout.p) + b * a.dout.sb + pos * a.dout.sl + (int64_t)h * a.dout.sh, unit * 8, a.D, a.vec);
    const int64_t at = b * a.o.sb + pos * a.o.sl + (int64_t)h * a.o.sh;
    o = load8(reinterpret_cast<const E*>(a.o.p) + at, unit * 8, a.D, a.vec);
    if constexpr (NP == 1)
      if (a.rest) rest = load8(reinterpret_cast<const E*>(a.rest) + at, unit * 8, a.D, a.vec);
  }
  bf16x8 P[2][NP];
  short* base = reinterpret_cast<short*>(a.row_img + tile * tile_bytes<NP, DP>());
  operands(qd, P);
  T::put(base, row, unit, P[0]);
  T::put(base + T::ELEMS, row, unit, P[1]);
  float s = dot8(qd[1], o);
  if constexpr (NP == 1) s += dot8(qd[1], rest);
#pragma unroll
  for (int off = UPR / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (unit == 0 && r < a.R) a.delta[(int64_t)bh * a.R + r] = s;
}

// the K, V blocks first, the row blocks behind them
template <typename E, int DP>
__global__ __launch_bounds__(256) void pack_kernel(const Args a, unsigned kv_blocks) {
  if (blockIdx.x < kv_blocks) pack_kv_block<E, DP>(a, blockIdx.x);
  else pack_rows_block<E, DP>(a, blockIdx.x - kv_blocks);
}

int64_t words_bytes(const neosr_attention_desc* d) {
  const int kt = tile_rows_of(d->dtype, d->D);
  return align256((int64_t)d->B * ((d->Lk + kt - 1) / kt) * 8);
}

template <typename E, int DP>
static int launch_pack(const Args& a, bool kv, bool rows, hipStream_t st) {
  constexpr int WGS = tile_rows<Pieces<E>::n, DP>() * DP / 8 / 256;
  const int64_t nkv = kv ? (int64_t)a.B * a.Hk * a.kv_tiles * 2 * WGS : 0, nrows = rows ? (int64_t)a.B * a.Hk * a.row_tiles * WGS : 0;
  NEOSR_CHECK(nkv + nrows <= MAX_GRID, "neosr_attention: %lld workgroups", (long long)(nkv + nrows));
  if (nkv + nrows == 0) return 0;
  pack_kernel<E, DP><<<(unsigned)(nkv + nrows), 256, 0, st>>>(a, (unsigned)nkv);
  NEOSR_LAUNCH_CHECK();
  return 0;
}

int pack(const neosr_attention_desc* d, const Args& a, bool kv, bool rows, hipStream_t st) {
  const int dp = padded(d->D);
  if (d->dtype == NEOSR_DT_F32)
    return dp == 32 ? launch_pack<float, 32>(a, kv, rows, st) : (dp == 64 ? launch_pack<float, 64>(a, kv, rows, st) : launch_pack<float, 128>(a, kv, rows, st));
  return dp == 32 ? launch_pack<__bf16, 32>(a, kv, rows, st)
                  : (dp == 64 ? launch_pack<__bf16, 64>(a, kv, rows, st) : launch_pack<__bf16, 128>(a, kv, rows, st));
}

}  // namespace attn
