// attention_bwd.hip — gradients of attention with the probabilities formed again from the row statistics:
//   P = 2^(cs S - lse),  dP = dO V^T,  delta = rowsum(dO * O),  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
//
// Two passes, seven products instead of five: dq_kernel owns 32-row blocks and walks the keys, dkv_kernel owns 32-key blocks
// and walks the rows (of the whole group: the gradients of shared heads are one sum).  Each output element is then one
// register chain in a fixed order — the five-product form has to add dQ across key blocks through memory, with float atomics
// in an order that changes from run to run or with B Hk R D floats for every key block.
// dq_kernel forms S and dP transposed (attention.h), so lse and delta (attention_pack.hip) are per-lane scalars and dS^T is the B operand of
// dQ^T = K^T dS^T; dkv_kernel forms them upright (keys are the columns), so P and dS are the B operands of dV^T = dO^T P and
// dK^T = Q^T dS.
//
// Measured: 4 x 4096 of 8 / 2 heads x 64 bf16 dQ 229 us and dK, dV 305 us (900 TFLOP/s of their own products, matrix pipe
// 42-45 % busy beside a vector pipe at 44-56 %); 2 x 4096 of 6 x 30 fp32 203 and 282 us.  128-wide heads hold 348 registers in the
// dK, dV kernel: one wave per SIMD, 154 us for 2 x 2047 of 16 / 4 in causal order (two waves spill: 177 us).
// Forms that keep registers in scratch: fp32 128-wide dK, dV (128 bytes a lane: 2 x 2047 of 8 x 128 434 us) and single-wave dQ (284),
// fp32 64-wide single-wave dQ (104), and 40 bytes in fp32 32-wide dK, dV, the price of its three waves per SIMD (677 -> 657 us of the
// whole call).
#include <math.h>
#include "attention.h"
#include "prof.h"

namespace attn {

constexpr int FINE = 1024;

// ---- dQ ----------------------------------------------------------------------------------------------------------------------
// FEW (bf16, where there are at most FINE keys or at most FINE rows): P and dS keep a second piece, and the gradients are off by
// their own rounding alone (1.66e-3 to 1.75e-3 of their norm).  With one piece the rounding of P or dS adds as much again, as the
// root of the squares: 2.3e-3 to 2.4e-3 at any length and in the first rows of a causal call, 2.6e-3 over 5 keys, where dS adds up to 0
// and its roundings do not.  Long calls pay for it in the vector pipe that bounds them: forward and backward of 4 x 4096 of 8 / 2 heads
// x 64 957 us instead of 750, of 2 x 2047 of 16 / 4 x 128 in causal order 388 instead of 330, which bf16 does not ask for.  With few
// rows or keys it is nearly free (8 x 16 rows over 4096 keys of 8 / 4 x 64: 44.1 us of kernels against 43.6), and at the rule's end (4 x
// 1000 rows and keys of 8 / 4 x 64: 70 against 54) it is a tenth of a call, most of whose 150 us are not these kernels.
template <typename E, int DP, int NW, bool PACKED, int OCC, bool FEW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC))) void dq_kernel(const Args a) {
  constexpr int NP = Pieces<E>::n, KT = tile_rows<NP, DP>(), NC = DP / 16, ND = DP / 32, UPR = DP / 8;
  constexpr int UNITS = PACKED ? 1 : KT * UPR / (64 * NW);
  typedef Tile<NP, DP, KT> T;
  __shared__ __attribute__((aligned(1024))) short lds[(PACKED ? 2 : 1) * 2 * T::ELEMS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;

  int64_t w = xcd_order(blockIdx.x, gridDim.x);
  const int rb = a.causal ? a.nblk - 1 - (int)(w % a.nblk) : (int)(w % a.nblk);
  w /= a.nblk;
  const int split = (int)(w % a.nsplit);
  const int bh = (int)(w / a.nsplit), b = bh / a.Hk, hk = bh % a.Hk;
  const int blk0 = rb * 32 * NW, wr0 = blk0 + wave * 32;
  const int last = a.causal ? min(a.Lk, (min(a.R, blk0 + 32 * NW) - 1) / a.G + a.off + 1) : a.Lk;
  const Range keys = share(0, last, split, a.nsplit);
  const int kbeg = keys.beg, kend = keys.end;
  constexpr int TB = tile_bytes<NP, DP>();
  const char* img = nullptr;
  unsigned at = 0;
  const unsigned long long* words = nullptr;
  if constexpr (PACKED) {
    img = a.kv_img + ((int64_t)bh * a.kv_tiles + kbeg / KT) * TB + wave * 1024 + lane * 16;
    at = lds_address(lds) + wave * 1024;
    words = a.words + (int64_t)b * a.kv_tiles;
    if (kbeg < kend) dma_tile<TB, NW>(img, at);
  }

  const int r = wr0 + (lane & 31);
  const int pos = r / a.G, g = r - pos * a.G;
  const int lim = a.causal ? pos + a.off : 0x7fffffff;
  bf16x8 Q[NC][NP], dO[NC][NP];
  // (a row without a key — and the lanes behind the last row — has lse = +inf: P = 0, and what its dO holds is not read)
  const float lse = r < a.R ? a.lse[(int64_t)bh * a.R + r] : INFINITY;
  const float delta = r < a.R ? a.delta[(int64_t)bh * a.R + r] : 0.f;
  {
    const E* qrow = reinterpret_cast<const E*>(a.q.p) + b * a.q.sb + pos * a.q.sl + (int64_t)(hk * a.G + g) * a.q.sh;
    const E* drow = reinterpret_cast<const E*>(a.dout.p) + b * a.dout.sb + pos * a.dout.sl + (int64_t)(hk * a.G + g) * a.dout.sh;
    Raw8<E> x[NC], y[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      zero(x[c]);
      zero(y[c]);
      if (lse != INFINITY) {
        x[c] = load8(qrow, 16 * c + 8 * half, a.D, a.vec);
        y[c] = load8(drow, 16 * c + 8 * half, a.D, a.vec);
      }
    }
    operands(x, Q);
    operands(y, dO);
  }

  f32x16 dQ[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) dQ[n][i] = 0.f;

  const E* kbase = reinterpret_cast<const E*>(a.k.p) + b * a.k.sb + (int64_t)hk * a.k.sh;
  const E* vbase = reinterpret_cast<const E*>(a.v.p) + b * a.v.sb + (int64_t)hk * a.v.sh;
  Raw8<E> kr[UNITS], vr[UNITS];
  bool ok[UNITS], okl = false;
  auto fetch = [&](int k0) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int idx = u * 64 * NW + tid, j = k0 + idx / UPR, d = (idx % UPR) * 8;
      zero(kr[u]);
      zero(vr[u]);
      ok[u] = key_ok(a, b, j);
      if (j < a.Lk) {
        kr[u] = load8(kbase + j * a.k.sl, d, a.D, a.vec);
        vr[u] = load8(vbase + j * a.v.sl, d, a.D, a.vec);
      }
    }
    okl = lane < KT && key_ok(a, b, k0 + lane);
  };

  if constexpr (!PACKED)
    if (kbeg < kend) fetch(kbeg);

  for (int k0 = kbeg, buf = 0; k0 < kend; k0 += KT, buf ^= 1) {
    const short* kt = lds;
    unsigned long long valid;
    if constexpr (PACKED) {
      kt = lds + buf * 2 * T::ELEMS;
      valid = words[k0 / KT];
      dma_wait();
      __syncthreads();
      img += TB;
      if (k0 + KT < kend) dma_tile<TB, NW>(img, at + (buf ^ 1) * TB);
    } else {
      __syncthreads();
      float top = 0.f;
      auto stage = [&](int u, auto split) {
        const int idx = u * 64 * NW + tid, row = idx / UPR, unit = idx % UPR;
        bf16x8 P[NP];
        split(kr[u], P);
        T::put(lds, row, unit, P);
        split(vr[u], P);
        T::put(lds + T::ELEMS, row, unit, P);
      };
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        if (!ok[u]) {
          zero(kr[u]);
          zero(vr[u]);
        }
        stage(u, [](const Raw8<E>& r, bf16x8 (&P)[NP]) { pieces(r, P); });
        top = largest(vr[u], largest(kr[u], top));
      }
      if (__any(top >= BEYOND)) {                                  // (the same lane writes the same places again)
#pragma unroll
        for (int u = 0; u < UNITS; ++u) stage(u, [](const Raw8<E>& r, bf16x8 (&P)[NP]) { pieces_beyond(r, P); });
      }
      valid = __ballot(okl);
      __syncthreads();
      if (k0 + KT < kend) fetch(k0 + KT);
    }
    const short* vt = kt + T::ELEMS;
    if (valid == 0) continue;

#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      unsigned bits = (unsigned)(valid >> (32 * kb)) >> (4 * half);
      f32x16 S, X;
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = X[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        bf16x8 A[NP];
        T::rows(kt, 32 * kb, c, lane, A);
        S = mac(A, Q[c], S);
        T::rows(vt, 32 * kb, c, lane, A);
        X = mac(A, dO[c], X);
      }
      const int rel = lim - (k0 + 32 * kb) - 4 * half;
      if (rel < 28) bits &= rel < 0 ? 0u : (2u << rel) - 1u;
      if (!__all((bits & 0x0f0f0f0fu) == 0x0f0f0f0fu)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(bits >> acc_row(i) & 1u)) S[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = __builtin_amdgcn_exp2f(fmaf(S[i], a.cs, -lse)) * (X[i] - delta);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x[8];
        bf16x8 P[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = S[8 * c + e];
        pieces_of(x, P);
        [[maybe_unused]] bf16x8 rest[NP];
        if constexpr (FEW) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] -= (float)(__bf16)x[e];
          pieces_of(x, rest);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          bf16x8 A[NP];
          T::cols(kt, 32 * kb + 16 * c, 32 * n, lane, A);
          if constexpr (FEW) dQ[n] = mac(A, rest, dQ[n]);
          dQ[n] = mac(A, P, dQ[n]);
        }
      }
    }
  }

  if (r >= a.R) return;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dQ[n][4 * j + e] * a.scale;
      const int64_t to = (((int64_t)b * a.Lq + pos) * a.H + hk * a.G + g) * a.D;
      if (a.nsplit > 1) store4(a.part + (int64_t)split * a.B * a.Lq * a.H * a.D + to, 32 * n + 8 * j + 4 * half, a.D, x);
      else store4(reinterpret_cast<E*>(a.dq) + to, 32 * n + 8 * j + 4 * half, a.D, x);
    }
}

// ---- dK, dV ------------------------------------------------------------------------------------------------------------------
template <typename E, int DP, int NW, int OCC, bool FEW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC))) void dkv_kernel(const Args a) {
  constexpr int NP = Pieces<E>::n, RT = tile_rows<NP, DP>(), NC = DP / 16, ND = DP / 32;
  typedef Tile<NP, DP, RT> T;
  __shared__ __attribute__((aligned(1024))) short lds[2 * 2 * T::ELEMS];
  __shared__ __attribute__((aligned(16))) float stats[2][2 * RT];   // lse | delta of a tile's rows
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;

  int64_t w = xcd_order(blockIdx.x, gridDim.x);
  const int cb = (int)(w % a.nblk);
  w /= a.nblk;
  const int split = (int)(w % a.nsplit);
  const int bh = (int)(w / a.nsplit), b = bh / a.Hk, hk = bh % a.Hk;
  const int blk0 = cb * 32 * NW;
  const int j = blk0 + wave * 32 + (lane & 31);
  const bool ok = key_ok(a, b, j);

  const int rmin = a.causal ? (j - a.off) * a.G : 0;                // first row that sees the key
  int first = 0;                                                    // ... any key of the workgroup
  if (a.causal) first = min(a.R, max(0, (blk0 - a.off) * a.G) / 64 * 64);
  const Range rows = share(first, a.R, split, a.nsplit);
  const int rbeg = rows.beg, rend = rows.end;
  constexpr int TB = tile_bytes<NP, DP>();
  const char* img = a.row_img + ((int64_t)bh * a.row_tiles + rbeg / RT) * TB + wave * 1024 + lane * 16;
  const unsigned at = lds_address(lds) + wave * 1024;
  if (rbeg < rend) dma_tile<TB, NW>(img, at);
  const bool any = __any(ok);

  bf16x8 K[NC][NP], V[NC][NP];
  {
    const E* krow = reinterpret_cast<const E*>(a.k.p) + b * a.k.sb + j * a.k.sl + (int64_t)hk * a.k.sh;
    const E* vrow = reinterpret_cast<const E*>(a.v.p) + b * a.v.sb + j * a.v.sl + (int64_t)hk * a.v.sh;
    Raw8<E> x[NC], y[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      zero(x[c]);
      zero(y[c]);
      if (ok) {
        x[c] = load8(krow, 16 * c + 8 * half, a.D, a.vec);
        y[c] = load8(vrow, 16 * c + 8 * half, a.D, a.vec);
      }
    }
    operands(x, K);
    operands(y, V);
  }

  f32x16 dK[ND], dV[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) dK[n][i] = dV[n][i] = 0.f;

  float st[2 * RT / (64 * NW) > 0 ? 2 * RT / (64 * NW) : 1];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int i = tid, n = 0; i < 2 * RT; i += 64 * NW, ++n) {
      const int r = r0 + (i & (RT - 1));
      st[n] = i < RT ? INFINITY : 0.f;                              // rows behind the last one: P = 0
      if (r < rend) st[n] = (i < RT ? a.lse : a.delta)[(int64_t)bh * a.R + r];
    }
  };
  if (rbeg < rend) fetch(rbeg);
  for (int r0 = rbeg, buf = 0; r0 < rend; r0 += RT, buf ^= 1) {
    const short* qt = lds + buf * 2 * T::ELEMS;
    dma_wait();
#pragma unroll
    for (int i = tid, n = 0; i < 2 * RT; i += 64 * NW, ++n) stats[buf][i] = st[n];
    __syncthreads();
    if (r0 + RT < rend) {
      img += TB;
      dma_tile<TB, NW>(img, at + (buf ^ 1) * TB);
      fetch(r0 + RT);
    }
    const short* dt = qt + T::ELEMS;

    if (!any) continue;
#pragma unroll
    for (int rb = 0; rb < RT / 32; ++rb) {
      const int rel = rmin - (r0 + 32 * rb) - 4 * half;             // first allowed row in the lane's numbering
      unsigned bits = ok ? 0x0f0f0f0fu : 0u;
      if (rel > 0) bits &= rel >= 28 ? 0u : ~0u << rel;
      if (!__any(bits != 0u)) continue;
      f32x16 S, X;
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = X[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        bf16x8 A[NP];
        T::rows(qt, 32 * rb, c, lane, A);
        S = mac(A, K[c], S);
        T::rows(dt, 32 * rb, c, lane, A);
        X = mac(A, V[c], X);
      }
      if (!__all(bits == 0x0f0f0f0fu)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(bits >> acc_row(i) & 1u)) S[i] = -INFINITY;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 ls = *reinterpret_cast<const f32x4*>(stats[buf] + 32 * rb + 8 * q + 4 * half);
        const f32x4 de = *reinterpret_cast<const f32x4*>(stats[buf] + RT + 32 * rb + 8 * q + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(S[4 * q + e], a.cs, -ls[e]));
          S[4 * q + e] = p;
          X[4 * q + e] = p * (X[4 * q + e] - de[e]);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x[8];
        bf16x8 P[NP], dS[NP];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = S[8 * c + e];
        pieces_of(x, P);
        [[maybe_unused]] bf16x8 Pr[NP], dSr[NP];
        if constexpr (FEW) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] -= (float)(__bf16)x[e];
          pieces_of(x, Pr);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = X[8 * c + e];
        pieces_of(x, dS);
        if constexpr (FEW) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] -= (float)(__bf16)x[e];
          pieces_of(x, dSr);
        }
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          bf16x8 A[NP];
          T::cols(dt, 32 * rb + 16 * c, 32 * n, lane, A);
          if constexpr (FEW) dV[n] = mac(A, Pr, dV[n]);
          dV[n] = mac(A, P, dV[n]);
          T::cols(qt, 32 * rb + 16 * c, 32 * n, lane, A);
          if constexpr (FEW) dK[n] = mac(A, dSr, dK[n]);
          dK[n] = mac(A, dS, dK[n]);
        }
      }
    }
  }

  if (j >= a.Lk) return;
  const int64_t to = (((int64_t)b * a.Lk + j) * a.Hk + hk) * a.D, all = (int64_t)a.B * a.Lk * a.Hk * a.D;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float x[4], y[4];
      const int d = 32 * n + 8 * q + 4 * half;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = dK[n][4 * q + e] * a.scale;
        y[e] = dV[n][4 * q + e];
      }
      if (a.nsplit > 1) {
        store4(a.part + (int64_t)split * 2 * all + to, d, a.D, x);
        store4(a.part + ((int64_t)split * 2 + 1) * all + to, d, a.D, y);
      } else {
        store4(reinterpret_cast<E*>(a.dk) + to, d, a.D, x);
        store4(reinterpret_cast<E*>(a.dv) + to, d, a.D, y);
      }
    }
}

// out[i] = sum over splits of part[s * stride + i], in order, for up to three tensors (blockIdx.y)
struct Sums {
  const float* part[3];
  char* out[3];
  int64_t n[3], stride[3];
  int nsplit[3], count;
};
template <typename E>
__global__ __launch_bounds__(256) void sum_splits_kernel(const Sums t) {
  const int y = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = t.stride[y];
  if (i >= t.n[y]) return;
  const float* part = t.part[y] + i;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < t.nsplit[y]; ++k) s += part[k * stride];
  reinterpret_cast<E*>(t.out[y])[i] = (E)s;
}

static Plan plan_dq(const neosr_attention_desc* d) {
  return plan((int64_t)d->B * d->Hk, (int64_t)d->Lq * (d->H / d->Hk), d->Lk, d->D);
}
static Plan plan_dkv(const neosr_attention_desc* d) {
  return plan((int64_t)d->B * d->Hk, d->Lk, (int64_t)d->Lq * (d->H / d->Hk), 0);
}

// delta | partials of dQ | partials of dK, dV | packed K, V | truth words | packed Q, dO
struct BwdSpace {
  int64_t delta, part_q, part_kv, kv, words, rows;
  int64_t total() const { return delta + part_q + part_kv + kv + words + rows; }
};
static BwdSpace bwd_space(const neosr_attention_desc* d, const Plan& q, const Plan& kv) {
  BwdSpace s = {};
  const int64_t nq = q.nsplit > 1 ? (int64_t)q.nsplit * d->B * d->Lq * d->H * d->D : 0;
  const int64_t nkv = kv.nsplit > 1 ? (int64_t)kv.nsplit * 2 * d->B * d->Lk * d->Hk * d->D : 0;
  s.delta = align256((int64_t)d->B * d->H * d->Lq * 4);
  s.part_q = align256(nq * 4);
  s.part_kv = align256(nkv * 4);
  if (q.packed) {
    s.kv = align256((int64_t)d->B * d->Hk * image_bytes(d->dtype, d->D, d->Lk));
    s.words = words_bytes(d);
  }
  s.rows = align256((int64_t)d->B * d->Hk * image_bytes(d->dtype, d->D, (int64_t)d->Lq * (d->H / d->Hk)));
  return s;
}

template <typename E, int DP, bool FEW>
static int launch_dq(const Args& a, bool packed, unsigned grid, hipStream_t st) {
  constexpr int OCC = sizeof(E) == 4 && DP == 128 ? 1 : 2;
  if (packed) dq_kernel<E, DP, 4, true, OCC, FEW><<<grid, 256, 0, st>>>(a);
  else dq_kernel<E, DP, 1, false, DP == 128 ? 1 : 2, FEW><<<grid, 64, 0, st>>>(a);
  NEOSR_LAUNCH_CHECK();
  return 0;
}
template <typename E, int DP>
static int launch_dq(const Args& a, bool packed, unsigned grid, hipStream_t st) {
  if constexpr (sizeof(E) == 2)
    if (min(a.Lk, a.R) <= FINE) return launch_dq<E, DP, true>(a, packed, grid, st);
  return launch_dq<E, DP, false>(a, packed, grid, st);
}
template <typename E, int DP, bool FEW>
static int launch_dkv(const Args& a, bool packed, unsigned grid, hipStream_t st) {
  constexpr int OCC = DP == 128 ? 1 : (sizeof(E) == 4 && DP == 32 ? 3 : 2);
  constexpr int OCC1 = sizeof(E) == 2 && DP == 32 ? 2 : 1;            // single waves: LDS holds four or fewer for each CU otherwise
  if (packed) dkv_kernel<E, DP, 4, OCC, FEW><<<grid, 256, 0, st>>>(a);
  else dkv_kernel<E, DP, 1, OCC1, FEW><<<grid, 64, 0, st>>>(a);
  NEOSR_LAUNCH_CHECK();
  return 0;
}
template <typename E, int DP>
static int launch_dkv(const Args& a, bool packed, unsigned grid, hipStream_t st) {
  if constexpr (sizeof(E) == 2)
    if (min(a.Lk, a.R) <= FINE) return launch_dkv<E, DP, true>(a, packed, grid, st);
  return launch_dkv<E, DP, false>(a, packed, grid, st);
}

template <typename E>
static int run_bwd(Args& a, const Plan& pq, const Plan& pkv, float* part_q, float* part_kv, hipStream_t st) {
  const int dp = padded(a.D);
  const int64_t nq = (int64_t)a.B * a.Lq * a.H * a.D, nkv = (int64_t)a.B * a.Lk * a.Hk * a.D;
  Sums t = {};
  int rc = 0;
  if (a.Lq > 0) {
    const Plan& p = pq;
    const int64_t grid = (int64_t)a.B * a.Hk * p.nsplit * p.nblk;
    NEOSR_CHECK(grid <= MAX_GRID, "neosr_attention_bwd: %lld workgroups", (long long)grid);
    a.nblk = p.nblk;
    a.nsplit = p.nsplit;
    a.part = part_q;
    rc = dp == 32 ? launch_dq<E, 32>(a, p.packed, (unsigned)grid, st)
                  : (dp == 64 ? launch_dq<E, 64>(a, p.packed, (unsigned)grid, st) : launch_dq<E, 128>(a, p.packed, (unsigned)grid, st));
    if (rc) return rc;
    if (p.nsplit > 1) {
      t.part[0] = part_q;
      t.out[0] = a.dq;
      t.n[0] = t.stride[0] = nq;
      t.nsplit[0] = p.nsplit;
      t.count = 1;
    }
  }
  if (a.Lk > 0) {
    const Plan& p = pkv;
    const int64_t grid = (int64_t)a.B * a.Hk * p.nsplit * p.nblk;
    NEOSR_CHECK(grid <= MAX_GRID, "neosr_attention_bwd: %lld workgroups", (long long)grid);
    a.nblk = p.nblk;
    a.nsplit = p.nsplit;
    a.part = part_kv;
    rc = dp == 32 ? launch_dkv<E, 32>(a, p.packed, (unsigned)grid, st)
                  : (dp == 64 ? launch_dkv<E, 64>(a, p.packed, (unsigned)grid, st) : launch_dkv<E, 128>(a, p.packed, (unsigned)grid, st));
    if (rc) return rc;
    if (p.nsplit > 1)
      for (int i = 0; i < 2; ++i) {
        t.part[t.count] = part_kv + i * nkv;
        t.out[t.count] = i ? a.dv : a.dk;
        t.n[t.count] = nkv;
        t.stride[t.count] = 2 * nkv;
        t.nsplit[t.count++] = p.nsplit;
      }
  }
  if (t.count) {
    int64_t n = 0;
    for (int i = 0; i < t.count; ++i) n = t.n[i] > n ? t.n[i] : n;
    NEOSR_CHECK((n + 255) / 256 <= MAX_GRID, "neosr_attention_bwd: %lld output elements", (long long)n);
    sum_splits_kernel<E><<<dim3((unsigned)((n + 255) / 256), t.count), 256, 0, st>>>(t);
    NEOSR_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace attn

using namespace attn;

extern "C" int64_t neosr_attention_bwd_workspace_bytes(const neosr_attention_desc* d) {
  if (check(d, true, "neosr_attention_bwd_workspace_bytes")) return -1;
  return bwd_space(d, plan_dq(d), plan_dkv(d)).total();
}

extern "C" int neosr_attention_bwd(const neosr_attention_desc* d, void* stream) {
  if (check(d, true, "neosr_attention_bwd")) return 1;
  if (d->B == 0 || (d->Lq == 0 && d->Lk == 0)) return 0;
  const Plan pq = plan_dq(d), pkv = plan_dkv(d);
  const BwdSpace s = bwd_space(d, pq, pkv);
  const int64_t need = s.total();
  NEOSR_CHECK(need <= d->workspace_bytes && (need == 0 || (d->workspace && (uintptr_t)d->workspace % 256 == 0)),
              "neosr_attention_bwd: workspace of %lld bytes, %lld needed (256-byte aligned)", (long long)d->workspace_bytes, (long long)need);
  Args a;
  fill(d, a);
  char* ws = (char*)d->workspace;
  a.delta = (float*)ws;
  float *part_q = (float*)(ws + s.delta), *part_kv = (float*)(ws + s.delta + s.part_q);
  a.kv_img = ws + s.delta + s.part_q + s.part_kv;
  a.words = (unsigned long long*)(a.kv_img + s.kv);
  a.row_img = a.kv_img + s.kv + s.words;
  const bool prof = neosr_prof_on();
  if (prof) {
    const double esz = d->dtype == NEOSR_DT_F32 ? 4 : 2, qo = (double)d->B * d->Lq * d->H * d->D, kv = (double)d->B * d->Lk * d->Hk * d->D;
    neosr_prof_begin(NEOSR_PROF_ATTN_BWD, stream, 10.0 * d->B * d->H * (double)d->Lq * d->Lk * d->D, esz * 4 * (qo + kv));
  }
  int rc = pack(d, a, pq.packed && d->Lq > 0, true, (hipStream_t)stream);
  if (!rc) rc = d->dtype == NEOSR_DT_F32 ? run_bwd<float>(a, pq, pkv, part_q, part_kv, (hipStream_t)stream)
                                         : run_bwd<__bf16>(a, pq, pkv, part_q, part_kv, (hipStream_t)stream);
  if (prof) neosr_prof_end(stream);
  return rc;
}
