// attention_fwd.hip — O = softmax(scale Q K^T) V over keys that are allowed, one pass over the keys with the running maximum
// and sum of the softmax (any lengths, head sizes to 128, shared key heads, key masks, causal order).
//
// A (batch, key head) has R = Lq * G rows, r = position * G + group: shared heads become more rows of the same problem, so K
// and V tiles are staged once for the whole group.  A wave owns 32 rows as accumulator COLUMNS
// (attention.h; 64 rows in bf16 were 7 % slower: two waves per SIMD instead of four to run one's vector work under another's
// MFMAs); NW waves share the staged tile of 64 or 32 keys, whose successor is in flight meanwhile.
//
// Bound by the vector pipe beside the matrix pipe: 5 issue slots a score for the softmax (its exponential 2), 5.5 more for the
// three pieces of an fp32 P.  Measured: 16384 tokens of 6 x 30 fp32 1.08-1.11 ms (174-180 TFLOP/s, what six-term products reach
// at a library matmul's rate); 4 x 4096 of 8 / 2 heads x 64 bf16 184-204 us (675-750 TFLOP/s; vector 69 %, matrix 36 % of the cycles).
#include <math.h>
#include "attention.h"
#include "prof.h"

namespace attn {

// PACKED: tiles come from the packed image by LDS-DMA, one in flight behind the one in use; else the workgroup stages them
// itself, through registers.
// PAD (fp32, D < DP): the packed V holds 1 in its first padding channel, so that channel of O is the row sum of P, for no
// instruction (an add for each score otherwise, a tenth of the vector work: 1114 us against 1076 for 16384 tokens of 6 x 30).  In
// bf16 it would be the sum of the rounded P, which over few keys is a poorer statistic for the backward pass.
template <typename E, int DP, int NW, bool PACKED, bool PAD, int OCC>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(OCC))) void fwd_kernel(const Args a) {
  constexpr int NP = Pieces<E>::n, KT = tile_rows<NP, DP>(), NC = DP / 16, ND = DP / 32, UPR = DP / 8;
  constexpr int UNITS = PACKED ? 1 : KT * UPR / (64 * NW);
  typedef Tile<NP, DP, KT> T;
  __shared__ __attribute__((aligned(1024))) short lds[(PACKED ? 2 : 1) * 2 * T::ELEMS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;

  int64_t w = xcd_order(blockIdx.x, gridDim.x);
  const int rb = a.causal ? a.nblk - 1 - (int)(w % a.nblk) : (int)(w % a.nblk);   // causal: the long rows first
  w /= a.nblk;
  const int split = (int)(w % a.nsplit);
  const int bh = (int)(w / a.nsplit), b = bh / a.Hk, hk = bh % a.Hk;

  const int blk0 = rb * 32 * NW;
  const int wr0 = blk0 + wave * 32;                 // the wave's first row
  const int last = a.causal ? min(a.Lk, (min(a.R, blk0 + 32 * NW) - 1) / a.G + a.off + 1) : a.Lk;
  const Range keys = share(0, last, split, a.nsplit);
  const int kbeg = keys.beg, kend = keys.end;

  // PACKED: the first tile is on its way while the rows are read
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

  // the wave's rows as B operands
  const int r = wr0 + (lane & 31);
  const int pos = r / a.G, g = r - pos * a.G;
  const int lim = a.causal ? pos + a.off : 0x7fffffff;   // last key the row may see
  bf16x8 Q[NC][NP];
  {
    const E* row = reinterpret_cast<const E*>(a.q.p) + b * a.q.sb + pos * a.q.sl + (int64_t)(hk * a.G + g) * a.q.sh;
    Raw8<E> x[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      zero(x[c]);
      if (r < a.R) x[c] = load8(row, 16 * c + 8 * half, a.D, a.vec);
    }
    operands(x, Q);
  }

  // O + Ol.  128-wide heads go without: single waves have no registers left for it, and their error is below the fp32 form's as it
  // is (8192 keys: 1.1e-6 of the output's norm, elementary fp32 operations 1.7e-6).
  constexpr bool LO = NP == 3 && DP <= 64;
  f32x16 O[ND], Ol[LO ? ND : 1];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) O[n][i] = 0.f;
  if constexpr (LO)
#pragma unroll
    for (int n = 0; n < ND; ++n) Ol[n] = O[n];

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
      __syncthreads();                                   // the tile is there, for all waves; the other buffer is read
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
        if (!ok[u]) {                                    // masked keys are never part of a product, whatever they hold
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

    // the whole tile's scores first: one maximum, one rescaling test for 64 keys, and independent MFMA chains
    constexpr int KB = KT / 32;
    f32x16 S[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) S[kb][i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      bf16x8 A[KB][NP];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) T::rows(kt, 32 * kb, c, lane, A[kb]);
      if constexpr (KB == 2 && NP == 3) {
        mac2(A[0], A[1], Q[c], S[0], S[1]);
      } else {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) S[kb] = mac(A[kb], Q[c], S[kb]);
      }
    }
    // masks: only tiles that hold a masked key or cross some row's limit
    if (!__all(lim - k0 >= KT - 1) || valid != (KT == 64 ? ~0ull : 0xffffffffull)) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        unsigned bits = (unsigned)(valid >> (32 * kb)) >> (4 * half);
        const int rel = lim - (k0 + 32 * kb) - 4 * half;     // index of the last allowed key in the lane's numbering
        if (rel < 28) bits &= rel < 0 ? 0u : (2u << rel) - 1u;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(bits >> acc_row(i) & 1u)) S[kb][i] = -INFINITY;
      }
    }
    float mx = S[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, S[kb][i]);
    mx = pair_max(mx) * a.cs;
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.f : mn;
    if (!__all(mn == m)) {
      const float al = __builtin_amdgcn_exp2f(m - ref);
      l *= al;
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          O[n][i] *= al;
          if constexpr (LO) Ol[n][i] *= al;
        }
      m = mn;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        S[kb][i] = __builtin_amdgcn_exp2f(fmaf(S[kb][i], a.cs, -ref));
        if constexpr (!PAD) l += S[kb][i];
      }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        bf16x8 P[NP];
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = S[kb][8 * c + e];
        pieces_of(x, P);
#pragma unroll
        for (int n = 0; n < ND; ++n) {
          bf16x8 A[NP];
          T::cols(vt, 32 * kb + 16 * c, 32 * n, lane, A);
          if constexpr (LO) mac_lo(A, P, Ol[n], O[n]);
          else O[n] = mac(A, P, O[n]);
        }
      }
  }

  if constexpr (PAD) {
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (32 * n + acc_row(i) + 4 * half == a.D) l = LO ? O[n][i] + Ol[LO ? n : 0][i] : O[n][i];
  }
  const float sum = pair_sum(l);
  if (r >= a.R) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const float lse = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
  const int64_t row = (int64_t)bh * a.R + r, prow = (int64_t)split * a.B * a.Hk * a.R + row;
  if (half == 0) {
    if (a.nsplit > 1) a.part_lse[prow] = lse;
    else if (a.lse) a.lse[row] = sum == 0.f ? INFINITY : lse;
  }
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[4];
      const int d = 32 * n + 8 * j + 4 * half;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (LO ? O[n][4 * j + e] + Ol[LO ? n : 0][4 * j + e] : O[n][4 * j + e]) * inv;
      if (a.nsplit > 1) store4(a.part + prow * a.D, d, a.D, x);
      else store_out<E>(a, (((int64_t)b * a.Lq + pos) * a.H + hk * a.G + g) * a.D, d, x);
    }
}

// joins the splits of the keys: weights 2^(lse_s - lse), fixed order.  One workgroup per 256 output elements.
template <typename E>
__global__ __launch_bounds__(256) void fwd_join_kernel(const Args a) {
  const int64_t rows = (int64_t)a.B * a.Hk * a.R;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= rows * a.D) return;
  const int64_t row = idx / a.D;
  const int d = (int)(idx - row * a.D);
  float m = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) m = fmaxf(m, a.part_lse[s * rows + row]);
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f, acc = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.nsplit; ++s) {       // (a split without a key: weight 0, output 0)
    const float wgt = __builtin_amdgcn_exp2f(a.part_lse[s * rows + row] - ref);
    sum += wgt;
    acc = fmaf(wgt, a.part[(s * rows + row) * a.D + d], acc);
  }
  const int bh = (int)(row / a.R), r = (int)(row % a.R), pos = r / a.G, g = r - pos * a.G;
  const int b = bh / a.Hk, hk = bh % a.Hk;
  const int64_t to = (((int64_t)b * a.Lq + pos) * a.H + hk * a.G + g) * a.D + d;
  const float o = sum == 0.f ? 0.f : acc / sum;
  reinterpret_cast<E*>(a.out)[to] = (E)o;
  if constexpr (sizeof(E) == 2)
    if (a.rest) reinterpret_cast<E*>(a.rest)[to] = (E)(o - (float)(E)o);
  if (d == 0 && a.lse) a.lse[row] = sum == 0.f ? INFINITY : m + __builtin_amdgcn_logf(sum);
}

// ---- host ------------------------------------------------------------------------------------------------------------------
int check(const neosr_attention_desc* d, bool bwd, const char* who) {
  NEOSR_CHECK(d, "%s: null descriptor", who);
  NEOSR_CHECK(d->dtype == NEOSR_DT_F32 || d->dtype == NEOSR_DT_BF16, "%s: dtype %d", who, d->dtype);
  NEOSR_CHECK(d->B >= 0 && d->Lq >= 0 && d->Lk >= 0 && d->H > 0 && d->Hk > 0 && d->H % d->Hk == 0,
              "%s: B %d Lq %d Lk %d H %d Hk %d (H a multiple of Hk)", who, d->B, d->Lq, d->Lk, d->H, d->Hk);
  NEOSR_CHECK(d->D >= 1 && d->D <= 128, "%s: head size %d (1 to 128)", who, d->D);
  NEOSR_CHECK(d->scale >= 1e-30f && d->scale <= 1e30f, "%s: scale must be positive (1e-30 to 1e30)", who);
  NEOSR_CHECK(d->H <= 65535 && (int64_t)d->Lq * (d->H / d->Hk) <= 0x3f000000 && (int64_t)d->Lk * (d->H / d->Hk) <= 0x3f000000 &&
                  (int64_t)d->B * d->Hk <= 0x7fffffff,
              "%s: Lq %d Lk %d H %d too large (row and key indices of a shared head are 32-bit)", who, d->Lq, d->Lk, d->H);
  const bool rows = d->B > 0 && d->Lq > 0, keys = d->B > 0 && d->Lk > 0;
  NEOSR_CHECK(!rows || (d->q && (bwd ? (d->dout && d->dq && d->lse && d->out) : d->out != nullptr)), "%s: null pointer (rows)", who);
  NEOSR_CHECK(!keys || (d->k && d->v && (!bwd || (d->dk && d->dv))), "%s: null pointer (keys)", who);
  const int64_t esz = d->dtype == NEOSR_DT_F32 ? 4 : 2;
  const void* ptrs[] = {d->q, d->k, d->v, d->out, d->out_rest, d->dout, d->dq, d->dk, d->dv};
  for (const void* p : ptrs) NEOSR_CHECK((uintptr_t)p % esz == 0, "%s: pointer not aligned to its element", who);
  NEOSR_CHECK(((uintptr_t)d->out | (uintptr_t)d->out_rest | (uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv) % 16 == 0,
              "%s: dense outputs must be 16-byte aligned", who);
  return 0;
}

void fill(const neosr_attention_desc* d, Args& a) {
  a = Args{};
  a.q = {(const char*)d->q, d->q_sb, d->q_sl, d->q_sh};
  a.k = {(const char*)d->k, d->k_sb, d->k_sl, d->k_sh};
  a.v = {(const char*)d->v, d->v_sb, d->v_sl, d->v_sh};
  a.dout = {(const char*)d->dout, d->do_sb, d->do_sl, d->do_sh};
  a.o = {(const char*)d->out, (int64_t)d->Lq * d->H * d->D, (int64_t)d->H * d->D, d->D};
  a.out = (char*)d->out;
  a.rest = d->dtype == NEOSR_DT_BF16 ? (char*)d->out_rest : nullptr;
  a.dq = (char*)d->dq;
  a.dk = (char*)d->dk;
  a.dv = (char*)d->dv;
  a.lse = d->lse;
  a.mask = d->key_mask;
  a.mask_sb = d->mask_sb;
  a.mask_sl = d->mask_sl;
  a.B = d->B;
  a.Lq = d->Lq;
  a.Lk = d->Lk;
  a.H = d->H;
  a.Hk = d->Hk;
  a.G = d->H / d->Hk;
  a.D = d->D;
  a.R = d->Lq * a.G;
  const int kt = tile_rows_of(d->dtype, d->D);
  a.kv_tiles = (d->Lk + kt - 1) / kt;
  a.row_tiles = (a.R + kt - 1) / kt;
  a.causal = d->causal;
  a.off = d->Lk - d->Lq;
  a.scale = d->scale;
  a.cs = (float)((double)d->scale * 1.4426950408889634);
  const int esz = d->dtype == NEOSR_DT_F32 ? 4 : 2;
  uint64_t low = 16 | (uint64_t)d->D * esz;
  auto add = [&](const Tensor4& t) {
    if (!t.p) return;
    low |= (uint64_t)(uintptr_t)t.p | (uint64_t)(t.sb * esz) | (uint64_t)(t.sl * esz) | (uint64_t)(t.sh * esz);
  };
  add(a.q);
  add(a.k);
  add(a.v);
  add(a.dout);
  if (d->dout) add(a.o);
  const int al = (int)(low & (~low + 1));
  a.vec = al == 16 ? 2 : (al >= 2 * esz ? 1 : 0);
}

// Four waves of 32 outer indices share every staged tile; they are taken when there are more outer indices than half of such a
// block, and the inner index is split (at least 2 tiles each, joined afterwards) until there are two workgroups for each CU.
// Few outer indices, or a chip that would stay half empty even so: single waves, split likewise, up to eight for each CU
// (what LDS holds of them at a time: 3 to 8, of dK and dV's 3 in fp32, 4 in 64-wide bf16, 2 and 1 with 128-wide heads; the rest
// follow) — unless
// the head size is odd: rows then allow no access wider than an element, and the packing pass has the whole chip for those
// (11 x 19 queries, 4439 keys, 8 / 4 heads x 65 bf16: 87 us against 266 in single waves, which load their own tiles; one query of
// 6 x 31 over 4096 keys: 40 against 35).
Plan plan(int64_t bh, int64_t outer, int64_t inner, int D) {
  const int64_t tiles = (inner + 63) / 64;
  auto splits = [&](int64_t blocks, int64_t goal, int64_t most) {
    int64_t n = blocks >= goal ? 1 : (goal + blocks - 1) / (blocks > 0 ? blocks : 1);
    if (n > most) n = most;
    if (n > 64) n = 64;
    return n > 0 ? n : 1;
  };
  Plan p = {};
  const int64_t wide = bh * ((outer + 127) / 128);
  int64_t want = splits(wide, 512, tiles / 2);
  p.packed = outer > (D % 2 ? 16 : 64) && wide * want >= 128;
  const int block = p.packed ? 128 : 32;
  p.nblk = (int)((outer + block - 1) / block);
  if (!p.packed) want = splits(bh * p.nblk, 2048, tiles / 2);
  const int64_t per = (tiles + want - 1) / want;
  p.nsplit = per > 0 ? (int)((tiles + per - 1) / per) : 1;
  return p;
}

static Plan plan_fwd(const neosr_attention_desc* d) {
  return plan((int64_t)d->B * d->Hk, (int64_t)d->Lq * (d->H / d->Hk), d->Lk, d->D);
}

// OCC: the waves per SIMD the registers are held to
template <typename E, int DP>
static int launch_fwd(const Args& a, bool packed, unsigned grid, hipStream_t st) {
  constexpr bool F32 = sizeof(E) == 4;
  constexpr int OCC = F32 && DP == 128 ? 1 : 2;
  if constexpr (F32)
    if (packed && a.D < DP) {
      fwd_kernel<E, DP, 4, true, true, OCC><<<grid, 256, 0, st>>>(a);
      NEOSR_LAUNCH_CHECK();
      return 0;
    }
  if (packed) fwd_kernel<E, DP, 4, true, false, OCC><<<grid, 256, 0, st>>>(a);
  else fwd_kernel<E, DP, 1, false, false, DP == 128 ? 1 : 2><<<grid, 64, 0, st>>>(a);
  NEOSR_LAUNCH_CHECK();
  return 0;
}

template <typename E>
static int run_fwd(Args& a, const Plan& p, hipStream_t st) {
  const int64_t grid = (int64_t)a.B * a.Hk * p.nsplit * p.nblk;
  NEOSR_CHECK(grid <= MAX_GRID, "neosr_attention_fwd: %lld workgroups", (long long)grid);
  int rc;
  if (a.D <= 32) rc = launch_fwd<E, 32>(a, p.packed, (unsigned)grid, st);
  else if (a.D <= 64) rc = launch_fwd<E, 64>(a, p.packed, (unsigned)grid, st);
  else rc = launch_fwd<E, 128>(a, p.packed, (unsigned)grid, st);
  if (rc) return rc;
  if (p.nsplit > 1) {
    const int64_t n = (int64_t)a.B * a.Hk * a.R * a.D;
    NEOSR_CHECK((n + 255) / 256 <= MAX_GRID, "neosr_attention_fwd: %lld output elements", (long long)n);
    fwd_join_kernel<E><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
    NEOSR_LAUNCH_CHECK();
  }
  return 0;
}

// row statistics and outputs of the splits | packed K, V | truth words
struct FwdSpace { int64_t lse, part, img, words; };
static FwdSpace fwd_space(const neosr_attention_desc* d, const Plan& p) {
  FwdSpace s = {};
  if (p.nsplit > 1) {
    const int64_t rows = (int64_t)p.nsplit * d->B * d->H * d->Lq;
    s.lse = align256(rows * 4);
    s.part = align256(rows * d->D * 4);
  }
  if (p.packed) {
    s.img = align256((int64_t)d->B * d->Hk * image_bytes(d->dtype, d->D, d->Lk));
    s.words = words_bytes(d);
  }
  return s;
}

}  // namespace attn

using namespace attn;

extern "C" int64_t neosr_attention_fwd_workspace_bytes(const neosr_attention_desc* d) {
  if (check(d, false, "neosr_attention_fwd_workspace_bytes")) return -1;
  const FwdSpace s = fwd_space(d, plan_fwd(d));
  return s.lse + s.part + s.img + s.words;
}

extern "C" int neosr_attention_fwd(const neosr_attention_desc* d, void* stream) {
  if (check(d, false, "neosr_attention_fwd")) return 1;
  if (d->B == 0 || d->Lq == 0) return 0;
  const Plan p = plan_fwd(d);
  const FwdSpace s = fwd_space(d, p);
  const int64_t need = s.lse + s.part + s.img + s.words;
  NEOSR_CHECK(need <= d->workspace_bytes && (need == 0 || (d->workspace && (uintptr_t)d->workspace % 256 == 0)),
              "neosr_attention_fwd: workspace of %lld bytes, %lld needed (256-byte aligned)", (long long)d->workspace_bytes, (long long)need);
  Args a;
  fill(d, a);
  a.nblk = p.nblk;
  a.nsplit = p.nsplit;
  char* ws = (char*)d->workspace;
  a.part_lse = (float*)ws;
  a.part = (float*)(ws + s.lse);
  a.kv_img = ws + s.lse + s.part;
  a.words = (unsigned long long*)(ws + s.lse + s.part + s.img);
  const bool prof = neosr_prof_on();
  if (prof) {
    const double esz = d->dtype == NEOSR_DT_F32 ? 4 : 2, qo = (double)d->B * d->Lq * d->H * d->D, kv = (double)d->B * d->Lk * d->Hk * d->D;
    neosr_prof_begin(NEOSR_PROF_ATTN_FWD, stream, 4.0 * d->B * d->H * (double)d->Lq * d->Lk * d->D, esz * 2 * (qo + kv));
  }
  int rc = pack(d, a, p.packed, false, (hipStream_t)stream);
  if (!rc) rc = d->dtype == NEOSR_DT_F32 ? run_fwd<float>(a, p, (hipStream_t)stream) : run_fwd<__bf16>(a, p, (hipStream_t)stream);
  if (prof) neosr_prof_end(stream);
  return rc;
}
