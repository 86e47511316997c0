// rope.hip — rotary positions with several axes: channel pair j of axis a's section turns by
//   angle = position[a] * theta^(-2 j / section_a),   (x, y) -> (x cos - y sin, x sin + y cos),
// channels behind the last section pass through; the backward pass is the turn by the negative angle.
//
// Bound by HBM: every element is read and written once.  One workgroup takes T tokens of one sample with all heads of q AND
// k, so the angles — the expensive part — are formed once per (token, pair) and shared by H + Hk heads from LDS.  Adjacent pairs
// (interleaved) lie in one vector: those rows go straight through registers.  The pairs of the split layout are section / 2 apart
// (7 floats for swinir's 30-wide heads), so their rows go through LDS and global accesses stay 16 bytes wide over the token's
// contiguous H * D row whatever the section sizes are.
// Measured: 65536 tokens of 10 x 64 bf16 (168 MB) 45 us, 77 % of a large copy's rate; 8 x 4096 tokens of 12 x 30 fp32 (94 MB) in
// the split layout 33 us, 59 %.  What holds that one back is less LDS than its loads: HIP's uint4 is a class, the array of a batch stays
// in scratch (80 bytes a lane in both 16-byte forms, none in the others), and every load is waited for before the next.
// The angle is formed in 64 bits in revolutions and reduced there to an eighth of a turn around a quarter: a position of 10^6
// times a frequency near 1 keeps every bit of the reduced angle, where a 32-bit product would keep none below 0.06 rad.
#include "common.h"
#include "../../include/neosr_amd.h"
#include <math.h>

namespace {

constexpr int ROPE_MAX_PAIRS = 128;
constexpr int ROPE_MAX_D = 256;
constexpr int ROPE_LDS_BYTES = 24576;   // most that the row buffer may take

struct RopeTensor {
  const char* in;
  char* out;
  int64_t sb, sn, sh;   // element strides of `in`
  int heads, hchunk;    // heads staged at a time
};

struct RopeArgs {
  double rev[ROPE_MAX_PAIRS];            // revolutions per unit of position
  unsigned char axis[ROPE_MAX_PAIRS];
  RopeTensor t[2];
  const void* pos;
  int64_t pos_sb, pos_sn, pos_sa;
  int base[4], half[4];                  // first channel and pairs of each section
  int ntensors, naxes, npairs, D, N, T, tiles, pos_kind, interleaved, flat[2];
  int rows_at, chan_at, lds;             // LDS layout in bytes
  float sign;
};

__device__ __forceinline__ float rope_get(const float* p) { return *p; }
__device__ __forceinline__ float rope_get(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void rope_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void rope_put(__bf16* p, float v) { *p = (__bf16)v; }

template <int VB> struct RopeVec;
template <> struct RopeVec<16> { typedef uint4 type; };
template <> struct RopeVec<8> { typedef uint2 type; };
template <> struct RopeVec<4> { typedef unsigned type; };
template <> struct RopeVec<2> { typedef unsigned short type; };

// cos and sin of the tile's tokens
__device__ __forceinline__ void rope_table(const RopeArgs& a, int b, int n0, int nt, float2* table) {
  for (int i = threadIdx.x; i < nt * a.npairs; i += 256) {
    const int t = i / a.npairs, j = i - t * a.npairs;
    const int64_t at = (int64_t)b * a.pos_sb + (int64_t)(n0 + t) * a.pos_sn + (int64_t)a.axis[j] * a.pos_sa;
    double p;
    if (a.pos_kind == NEOSR_POS_F32) p = (double)((const float*)a.pos)[at];
    else if (a.pos_kind == NEOSR_POS_I32) p = (double)((const int32_t*)a.pos)[at];
    else p = (double)((const int64_t*)a.pos)[at];
    const double turn = p * a.rev[j];
    const double quarter = rint(4.0 * turn);
    const float r = (float)(turn - 0.25 * quarter);     // |r| <= 1/8 revolution, exact difference
    const int q = (int)(quarter - 4.0 * floor(0.25 * quarter));
    float s, c;
    sincospif(2.f * r, &s, &c);
    const float cs = (q & 1) ? s : c, sn = (q & 1) ? c : s;
    table[i] = make_float2((q == 1 || q == 2) ? -cs : cs, a.sign * ((q & 2) ? -sn : sn));
  }
}

// VB: bytes of one global access (the largest power of two that divides every row's address and length).  PAIRS: the two
// channels of a pair are neighbours and a vector holds whole pairs.
template <typename E, int VB, bool PAIRS>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs a) {
  typedef typename RopeVec<VB>::type vec_t;
  constexpr int EV = VB / (int)sizeof(E), U = 4;
  // [tokens][pairs] cos, sin | (split layout) rows | partner channel of each channel: as large as the call needs, which for 30-wide
  // heads leaves room for every workgroup a CU can hold
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float2* table = reinterpret_cast<float2*>(smem);
  const int tid = threadIdx.x;
  const int b = blockIdx.x / a.tiles, n0 = (blockIdx.x % a.tiles) * a.T;
  const int nt = min(a.T, a.N - n0);

  if constexpr (PAIRS) {
    bool ready = false;
    for (int w = 0; w < a.ntensors; ++w) {
      const RopeTensor& x = a.t[w];
      const int row = x.heads * a.D, rv = row / EV, n = nt * rv;
      for (int i0 = tid; i0 < n || !ready; i0 += 256 * U) {
        union { vec_t v; E el[EV]; } r[U];
        int tok[U], ch[U], at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {                   // U loads in flight; the first of them pass the table's time
          const int i = i0 + 256 * u;
          if (i < n) {
            tok[u] = i / rv;
            const int e = (i - tok[u] * rv) * EV, h = e / a.D;
            at[u] = e;
            ch[u] = e - h * a.D;
            const E* src = reinterpret_cast<const E*>(x.in) + (int64_t)b * x.sb + (int64_t)(n0 + tok[u]) * x.sn +
                           (a.flat[w] ? (int64_t)e : (int64_t)h * x.sh + ch[u]);
            r[u].v = *reinterpret_cast<const vec_t*>(src);
          }
        }
        if (!ready) {
          rope_table(a, b, n0, nt, table);
          __syncthreads();
          ready = true;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i0 + 256 * u >= n) continue;
          int d = ch[u];
#pragma unroll
          for (int k = 0; k < EV / 2; ++k) {
            if (d < 2 * a.npairs) {
              const float2 cs = table[tok[u] * a.npairs + (d >> 1)];
              const float p = rope_get(&r[u].el[2 * k]), q = rope_get(&r[u].el[2 * k + 1]);
              rope_put(&r[u].el[2 * k], p * cs.x - q * cs.y);
              rope_put(&r[u].el[2 * k + 1], p * cs.y + q * cs.x);
            }
            d += 2;
            if (d == a.D) d = 0;
          }
          E* dst = reinterpret_cast<E*>(x.out) + ((int64_t)b * a.N + n0 + tok[u]) * row + at[u];
          *reinterpret_cast<vec_t*>(dst) = r[u].v;
        }
        if (i0 >= n) break;
      }
    }
  } else {
    E* lds = reinterpret_cast<E*>(smem + a.rows_at);
    int* chan = reinterpret_cast<int*>(smem + a.chan_at);   // partner | pair << 10 | role << 20 (0 pass, 1 first, 2 second)
    for (int d = tid; d < a.D; d += 256) {
      int code = d, pair0 = 0;
      for (int s = 0; s < a.naxes; ++s) {
        const int r = d - a.base[s];
        if (r >= 0 && r < 2 * a.half[s]) {
          const int j = a.interleaved ? r >> 1 : (r < a.half[s] ? r : r - a.half[s]);
          const int second = a.interleaved ? r & 1 : r >= a.half[s];
          const int partner = a.interleaved ? d ^ 1 : (second ? d - a.half[s] : d + a.half[s]);
          code = partner | (pair0 + j) << 10 | (1 + second) << 20;
        }
        pair0 += a.half[s];
      }
      chan[d] = code;
    }
    bool ready = false;
    for (int w = 0; w < a.ntensors; ++w) {
      const RopeTensor& x = a.t[w];
      for (int h0 = 0; h0 < x.heads; h0 += x.hchunk) {
        const int nh = min(x.hchunk, x.heads - h0);
        const int row = nh * a.D;                         // elements of one token's chunk
        const int rv = row / EV, n = nt * rv;             // (row and D are whole vectors on the wide paths)
        if (ready) __syncthreads();                       // the chunk before is read
        for (int i0 = tid; i0 < n; i0 += 256 * U) {
          vec_t r[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int i = i0 + 256 * u;
            if (i < n) {
              const int t = i / rv, e = (i - t * rv) * EV;
              const int h = a.flat[w] ? 0 : e / a.D;      // heads side by side: the row is one run
              r[u] = *reinterpret_cast<const vec_t*>(reinterpret_cast<const E*>(x.in) + (int64_t)b * x.sb + (int64_t)(n0 + t) * x.sn +
                                                     (int64_t)(h0 + h) * x.sh + (e - h * a.D));
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i0 + 256 * u < n) *reinterpret_cast<vec_t*>(lds + (i0 + 256 * u) * EV) = r[u];
        }
        if (!ready) rope_table(a, b, n0, nt, table);
        ready = true;
        __syncthreads();
        for (int i = tid; i < n; i += 256) {
          const int t = i / rv, e = (i - t * rv) * EV;
          int h = e / a.D, d = e - h * a.D;
          const E* src = lds + t * row;
          union { vec_t v; E el[EV]; } out;
          out.v = *reinterpret_cast<const vec_t*>(src + e);
#pragma unroll
          for (int u = 0; u < EV; ++u) {
            const int code = chan[d];
            const float own = rope_get(&out.el[u]);
            float y = own;
            if (code >> 20) {
              const float2 cs = table[t * a.npairs + ((code >> 10) & 1023)];
              const float other = rope_get(src + h * a.D + (code & 1023));
              y = (code >> 20) == 1 ? own * cs.x - other * cs.y : other * cs.y + own * cs.x;
            }
            rope_put(&out.el[u], y);
            if (++d == a.D) { d = 0; ++h; }
          }
          E* dst = reinterpret_cast<E*>(x.out) + (((int64_t)b * a.N + n0 + t) * x.heads + h0) * a.D + e;
          *reinterpret_cast<vec_t*>(dst) = out.v;
        }
      }
    }
  }
}

template <typename E, int VB>
void launch_rope(const RopeArgs& a, unsigned grid, hipStream_t st) {
  if constexpr (VB >= 2 * (int)sizeof(E)) {
    if (a.interleaved && a.D % 2 == 0) {
      rope_kernel<E, VB, true><<<grid, 256, a.rows_at, st>>>(a);
      return;
    }
  }
  rope_kernel<E, VB, false><<<grid, 256, a.lds, st>>>(a);
}

template <typename E>
int run_rope(const RopeArgs& a, int vb, unsigned grid, hipStream_t st) {
  if (vb == 16) launch_rope<E, 16>(a, grid, st);
  else if (vb == 8) launch_rope<E, 8>(a, grid, st);
  else if (vb == 4) launch_rope<E, 4>(a, grid, st);
  else launch_rope<E, (int)sizeof(E)>(a, grid, st);
  NEOSR_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int neosr_axial_rope(const neosr_rope_desc* d, void* stream) {
  NEOSR_CHECK(d && d->q && d->q_out && d->positions, "neosr_axial_rope: null pointer");
  NEOSR_CHECK(!d->k == !d->k_out, "neosr_axial_rope: k and k_out go together");
  NEOSR_CHECK(d->dtype == NEOSR_DT_F32 || d->dtype == NEOSR_DT_BF16, "neosr_axial_rope: dtype %d", d->dtype);
  NEOSR_CHECK(d->pos_kind >= NEOSR_POS_F32 && d->pos_kind <= NEOSR_POS_I64, "neosr_axial_rope: position type %d", d->pos_kind);
  NEOSR_CHECK(d->B >= 0 && d->N >= 0 && d->H > 0 && d->D > 0 && d->D <= ROPE_MAX_D && (!d->k || d->Hk > 0),
              "neosr_axial_rope: B %d N %d H %d Hk %d D %d (D at most %d)", d->B, d->N, d->H, d->Hk, d->D, ROPE_MAX_D);
  NEOSR_CHECK(d->naxes >= 1 && d->naxes <= 4, "neosr_axial_rope: %d axes (1 to 4)", d->naxes);
  NEOSR_CHECK(d->theta > 1.0 && d->theta < HUGE_VAL, "neosr_axial_rope: theta must be above 1");
  RopeArgs a = {};
  int at = 0, pairs = 0;
  for (int s = 0; s < d->naxes; ++s) {
    const int sec = d->sections[s];
    NEOSR_CHECK(sec >= 0 && sec % 2 == 0 && at + sec <= d->D, "neosr_axial_rope: section %d of %d channels does not fit D = %d", s,
                sec, d->D);
    a.base[s] = at;
    a.half[s] = sec / 2;
    for (int j = 0; j < sec / 2; ++j) {
      a.rev[pairs] = pow(d->theta, -2.0 * j / sec) / 6.283185307179586476925286766559;
      a.axis[pairs++] = (unsigned char)s;
    }
    at += sec;
  }
  if (d->B == 0 || d->N == 0) return 0;
  const int esz = d->dtype == NEOSR_DT_F32 ? 4 : 2;
  a.ntensors = d->k ? 2 : 1;
  a.t[0] = {(const char*)d->q, (char*)d->q_out, d->q_sb, d->q_sn, d->q_sh, d->H, 0};
  a.t[1] = {(const char*)d->k, (char*)d->k_out, d->k_sb, d->k_sn, d->k_sh, d->Hk, 0};
  a.pos = d->positions;
  a.pos_sb = d->pos_sb;
  a.pos_sn = d->pos_sn;
  a.pos_sa = d->pos_sa;
  a.naxes = d->naxes;
  a.npairs = pairs;
  a.D = d->D;
  a.N = d->N;
  a.pos_kind = d->pos_kind;
  a.interleaved = d->interleaved;
  a.sign = d->inverse ? -1.f : 1.f;
  // tokens per workgroup: as many as the row buffer holds (16 at most, the table's size), fewer while that leaves the chip
  // short of workgroups
  const int hmax = d->k && d->Hk > d->H ? d->Hk : d->H;
  int T = 16;
  while (T > 1 && ((int64_t)T * hmax * d->D * esz > ROPE_LDS_BYTES || (int64_t)d->B * ((d->N + T - 1) / T) < 1024)) T >>= 1;
  a.T = T;
  a.tiles = (d->N + T - 1) / T;
  uint64_t low = 16;                     // collects every low address / length bit
  for (int w = 0; w < a.ntensors; ++w) {
    RopeTensor& x = a.t[w];
    x.hchunk = ROPE_LDS_BYTES / (T * d->D * esz);
    if (x.hchunk > x.heads) x.hchunk = x.heads;
    a.flat[w] = x.sh == d->D;
    const uint64_t run = (uint64_t)d->D * esz;
    low |= (uint64_t)(uintptr_t)x.in | (uint64_t)(uintptr_t)x.out | (uint64_t)(x.sb * esz) | (uint64_t)(x.sn * esz);
    if (a.flat[w] && x.hchunk == x.heads) low |= run * x.heads;
    else low |= run | (uint64_t)(x.sh * esz);
  }
  const int vb = (int)(low & (~low + 1));
  int rows_bytes = 0;
  for (int w = 0; w < a.ntensors; ++w) {
    const int n = T * a.t[w].hchunk * d->D * esz;
    if (n > rows_bytes) rows_bytes = n;
  }
  a.rows_at = (T * (pairs > 0 ? pairs : 1) * 8 + 15) / 16 * 16;
  a.chan_at = a.rows_at + (rows_bytes + 15) / 16 * 16;
  a.lds = a.chan_at + d->D * 4;
  NEOSR_CHECK(vb >= esz, "neosr_axial_rope: pointer not aligned to its element");
  const int64_t grid = (int64_t)d->B * a.tiles;
  NEOSR_CHECK(grid <= 0xffffffffll / 256,   // a launch holds less than 2^32 threads
              "neosr_axial_rope: %lld workgroups", (long long)grid);
  return esz == 4 ? run_rope<float>(a, vb, (unsigned)grid, (hipStream_t)stream)
                  : run_rope<__bf16>(a, vb, (unsigned)grid, (hipStream_t)stream);
}
