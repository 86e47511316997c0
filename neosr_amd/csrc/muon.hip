// muon.hip — one optimizer step over a flat parameter arena: matrices get orthogonalised momentum (newton_schulz.hip), every
// other parameter AdamW; clip, decoupled decay and the EMA shadow ride in the same sweeps as in the other fused optimizers.
//   matrices: m <- m + (1 - mu)(g - m),  u = nesterov ? g + mu (m - g) : m,  p <- (1 - lr wd) p - lr s NS(u)
//   others:   AdamW with beta1, beta2, eps
// Two element-wise sweeps around the Newton-Schulz launches: bound by HBM (matrices: read p, g, m, u, write m, u, p).
// A step of swinir_medium (11.9 M parameters, gradients in their arena) takes 833-844 us, 560 of them the Newton-Schulz products, 40
// and 31 the two sweeps; AdamW's 249-259, all of it the host's (its kernel: 54).  esrgan (16.7 M): 994-1002 against 342.
// A workgroup takes one chunk of at most 4096 elements of ONE parameter, so what kind of update an element gets is uniform.
#include "common.h"
#include "../../include/neosr_amd.h"

namespace {

__device__ __forceinline__ void muon_ema(float* ema, int64_t i, float p, float decay) {
  if (!ema) return;
  ema[i] = decay < 0.f ? p : ema[i] + (p - ema[i]) * (1.f - decay);
}

__global__ __launch_bounds__(256) void muon_moments_kernel(const neosr_muon_desc d) {
  const int32_t* c = d.chunks + 4 * (int64_t)blockIdx.x;
  const int64_t at = 4 * (int64_t)c[0];
  const int n = c[1], matrix = c[2];
  float clip = d.grad_scale;
  if (d.max_norm > 0.f) clip *= fminf(d.max_norm / (d.norm_ws[0] + 1e-6f), 1.f);
  for (int k = threadIdx.x; k < n; k += 256) {
    const int64_t i = at + k;
    const float g = d.grad[i] * clip;
    float m = d.exp_avg[i];
    if (matrix) {
      m = m + (g - m) * (1.f - d.momentum);
      d.update[i] = d.nesterov ? g + (m - g) * d.momentum : m;
    } else {
      m = m + (g - m) * (1.f - d.beta1);
      const float v = d.exp_avg_sq[i] * d.beta2 + (1.f - d.beta2) * g * g;
      float p = d.param[i] * (1.f - d.lr * d.weight_decay);
      p -= d.lr / d.bias_correction1 * (m / (sqrtf(v) / d.bias_correction2_sqrt + d.eps));
      d.exp_avg_sq[i] = v;
      d.param[i] = p;
      muon_ema(d.ema, i, p, d.ema_decay);
    }
    d.exp_avg[i] = m;
  }
}

__global__ __launch_bounds__(256) void muon_apply_kernel(const neosr_muon_desc d) {
  const int32_t* c = d.chunks + 4 * (int64_t)blockIdx.x;
  const int64_t at = 4 * (int64_t)c[0];
  const int n = c[1];
  const float step = d.lr * __int_as_float(c[3]), keep = 1.f - d.lr * d.weight_decay;
  for (int k = threadIdx.x; k < n; k += 256) {
    const int64_t i = at + k;
    const float p = d.param[i] * keep - step * d.update[i];
    d.param[i] = p;
    muon_ema(d.ema, i, p, d.ema_decay);
  }
}

}  // namespace

extern "C" int neosr_muon_step(const neosr_muon_desc* dp, void* stream) {
  NEOSR_CHECK(dp, "muon_step: null descriptor");
  const neosr_muon_desc& d = *dp;
  NEOSR_CHECK(d.param && d.grad && d.exp_avg && d.exp_avg_sq && d.chunks && d.n > 0, "muon_step: bad args");
  NEOSR_CHECK(d.nchunks > 0 && d.nmatrix >= 0 && d.nmatrix <= d.nchunks && (d.nmatrix == 0) == (d.nitems == 0),
              "muon_step: %d chunks, %d of matrices, %d matrices", d.nchunks, d.nmatrix, d.nitems);
  NEOSR_CHECK(d.nitems == 0 || (d.items && d.update && d.coefficients), "muon_step: matrices need items, update and coefficients");
  if (d.nitems > 0) {   // (before anything is written)
    const int64_t need = neosr_newton_schulz_workspace_bytes(d.items, d.nitems, NEOSR_DT_F32);
    if (need < 0) return 1;
    NEOSR_CHECK(d.ns_steps >= 1 && d.ns_steps <= 64 && d.ns_eps >= 0.f, "muon_step: %d steps", d.ns_steps);
    NEOSR_CHECK(d.workspace && (uintptr_t)d.workspace % 16 == 0 && d.workspace_bytes >= need,
                "muon_step: workspace of %lld bytes, %lld needed (16-byte aligned)", (long long)d.workspace_bytes, (long long)need);
  }
  hipStream_t st = (hipStream_t)stream;
  if (d.max_norm > 0.f) {
    NEOSR_CHECK(d.norm_ws, "muon_step: clipping needs norm_ws");
    if (int rc = neosr_grad_norm(d.grad, d.n, d.grad_scale, d.norm_ws, stream)) return rc;
  }
  muon_moments_kernel<<<d.nchunks, 256, 0, st>>>(d);
  NEOSR_LAUNCH_CHECK();
  if (d.nitems == 0) return 0;
  if (int rc = neosr_newton_schulz(d.items, d.nitems, NEOSR_DT_F32, d.ns_steps, d.coefficients, d.ns_eps, d.workspace, d.workspace_bytes,
                                   stream))
    return rc;
  muon_apply_kernel<<<d.nmatrix, 256, 0, st>>>(d);
  NEOSR_LAUNCH_CHECK();
  return 0;
}
