// vr_sh_factors.h -- the dense SH gradient row of one Gaussian from its factors, as optim.hip's kernels consume it and
// gradnorm.hip's squares it: one definition, so that the norm is that of exactly the values the optimizer steps with.
#pragma once
#include "vr_host.h"

namespace vr {

constexpr int SHF_ROW_MAX = 48;
struct ShAdamSeg {
    float* p; float* m; float* v;          // Adam mode
    float* out;                            // store mode
    float step_size, inv_bc2_sqrt;
};
struct ShFactorArgs {
    const float* means3D; const float* campos; const float* factors;
    long view_stride;                      // floats between the factor blocks of consecutive views (3 P when packed)
    int P, n_views, deg, M;
    float scale;
    ShAdamSeg dc, rest;                    // rest.p / rest.out == nullptr: `dc` is the whole [P,M,3] tensor
    float one_minus_b1, b2, one_minus_b2, eps;
    const float* norm;                     // clipped Adam: the global gradient norm (NULL: not clipped) and its bound
    float max_norm;
};

// g[3 k + c] = sum_v basis_k(normalize(means[i] - campos[v])) * factors[v][i][c], zeros from (deg+1)^2 on (unscaled)
__device__ __forceinline__ void sh_row_from_factors(const ShFactorArgs& a, int i, float* g)
{
    const int K = (a.deg + 1) * (a.deg + 1);
    const float px = a.means3D[3 * (size_t)i], py = a.means3D[3 * (size_t)i + 1], pz = a.means3D[3 * (size_t)i + 2];
    for (int v = 0; v < a.n_views; ++v) {
        const float* f = a.factors + (size_t)v * a.view_stride + (size_t)i * 3;
        const float f0 = f[0], f1 = f[1], f2v = f[2];
        if (f0 == 0.0f && f1 == 0.0f && f2v == 0.0f) continue;      // not visible in this view (or fully clamped)
        const float d0 = px - a.campos[3 * v], d1 = py - a.campos[3 * v + 1], d2 = pz - a.campos[3 * v + 2];
        const float il = 1.0f / sqrtf(d0 * d0 + d1 * d1 + d2 * d2);
        float bas[16];
        sh_basis(a.deg, d0 * il, d1 * il, d2 * il, bas);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (k < K) {
                g[3 * k + 0] = fmaf(bas[k], f0, g[3 * k + 0]);
                g[3 * k + 1] = fmaf(bas[k], f1, g[3 * k + 1]);
                g[3 * k + 2] = fmaf(bas[k], f2v, g[3 * k + 2]);
            }
        }
    }
}

// (optim.hip) checks the arguments the factor entries share and fills `a` for them; Adam / store segments cleared
int sh_factor_args(ShFactorArgs& a, const float* means3D, int32_t P, const float* campos, const float* factors,
                   int32_t n_views, int64_t view_stride, int32_t sh_degree, int32_t M, float scale);

// The factor a gradient is clipped with: min(1, max_norm / (norm + 1e-6)); a NaN norm stays NaN, an infinite one gives 0
// (both as torch.nn.utils.clip_grad_norm_ does).
__device__ __forceinline__ float clip_factor(float norm, float max_norm)
{
    const float c = max_norm / (norm + 1e-6f);
    return c >= 1.0f ? 1.0f : c;
}

}  // namespace vr
