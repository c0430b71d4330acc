// Forward of the norms around a residual block: y = x + a * scale * act(gate) * N(branch), h = N(y), one pass over x, branch and gate.
#include "fnet_block_norm.h"

namespace {

// One row: load, (mean,) sum of squares about it, the residual sum, and the same for the norm of y, all from registers; y enters the second
// norm before it is rounded.  The variance is the mean square about the mean, not E[v^2] - mean^2, which loses everything for rows far from
// zero.  Rows are dealt to blocks in turn; weights and scale are loaded once per block.
template <typename T, int L, int E>
__global__ __launch_bounds__((RowShape<T, L, E>::THREADS)) void k_block_norm_fwd(FnetBlockNorm a) {
    using S = RowShape<T, L, E>;
    constexpr int V = S::V, K = S::K;
    __shared__ float red[2 * RowSum<L, 1>::W];
    RowSum<L, 1> sum(red);
    const int C = a.width, lane = threadIdx.x % L;
    const bool pf = a.param_dtype == FNET_F32, gf = a.gate_dtype == FNET_F32, layer = a.kind == FNET_NORM_LAYER;
    const float inv_c = 1.f / (float)C;
    const bool have_branch = a.branch != 0, post = a.post != 0, pre = a.h != 0;

    int left[K];                                     // elements of each of this lane's chunks
    float wpost[K][V], wpre[K][V], sc[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * L + lane) * V;
        left[k] = min(max(C - c, 0), V);
#pragma unroll
        for (int i = 0; i < V; ++i) { wpost[k][i] = 1.f; wpre[k][i] = 1.f; sc[k][i] = a.residual_scale; }
        if (left[k] > 0) {
            if (a.post_weight) load_param<T>(a.post_weight, c, pf, left[k], wpost[k]);
            if (a.pre_weight) load_param<T>(a.pre_weight, c, pf, left[k], wpre[k]);
            if (a.scale) {
                load_param<T>(a.scale, c, pf, left[k], sc[k]);
#pragma unroll
                for (int i = 0; i < V; ++i) sc[k][i] *= a.residual_scale;
            }
        }
    }

    for (long long row = (long long)blockIdx.x * S::RPB + threadIdx.x / L; row < a.rows; row += (long long)gridDim.x * S::RPB) {
        float y[K][V], o[K][V];
        const T* px = gptr<const T>(a.x) + row * a.x_stride;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * L + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) { y[k][i] = 0.f; o[k][i] = 0.f; }
            if (left[k] > 0) {
                load_chunk<T>(px + c, left[k], y[k]);
                if (have_branch) load_chunk<T>(gptr<const T>(a.branch) + row * a.branch_stride + c, left[k], o[k]);
            }
        }
        float v1[1];
        auto statistics = [&](float (&v)[K][V], float& mu, float& r) {
            mu = 0.f;
            if (layer) {
                v1[0] = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) v1[0] += i < left[k] ? v[k][i] : 0.f;   // behind the row lies the norm of zeros
                sum(v1);
                mu = v1[0] * inv_c;
            }
            v1[0] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = i < left[k] ? v[k][i] - mu : 0.f;
                    v1[0] = fmaf(d, d, v1[0]);
                }
            sum(v1);
            r = 1.f / sqrtf(v1[0] * inv_c + a.eps);
        };
        if (have_branch) {
            if (post) {
                float mu, r;
                statistics(o, mu, r);
                if (a.stats && lane == 0) {
                    gptr<float>(a.stats)[row] = mu;
                    gptr<float>(a.stats)[a.rows + row] = r;
                }
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int i = 0; i < V; ++i) o[k][i] = (o[k][i] - mu) * r * wpost[k][i];
                    if (a.post_bias && left[k] > 0) {
                        float b[V];
                        load_param<T>(a.post_bias, (k * L + lane) * V, pf, left[k], b);
#pragma unroll
                        for (int i = 0; i < V; ++i) o[k][i] += b[i];
                    }
                }
            }
            if (a.gate_kind == FNET_GATE_TOKEN) {
                const float g = gate_value(load_param1<T>(a.gate, row * a.gate_stride, gf), a.gate_act);
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) o[k][i] *= g;
            } else if (a.gate_kind != FNET_GATE_NONE) {
                const long long at = a.gate_kind == FNET_GATE_ELEMENT ? row * a.gate_stride
                                     : a.gate_kind == FNET_GATE_SAMPLE ? (long long)((uint32_t)row / (uint32_t)a.tokens) * a.gate_stride : 0;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (left[k] <= 0) continue;
                    float g[V];
                    load_param<T>(a.gate, at + (k * L + lane) * V, gf, left[k], g);
#pragma unroll
                    for (int i = 0; i < V; ++i) o[k][i] *= gate_value(g[i], a.gate_act);
                }
            }
            T* py = gptr<T>(a.y) + row * (long long)C;
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) y[k][i] = fmaf(sc[k][i], o[k][i], y[k][i]);
                if (left[k] > 0) store_chunk<T>(py + (k * L + lane) * V, left[k], y[k]);
            }
        }
        if (pre) {
            float mu, r;
            statistics(y, mu, r);
            if (a.stats && lane == 0) {
                gptr<float>(a.stats)[2 * a.rows + row] = mu;
                gptr<float>(a.stats)[3 * a.rows + row] = r;
            }
            T* ph = gptr<T>(a.h) + row * (long long)C;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (left[k] <= 0) continue;
                float b[V];
#pragma unroll
                for (int i = 0; i < V; ++i) b[i] = 0.f;
                if (a.pre_bias) load_param<T>(a.pre_bias, (k * L + lane) * V, pf, left[k], b);
#pragma unroll
                for (int i = 0; i < V; ++i) b[i] = fmaf((y[k][i] - mu) * r, wpre[k][i], b[i]);
                store_chunk<T>(ph + (k * L + lane) * V, left[k], b);
            }
        }
    }
}

bool type_ok(int d, int operand) { return d == FNET_F32 || d == operand; }
bool aligned(uint64_t p, int dtype) { return p % (dtype == FNET_F32 ? 4 : 2) == 0; }

}  // namespace

int fnet_block_norm_check(const FnetBlockNorm* a) {
    FNET_CHECK_ARG(a && (a->dtype == FNET_F32 || a->dtype == FNET_BF16 || a->dtype == FNET_F16));
    FNET_CHECK_ARG(type_ok(a->param_dtype, a->dtype) && type_ok(a->gate_dtype, a->dtype));
    FNET_CHECK_ARG(a->rows >= 0 && a->rows < (1ll << 31) && a->width >= 1 && a->width <= FNET_BLOCK_NORM_MAX_WIDTH);
    FNET_CHECK_ARG(a->kind == FNET_NORM_RMS || a->kind == FNET_NORM_LAYER);
    FNET_CHECK_ARG(a->eps >= 0.f && a->residual_scale == a->residual_scale);
    FNET_CHECK_ARG(a->gate_kind >= FNET_GATE_NONE && a->gate_kind <= FNET_GATE_CHANNEL && a->gate_act >= FNET_GATE_IDENTITY && a->gate_act <= FNET_GATE_TANH);
    FNET_CHECK_ARG((a->gate_kind != FNET_GATE_NONE) == (a->gate != 0));
    FNET_CHECK_ARG(a->gate_kind != FNET_GATE_SAMPLE || (a->tokens > 0 && a->tokens < (1ll << 31) && a->rows % a->tokens == 0));
    // without a branch there is nothing to gate, scale or normalise after
    FNET_CHECK_ARG(a->branch != 0 || (a->gate == 0 && a->scale == 0 && !a->post));
    FNET_CHECK_ARG(a->post || (a->post_weight == 0 && a->post_bias == 0));
    FNET_CHECK_ARG(a->x_stride >= 0 && a->branch_stride >= 0 && a->gate_stride >= 0 && a->dy_stride >= 0 && a->dh_stride >= 0);
    FNET_CHECK_ARG(aligned(a->x, a->dtype) && aligned(a->branch, a->dtype) && aligned(a->gate, a->gate_dtype) && aligned(a->stats, FNET_F32));
    FNET_CHECK_ARG(aligned(a->scale | a->post_weight | a->post_bias | a->pre_weight | a->pre_bias, a->param_dtype));
    FNET_CHECK_ARG(a->rows == 0 || a->x != 0);
    return FNET_OK;
}

int fnet_block_norm_fwd(const FnetBlockNorm* host_args, void* stream) {
    const int rc = fnet_block_norm_check(host_args);
    if (rc != FNET_OK) return rc;
    const FnetBlockNorm& a = *host_args;
    if (a.rows == 0) return FNET_OK;
    FNET_CHECK_ARG((a.branch != 0) == (a.y != 0) && (a.y != 0 || a.h != 0) && (a.h != 0 || (a.pre_weight == 0 && a.pre_bias == 0)));
    FNET_CHECK_ARG(aligned(a.y | a.h, a.dtype));
    DISPATCH_T3(a.dtype, DISPATCH_ROW(a.width, {
        using S = RowShape<T, L, E>;
        const long long steps = (a.rows + S::RPB - 1) / S::RPB;
        const long long most = 256 * (2048 / S::THREADS);              // what the chip holds at once
        hipLaunchKernelGGL((k_block_norm_fwd<T, L, E>), dim3((unsigned)(steps < most ? steps : most)), dim3(S::THREADS), 0, (hipStream_t)stream, a);
    }));
    FNET_LAUNCH_CHECK();
    return FNET_OK;
}
