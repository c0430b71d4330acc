// Forward of the norms around a residual block: y = x + a * scale * act(gate) * N(branch), h = N(y), one pass over x, branch and gate.
#include "fnet_block_norm.h"

namespace {

// How the gate enters: constant over the rows (none, per channel: part of the weight in registers), one value per row, or a row of values
enum { GM_CONST = 0, GM_ROW = 1, GM_VECTOR = 2 };

// One row: load, (mean,) sum of squares about it, the residual sum, and the same for the norm of y, all from registers; y enters the second
// norm before it is rounded.  The variance is the mean square about the mean, not E[v^2] - mean^2, which loses everything for rows far from
// zero.  Rows are dealt to blocks in turn; what multiplies a normalised value is loaded once per block.
template <typename T, int L, int E, int GM, bool LAYER>
__global__ __launch_bounds__((RowShape<T, L, E>::MAX_THREADS)) void k_block_norm_fwd(FnetBlockNorm a, RowLaunch rl) {
    using S = RowShape<T, L, E>;
    constexpr int V = S::V, K = S::K;
    __shared__ float red[RowSum<L, 1>::SIZE];
    RowSum<L, 1> sum(red);
    const RowPlace<L> at(rl);
    const int C = a.width;
    const bool pf = a.param_dtype == FNET_F32, gf = a.gate_dtype == FNET_F32;
    const float inv_c = 1.f / (float)C;
    const bool have_branch = a.branch != 0, post = a.post != 0, pre = a.h != 0;

    int col[K], left[K];                             // first element of each of this lane's chunks, and how many of its elements there are
    bool full = true;
    float wo[K][V], wy[K][V];                        // residual_scale * scale * post_weight (* act(gate)), pre_weight
#pragma unroll
    for (int k = 0; k < K; ++k) {
        col[k] = (k * at.lanes + at.lane) * V;
        left[k] = min(max(C - col[k], 0), V);
        full = full && left[k] == V;
        float s[V];
        load_param_or<T, S::TINY>(a.post_weight, col[k], pf, left[k], 1.f, wo[k]);
        load_param_or<T, S::TINY>(a.pre_weight, col[k], pf, left[k], 1.f, wy[k]);
        load_param_or<T, S::TINY>(a.scale, col[k], pf, left[k], 1.f, s);
#pragma unroll
        for (int i = 0; i < V; ++i) wo[k][i] *= a.residual_scale * s[i];
        if (GM == GM_CONST && a.gate) {
            load_param_or<T, S::TINY>(a.gate, col[k], gf, left[k], 1.f, s);
            gate_values<V>(s, a.gate_act);
#pragma unroll
            for (int i = 0; i < V; ++i) wo[k][i] *= s[i];
        }
    }
    full = __all(full);                              // of this wave: no element of its chunks lies behind the row

    // 1 / deviation of a row (and its mean, taken off)
    auto normalise = [&](float (&v)[K][V], float& mu) {
        float s[1];
        mu = 0.f;
        if (LAYER) {
            s[0] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) s[0] += v[k][i];
            sum(s, at);
            mu = s[0] * inv_c;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) v[k][i] -= mu;
            if (!full) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) v[k][i] = i < left[k] ? v[k][i] : 0.f;
            }
        }
        s[0] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] = fmaf(v[k][i], v[k][i], s[0]);
        sum(s, at);
        return 1.f / sqrtf(s[0] * inv_c + a.eps);
    };

    // several waves to a row go through the barriers of its sums together: a block's groups take the same number of steps
    for (long long first = (long long)blockIdx.x * rl.rpb; first < a.rows; first += (long long)gridDim.x * rl.rpb) {
        const long long row = S::row(first + at.group);
        const bool here = row < a.rows;
        if (!S::WAVES && !here) break;
        float y[K][V], o[K][V];
        {
            u32x4 rx[K], ro[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                rx[k] = ro[k] = (u32x4){0u, 0u, 0u, 0u};
                if (here && left[k] > 0) {
                    rx[k] = load_row<T, S::TINY>(gptr<const T>(a.x) + row * a.x_stride + col[k], left[k]);
                    if (have_branch) ro[k] = load_row<T, S::TINY>(gptr<const T>(a.branch) + row * a.branch_stride + col[k], left[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                unpack16<T>(rx[k], y[k]);
                unpack16<T>(ro[k], o[k]);
            }
        }
        if (have_branch) {
            float r = 1.f, mu = 0.f, gt = 1.f;
            if (GM == GM_ROW && here) gt = gate_value(load_param1<T>(a.gate, row * a.gate_stride, gf), a.gate_act);
            if (post) {
                r = normalise(o, mu);
                if (a.stats && here && at.lane == 0) {
                    gptr<float>(a.stats)[row] = mu;
                    gptr<float>(a.stats)[a.rows + row] = r;
                }
            }
            const long long gate_at = GM != GM_VECTOR ? 0 : a.gate_kind == FNET_GATE_ELEMENT ? row * a.gate_stride
                                      : (long long)((uint32_t)row / (uint32_t)a.tokens) * a.gate_stride;
            const float rg = GM == GM_ROW ? r * gt : r;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float g[V], b[V];
                if (GM == GM_VECTOR) {
                    load_param_or<T, S::TINY>(a.gate, gate_at + col[k], gf, here ? left[k] : 0, 0.f, g);
                    gate_values<V>(g, a.gate_act);
                }
                if (a.post_bias) {                   // (v r w + b) = (v r) w + b, with the gate and scale on both
                    float s[V];
                    load_param_or<T, S::TINY>(a.post_bias, col[k], pf, left[k], 0.f, b);
                    load_param_or<T, S::TINY>(a.scale, col[k], pf, left[k], 1.f, s);
#pragma unroll
                    for (int i = 0; i < V; ++i) b[i] *= a.residual_scale * s[i];
                    if (GM == GM_CONST && a.gate) {
                        load_param_or<T, S::TINY>(a.gate, col[k], gf, left[k], 1.f, s);
                        gate_values<V>(s, a.gate_act);
#pragma unroll
                        for (int i = 0; i < V; ++i) b[i] *= s[i];
                    }
                    if (GM == GM_ROW) {
#pragma unroll
                        for (int i = 0; i < V; ++i) b[i] *= gt;
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) o[k][i] = fmaf(o[k][i] * rg, wo[k][i], b[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) o[k][i] = o[k][i] * rg * wo[k][i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) y[k][i] = GM == GM_VECTOR ? fmaf(o[k][i], g[i], y[k][i]) : y[k][i] + o[k][i];
                if (here && left[k] > 0) store_chunk<T>(gptr<T>(a.y) + row * (long long)C + col[k], left[k], y[k]);
            }
        }
        if (pre) {
            float mu;
            const float r = normalise(y, mu);
            if (a.stats && here && at.lane == 0) {
                gptr<float>(a.stats)[2 * a.rows + row] = mu;
                gptr<float>(a.stats)[3 * a.rows + row] = r;
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (a.pre_bias) {
                    float b[V];
                    load_param_or<T, S::TINY>(a.pre_bias, col[k], pf, left[k], 0.f, b);
#pragma unroll
                    for (int i = 0; i < V; ++i) y[k][i] = fmaf(y[k][i] * r, wy[k][i], b[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) y[k][i] = y[k][i] * r * wy[k][i];
                }
                if (here && left[k] > 0) store_chunk<T>(gptr<T>(a.h) + row * (long long)C + col[k], left[k], y[k]);
            }
        }
    }
}

template <typename T, int L, int E>
void run_fwd(const FnetBlockNorm& a, int gm, hipStream_t st) {
    const RowLaunch rl = row_launch(L, E, a.width);
    const long long steps = (a.rows + rl.rpb - 1) / rl.rpb;
    const long long most = 256 * (2048 / rl.threads);                  // what the chip holds at once
    const dim3 grid((unsigned)(steps < most ? steps : most)), block(rl.threads);
    const bool layer = a.kind == FNET_NORM_LAYER;
#define FNET_FWD(GM, LAYER) hipLaunchKernelGGL((k_block_norm_fwd<T, L, E, GM, LAYER>), grid, block, 0, st, a, rl)
    if (gm == GM_CONST) { if (layer) FNET_FWD(GM_CONST, true); else FNET_FWD(GM_CONST, false); }
    else if (gm == GM_ROW) { if (layer) FNET_FWD(GM_ROW, true); else FNET_FWD(GM_ROW, false); }
    else { if (layer) FNET_FWD(GM_VECTOR, true); else FNET_FWD(GM_VECTOR, false); }
#undef FNET_FWD
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
    const int gm = a.gate_kind == FNET_GATE_TOKEN ? GM_ROW : a.gate_kind == FNET_GATE_ELEMENT || a.gate_kind == FNET_GATE_SAMPLE ? GM_VECTOR : GM_CONST;
    DISPATCH_T3(a.dtype, DISPATCH_ROW(a.width, { run_fwd<T, L, E>(a, gm, (hipStream_t)stream); }));
    FNET_LAUNCH_CHECK();
    return FNET_OK;
}
