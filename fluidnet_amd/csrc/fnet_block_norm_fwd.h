// The forward kernel of the norms around a residual block, for one operand type; fnet_block_norm_{f32,bf16,f16}.hip instantiate it.
#pragma once
#include "fnet_block_norm.h"

namespace {

// One row: load, (mean,) sum of squares about it, the residual sum, and the same for the norm of y, all from registers; y enters the second
// norm before it is rounded.  The variance is the mean square about the mean, not E[v^2] - mean^2, which loses everything for rows far from
// zero.  A sample's rows are dealt to its parts in turn, so that the blocks read neighbouring rows at a time: runs of rows of their own put them
// a power of two apart where the rows are, on the same memory channels (4096 x 8192 bf16: 54 us in runs, 45 in turn).  What multiplies a
// normalised value is loaded once per segment.
template <typename T, int L, int E, int GM, bool LAYER, bool BIAS>
__global__ __launch_bounds__((RowShape<T, L, E>::MAX_THREADS)) void k_block_norm_fwd(FnetBlockNorm a, RowCut cut, RowLaunch rl) {
    using S = RowShape<T, L, E>;
    constexpr int V = S::V, K = S::K;
    __shared__ float red[RowSum<L, 2>::SIZE];
    RowSum<L, 2> sum(red);
    const RowPlace<L> at(rl);
    RowMoments<L> moments(sum, at, a.width, V, K);
    const int C = a.width;
    const bool pf = a.param_dtype == FNET_F32, gf = a.gate_dtype == FNET_F32;
    const float inv_c = 1.f / (float)C;
    const bool have_branch = a.branch != 0, post = a.post != 0, pre = a.h != 0;

    int col[K], left[K];                             // first element of each of this lane's chunks, and how many of its elements there are
    bool full = true;
    // residual_scale * scale (* act(gate), where that is constant over the run) times post_weight and post_bias; pre_weight, pre_bias
    float wo[K][V], wy[K][V], bo[BIAS ? K : 1][V], by[BIAS ? K : 1][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        col[k] = (k * at.lanes + at.lane) * V;
        left[k] = min(max(C - col[k], 0), V);
        full = full && left[k] == V;
        load_param_or<T, S::TINY>(a.pre_weight, col[k], pf, left[k], 1.f, wy[k]);
        if (BIAS) load_param_or<T, S::TINY>(a.pre_bias, col[k], pf, left[k], 0.f, by[BIAS ? k : 0]);
    }
    auto load_branch_side = [&](long long gate_at) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s[V];
            load_param_or<T, S::TINY>(a.post_weight, col[k], pf, left[k], 1.f, wo[k]);
            load_param_or<T, S::TINY>(a.scale, col[k], pf, left[k], 1.f, s);
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] *= a.residual_scale;
            if ((GM == GM_CONST || GM == GM_SAMPLE) && a.gate) {
                float g[V];
                load_param_or<T, S::TINY>(a.gate, gate_at + col[k], gf, left[k], 1.f, g);
                gate_values<V>(g, a.gate_act, gf);
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] *= g[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) wo[k][i] *= s[i];
            if (BIAS) {
                load_param_or<T, S::TINY>(a.post_bias, col[k], pf, left[k], 0.f, bo[BIAS ? k : 0]);
#pragma unroll
                for (int i = 0; i < V; ++i) bo[BIAS ? k : 0][i] *= s[i];
            }
        }
    };
    full = __all(full);                              // of this wave: no element of its chunks lies behind the row

    // 1 / deviation of a row (and its mean, taken off)
    auto normalise = [&](float (&v)[K][V], float& mu) {
        float s[1] = {0.f};
        mu = 0.f;
        if (LAYER) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) s[0] += v[k][i];
            s[0] = moments(s[0], [&](float m) {
                float q = 0.f;
                if (full) {
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int i = 0; i < V; ++i) q = fmaf(v[k][i] - m, v[k][i] - m, q);
                } else {
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float d = i < left[k] ? v[k][i] - m : 0.f;
                            q = fmaf(d, d, q);
                        }
                }
                return q;
            }, mu, at);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) v[k][i] = full || i < left[k] ? v[k][i] - mu : 0.f;
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) s[0] = fmaf(v[k][i], v[k][i], s[0]);
            sum(s, at);
        }
        return 1.f / sqrtf(s[0] * inv_c + a.eps);
    };

    // one segment to a block, except with a gate per sample
    int seg = blockIdx.x;
    if (GM != GM_SAMPLE) load_branch_side(0);
    do {
    const int sample = GM == GM_SAMPLE ? seg / cut.parts : 0;
    const long long end = GM == GM_SAMPLE ? (sample + 1) * cut.sample_rows : a.rows;
    if (GM == GM_SAMPLE) load_branch_side((long long)sample * a.gate_stride);
    // several waves to a row go through the barriers of its sums together: a block's groups take the same number of steps
    for (long long step = sample * cut.sample_rows + (long long)(seg - sample * cut.parts) * rl.rpb; step < end; step += (long long)cut.parts * rl.rpb) {
        const long long row = S::row(step + at.group);
        const bool here = row < end;
        if (!S::WAVES && !here) break;
        float y[K][V], o[K][V], g[GM == GM_VECTOR ? K : 1][V], gt = 1.f;
        if (GM == GM_ROW && here) gt = load_param1<T>(a.gate, row * a.gate_stride, gf);
        {
            u32x4 rx[K], ro[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                rx[k] = ro[k] = (u32x4){0u, 0u, 0u, 0u};
                if (GM == GM_VECTOR) load_param_or<T, S::TINY>(a.gate, row * a.gate_stride + col[k], gf, here ? left[k] : 0, 0.f, g[GM == GM_VECTOR ? k : 0]);
                if (here && left[k] > 0) {
                    rx[k] = load_row<T, S::TINY>(gptr<const T>(a.x) + row * a.x_stride + col[k], left[k]);
                    if (have_branch) ro[k] = load_row<T, S::TINY>(gptr<const T>(a.branch) + row * a.branch_stride + col[k], left[k]);
                }
            }
            if (!full) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    align_row<T, S::TINY>(rx[k], left[k]);
                    align_row<T, S::TINY>(ro[k], left[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                unpack16<T>(rx[k], y[k]);
                unpack16<T>(ro[k], o[k]);
            }
        }
        if (have_branch) {
            float r = 1.f, mu = 0.f;
            if (GM == GM_ROW) gt = S::row_value(gate_value(gt, a.gate_act, true));
            if (post) {
                r = normalise(o, mu);
                if (a.stats && here && at.lane == 0) {
                    gptr<float>(a.stats)[row] = mu;
                    gptr<float>(a.stats)[a.rows + row] = r;
                }
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (GM == GM_VECTOR) gate_values<V>(g[GM == GM_VECTOR ? k : 0], a.gate_act, gf);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    o[k][i] = BIAS ? fmaf(o[k][i] * r, wo[k][i], bo[BIAS ? k : 0][i]) : o[k][i] * r * wo[k][i];
                    y[k][i] = GM == GM_CONST || GM == GM_SAMPLE ? y[k][i] + o[k][i] : fmaf(o[k][i], GM == GM_ROW ? gt : g[GM == GM_VECTOR ? k : 0][i], y[k][i]);
                }
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
#pragma unroll
                for (int i = 0; i < V; ++i) y[k][i] = BIAS ? fmaf(y[k][i] * r, wy[k][i], by[BIAS ? k : 0][i]) : y[k][i] * r * wy[k][i];
                if (here && left[k] > 0) store_chunk<T>(gptr<T>(a.h) + row * (long long)C + col[k], left[k], y[k]);
            }
        }
    }
    } while (GM == GM_SAMPLE && (seg += gridDim.x) < cut.samples * cut.parts);
}

}  // namespace

template <typename T, int L, int E>
int fnet_block_norm_fwd_launch(const FnetBlockNorm& a, hipStream_t st) {
    const RowLaunch rl = row_launch(L, E, a.width);
    const bool layer = a.kind == FNET_NORM_LAYER, bias = a.post_bias || a.pre_bias;
#define FNET_FWD(GM)                                                                                                                 \
    (layer ? (bias ? (const void*)k_block_norm_fwd<T, L, E, GM, true, true> : (const void*)k_block_norm_fwd<T, L, E, GM, true, false>) \
           : (bias ? (const void*)k_block_norm_fwd<T, L, E, GM, false, true> : (const void*)k_block_norm_fwd<T, L, E, GM, false, false>))
    const void* kernel = a.gate_kind == FNET_GATE_TOKEN ? FNET_FWD(GM_ROW) : a.gate_kind == FNET_GATE_ELEMENT ? FNET_FWD(GM_VECTOR)
                         : a.gate_kind == FNET_GATE_SAMPLE ? FNET_FWD(GM_SAMPLE) : FNET_FWD(GM_CONST);
#undef FNET_FWD
    // one block for each that the GPU holds: a second round would run with part of the GPU idle
    int most = fnet_resident_blocks(kernel, rl.threads, 0, 256 * 1024 / rl.threads);
    // ... up to 24 waves a CU, but two blocks.  30 M bf16 elements, rms, none / with a gate per token: 4096 wide 41 / 42 us with three blocks of 8
    // waves, 43 / 51 with four; 4608 wide 41 / 46 with two of 9, 42 / 55 with three; 2304 wide 41 / 43 with four of 5, 49 / 52 with six; 8192
    // wide 50 / 55 with one of 16, 42 / 60 with two.
    most = std::min(most, 256 * std::max(2, 24 * 64 / rl.threads));
    RowCut cut = cut_rows(a, rl.rpb, most, 1);
    FnetBlockNorm arg = a;
    RowLaunch r = rl;
    void* args[] = {&arg, &cut, &r};
    const int segments = cut.samples * cut.parts;
    const hipError_t e = hipLaunchKernel(kernel, dim3(segments < most ? segments : most), dim3(rl.threads), args, 0, st);
    if (e != hipSuccess) { g_fnet_last_hip_error = (int)e; return FNET_E_HIP; }
    return FNET_OK;
}
#define FNET_BLOCK_NORM_FWD_INSTANCE(T, L, E) template int fnet_block_norm_fwd_launch<T, L, E>(const FnetBlockNorm&, hipStream_t);
