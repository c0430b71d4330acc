// The backward kernel of the norms around a residual block, for one operand type; fnet_block_norm_{f32,bf16,f16}.hip instantiate it.
#pragma once
#include <type_traits>

#include "fnet_block_norm.h"

// gradients that are sums over rows
enum { SUM_PRE_W = 0, SUM_PRE_B, SUM_POST_W, SUM_POST_B, SUM_SCALE, SUM_GATE, SUM_COUNT };

struct BwdPlan {
    uint64_t dst[SUM_COUNT];     // where a block leaves a sum: its row of the partial sums, or (direct) the gradient itself; 0: nowhere
    int direct;                  // bit i: dst[i] is the gradient, in its own type
    // the gate's sums are left per segment, the others per block; only with a gate per sample does a block go through several segments
    RowCut cut;
    int in_turn;                 // a sample's rows are dealt to its parts in turn; otherwise each part is a run of rows
};

// Waves per SIMD that the kernel is compiled for.  4 leave 128 registers to each; two more sums or a gate in registers do not fit those, and
// 3 waves without spilling are faster than 4 with it.  Two exceptions are told so where the compiler would take one or two registers more:
// 16-bit rows of 8 lanes, and bf16 rows of 16 without biases (16 M elements, 100 wide, a gate per element: 87 us with 3 waves, 79 with 4).
// L = 0 is one kernel for blocks of 5 to 16 waves and has to be compiled for 16, which is 128 registers: of up to 8192 elements a row the forms
// with biases spill 8 to 33 registers and those with a gate per element alone up to 8, wider rows 57 to 167 without biases and 219 to 395 with.
template <typename T>
constexpr int bwd_waves(int L, int gm, bool bias) {
    if (L == 0 || (L == 8 && gm != GM_VECTOR && sizeof(T) == 2) || (L == 16 && !bias && std::is_same<T, bf16_t>::value)) return 4;
    return bias || gm == GM_VECTOR ? 3 : 4;
}

// arrays of weights that the kernel keeps in the LDS; rows of more than 8192 elements leave no room for the third
constexpr int bwd_lds_arrays(int E, bool bias) { return bias && E == 8 ? 3 : 2; }

// one instance: launches the kernel (bias: sums for biases too); how many of its blocks the GPU holds
template <typename T, int L, int E>
int fnet_block_norm_bwd_resident(const RowLaunch& rl, int gm, bool bias, bool layer);
template <typename T, int L, int E>
int fnet_block_norm_bwd_launch(const FnetBlockNorm& a, const BwdPlan& plan, const RowLaunch& rl, int blocks, int gm, bool bias, hipStream_t st);

#ifdef FNET_BLOCK_NORM_KERNELS
namespace {

// With z the normalised branch (or the branch itself), W = residual_scale * scale * post_weight, B = residual_scale * scale * post_bias and
// f = act(gate):   y = x + f (W z + B),   d = gradient of y (of the row's own dy and of h through the second norm)
//   dbranch: q = f d W through the norm;    dgate = act'(gate) d (W z + B)
//   dpost_weight = residual_scale * scale * sum f d z,  dpost_bias = residual_scale * scale * sum f d,
//   dscale = residual_scale * (post_weight * sum f d z + post_bias * sum f d)
// so two sums over rows (one without biases) give every gradient on the branch's side, and where f is constant over the rows it enters only
// when they are left: f is part of W and B, and dgate of a channel or sample comes from the same two sums.
// A row's arithmetic is 18 to 40 operations an element, which keeps it below the time of the 10 to 14 bytes it moves (bf16).
template <typename T, int L, int E, int GM, bool LAYER, bool BIAS>
__global__ __launch_bounds__((RowShape<T, L, E>::MAX_THREADS), bwd_waves<T>(L, GM, BIAS)) void k_block_norm_bwd(FnetBlockNorm a, BwdPlan plan, RowLaunch rl) {
    using S = RowShape<T, L, E>;
    constexpr int V = S::V, K = S::K;
    constexpr bool WY_LDS = bwd_lds_arrays(E, BIAS) == (BIAS ? 3 : 2);
    __shared__ float red[RowSum<L, 3>::SIZE];
    __shared__ float sm[L ? 256 * E : 1];            // several row groups: 256 lanes
    RowSum<L, 3> sum(red);
    const RowPlace<L> at(rl);
    const int C = a.width, groups = rl.rpb;
    const bool pf = a.param_dtype == FNET_F32, gf = a.gate_dtype == FNET_F32;
    const float inv_c = 1.f / (float)C;
    const bool post = a.post != 0, pre = a.dh != 0;
    // the branch is read for y (through the second norm) and for the gradients on its side
    const bool branch_grads = a.branch != 0 && (a.dbranch || a.dgate || a.dscale || a.dpost_weight || a.dpost_bias);
    const bool need_branch = a.branch != 0 && (pre || branch_grads);

    int col[K], left[K];
    bool full = true;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        col[k] = (k * at.lanes + at.lane) * V;
        left[k] = min(max(C - col[k], 0), V);
        full = full && left[k] == V;
    }
    full = __all(full);

    // pre_weight, W and B (above; with f, where that is constant) lie in the LDS, for all rows of the block: in registers they would cost
    // a wave in flight.  Four of a chunk's values to a plane, so that the lanes' 16-byte reads lie side by side.
    extern __shared__ float weights[];
    const int plane = at.lanes * K * 4, pitch = plane * (V / 4);
    float wy_reg[WY_LDS ? 1 : K][V];
    auto put = [&](int which, int k, const float* v) {
        if (at.group == 0) {
#pragma unroll
            for (int p = 0; p < V / 4; ++p)
                *reinterpret_cast<float4*>(weights + which * pitch + p * plane + (k * at.lanes + at.lane) * 4) = make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
        }
    };
    auto get = [&](int which, int k, int p, float* v) {
        const float4 w = *reinterpret_cast<const float4*>(weights + which * pitch + p * plane + (k * at.lanes + at.lane) * 4);
        v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    };
    enum { W_O = 0, W_B = 1, W_Y = BIAS ? 2 : 1 };
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float w[V];
        load_param_or<T, S::TINY>(a.pre_weight, col[k], pf, left[k], 1.f, w);
        if (WY_LDS) put(W_Y, k, w);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) wy_reg[WY_LDS ? 0 : k][i] = w[i];
        }
    }
    auto load_branch_side = [&](long long gate_at) {
        __syncthreads();                             // the segment before has been read
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s[V], w[V];
            load_param_or<T, S::TINY>(a.scale, col[k], pf, left[k], 1.f, s);
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] *= a.residual_scale;
            if (GM == GM_CONST && a.gate) {
                load_param_or<T, S::TINY>(a.gate, gate_at + col[k], gf, left[k], 1.f, w);
                gate_values<V>(w, a.gate_act, gf);
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] *= w[i];
            }
            load_param_or<T, S::TINY>(a.post_weight, col[k], pf, left[k], 1.f, w);
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] *= s[i];
            put(W_O, k, w);
            if (BIAS) {
                load_param_or<T, S::TINY>(a.post_bias, col[k], pf, left[k], 0.f, w);
#pragma unroll
                for (int i = 0; i < V; ++i) w[i] *= s[i];
                put(W_B, k, w);
            }
        }
        __syncthreads();
    };

    float ay[K][V], ay0[BIAS ? K : 1][V], ao[K][V], ao0[BIAS ? K : 1][V];       // sums of dh y_hat, dh, f d z, f d
    auto clear = [](auto& s) {
        for (auto& r : s)
            for (auto& e : r) e = 0.f;
    };
    clear(ay);
    clear(ay0);
    clear(ao);
    clear(ao0);

    // A sum over the block's rows, one value per column, into array `which` of the LDS (in place of weights that are not read any more): the
    // lanes' own columns side by side, several row groups added up in order.
    auto collect = [&](const auto& acc, int which) {
        float* out = weights + which * pitch;
        if (groups == 1) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int p = 0; p < V / 4; ++p)
                    *reinterpret_cast<float4*>(out + col[k] + 4 * p) = make_float4(acc[k][4 * p], acc[k][4 * p + 1], acc[k][4 * p + 2], acc[k][4 * p + 3]);
        } else {
            __syncthreads();                         // the sum before has been read
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) sm[at.group * pitch + col[k] + i] = acc[k][i];
            __syncthreads();
            for (int c = threadIdx.x; c < C; c += blockDim.x) {
                float s = 0.f;
                for (int g = 0; g < groups; ++g) s += sm[g * pitch + c];
                out[c] = s;
            }
        }
    };
    auto leave = [&](int which, long long row, int c, float v, bool f32) {
        const long long to = row * C + c;
        if ((plan.direct >> which & 1) && !f32) gptr<T>(plan.dst[which])[to] = f_to_elem<T>(v);
        else gptr<float>(plan.dst[which])[to] = v;
    };
    // a sum of several segments: a sample's gate is part of each, so they are added up where the block leaves them (always the same thread's
    // column).  A row of partial sums per segment instead: 262144 samples of 2 x 64 bf16 2165 us, now 1380; 65536 of 8 x 512 1273 and 996.
    auto leave_more = [&](int which, bool more, int c, float v) {
        if (more) v += gptr<const float>(plan.dst[which])[(long long)blockIdx.x * C + c];
        leave(which, blockIdx.x, c, v, pf);
    };
    // the branch's sums over a segment, each times its factor (see above): one column per thread
    auto leave_branch_sums = [&](int seg, long long gate_at) {
        const bool more = seg != (int)blockIdx.x;
        if (!(plan.dst[SUM_POST_W] || plan.dst[SUM_POST_B] || plan.dst[SUM_SCALE] || plan.dst[SUM_GATE])) return;
        __syncthreads();
        collect(ao, W_O);
        if (BIAS) collect(ao0, W_B);
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += blockDim.x) {
            const float p1 = weights[W_O * pitch + c], p0 = BIAS ? weights[W_B * pitch + c] : 0.f;
            const float sc = a.residual_scale * (a.scale ? load_param1<T>(a.scale, c, pf) : 1.f);
            const float g = GM == GM_CONST && a.gate ? load_param1<T>(a.gate, gate_at + c, gf) : 0.f;
            const float f = GM == GM_CONST && a.gate ? gate_value(g, a.gate_act, gf) : 1.f;
            if (plan.dst[SUM_POST_W]) leave_more(SUM_POST_W, more, c, sc * f * p1);
            if (BIAS && plan.dst[SUM_POST_B]) leave_more(SUM_POST_B, more, c, sc * f * p0);
            if (plan.dst[SUM_SCALE] || plan.dst[SUM_GATE]) {
                const float u = (a.post_weight ? load_param1<T>(a.post_weight, c, pf) : 1.f) * p1 + (BIAS && a.post_bias ? load_param1<T>(a.post_bias, c, pf) * p0 : 0.f);
                if (plan.dst[SUM_SCALE]) leave_more(SUM_SCALE, more, c, a.residual_scale * f * u);
                if (plan.dst[SUM_GATE]) leave(SUM_GATE, seg, c, sc * gate_slope(g, a.gate_act, gf) * u, gf);
            }
        }
    };

    const int segments = plan.cut.samples * plan.cut.parts;
    for (int seg = blockIdx.x; seg < segments; seg += gridDim.x) {
        const int sample = seg / plan.cut.parts;
        const long long begin = sample * plan.cut.sample_rows, part = seg - sample * plan.cut.parts;
        const long long first = begin + part * (plan.in_turn ? groups : plan.cut.part_rows);
        const long long end = min(plan.in_turn ? begin + plan.cut.sample_rows : first + plan.cut.part_rows, begin + plan.cut.sample_rows);
        const long long stride = plan.in_turn ? (long long)plan.cut.parts * groups : groups;
        const long long sample_gate = a.gate_kind == FNET_GATE_SAMPLE ? (long long)sample * a.gate_stride : 0;
        load_branch_side(sample_gate);
        struct Row {
            u32x4 x[K], o[K], d[K], t[K];            // x, branch, dy, dh as loaded
            float mu_o, r_o, mu_y, r_y, gate;
        };
        auto load = [&](long long row, bool here, Row& r) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                r.x[k] = r.o[k] = r.d[k] = r.t[k] = (u32x4){0u, 0u, 0u, 0u};
                if (here && left[k] > 0) {
                    if (need_branch) r.o[k] = load_row<T, S::TINY>(gptr<const T>(a.branch) + row * a.branch_stride + col[k], left[k]);
                    if (pre) {
                        r.x[k] = load_row<T, S::TINY>(gptr<const T>(a.x) + row * a.x_stride + col[k], left[k]);
                        r.t[k] = load_row<T, S::TINY>(gptr<const T>(a.dh) + row * a.dh_stride + col[k], left[k]);
                    }
                    if (a.dy) r.d[k] = load_row<T, S::TINY>(gptr<const T>(a.dy) + row * a.dy_stride + col[k], left[k]);
                }
            }
            r.mu_o = r.mu_y = r.gate = 0.f;
            r.r_o = r.r_y = 1.f;
            if (here) {
                if (post) { r.mu_o = gptr<const float>(a.stats)[row]; r.r_o = gptr<const float>(a.stats)[a.rows + row]; }
                if (pre) { r.mu_y = gptr<const float>(a.stats)[2 * a.rows + row]; r.r_y = gptr<const float>(a.stats)[3 * a.rows + row]; }
                if (GM == GM_ROW) r.gate = load_param1<T>(a.gate, row * a.gate_stride, gf);
            }
            if (!full) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    align_row<T, S::TINY>(r.o[k], left[k]);
                    align_row<T, S::TINY>(r.x[k], left[k]);
                    align_row<T, S::TINY>(r.t[k], left[k]);
                    align_row<T, S::TINY>(r.d[k], left[k]);
                }
            }
        };
        // several waves to a row go through the barriers of its sums together: a block's groups take the same number of steps
        for (long long step = first; step < end; step += stride) {
            const long long row = S::row(step + at.group);
            const bool here = row < end;
            if (!S::WAVES && !here) break;
            Row now;
            load(row, here, now);
            const float mu_o = now.mu_o, r_o = now.r_o, mu_y = now.mu_y, r_y = now.r_y, gt = now.gate;
            const float ft = GM == GM_ROW ? S::row_value(gate_value(gt, a.gate_act, true)) : 1.f;
            float z[K][V], d[K][V], f[GM == GM_VECTOR ? K : 1][V];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                unpack16<T>(now.o[k], z[k]);
                if (GM == GM_VECTOR) {
                    float(&fk)[V] = f[GM == GM_VECTOR ? k : 0];
                    load_param_or<T, S::TINY>(a.gate, row * a.gate_stride + col[k], gf, here ? left[k] : 0, 0.f, fk);
                    gate_values<V>(fk, a.gate_act, gf);
                }
                if (post) {
#pragma unroll
                    for (int i = 0; i < V; ++i) z[k][i] = LAYER ? (z[k][i] - mu_o) * r_o : z[k][i] * r_o;
                }
            }
            if (!pre) {
#pragma unroll
                for (int k = 0; k < K; ++k) unpack16<T>(now.d[k], d[k]);
            } else {
                float y[K][V], t[K][V], s2[2] = {0.f, 0.f}, wo[4], bo[4], wy[4];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    unpack16<T>(now.x[k], y[k]);
                    unpack16<T>(now.t[k], t[k]);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        if (i % 4 == 0) {            // four columns at a time, to keep fewer weights in registers
                            if (i) __builtin_amdgcn_sched_barrier(0);
                            get(W_O, k, i / 4, wo);
                            if (BIAS) get(W_B, k, i / 4, bo);
                            if (WY_LDS) get(W_Y, k, i / 4, wy);
                        }
                        if (!WY_LDS) wy[i % 4] = wy_reg[WY_LDS ? 0 : k][i];
                        if (GM == GM_CONST) {
                            y[k][i] = fmaf(wo[i % 4], z[k][i], BIAS ? y[k][i] + bo[i % 4] : y[k][i]);
                        } else {
                            const float u = BIAS ? fmaf(wo[i % 4], z[k][i], bo[i % 4]) : wo[i % 4] * z[k][i];
                            y[k][i] = fmaf(GM == GM_ROW ? ft : f[GM == GM_VECTOR ? k : 0][i], u, y[k][i]);
                        }
                        y[k][i] = LAYER ? (y[k][i] - mu_y) * r_y : y[k][i] * r_y;
                        ay[k][i] = fmaf(t[k][i], y[k][i], ay[k][i]);
                        if (BIAS) ay0[BIAS ? k : 0][i] += t[k][i];
                        t[k][i] *= wy[i % 4];
                        if (LAYER) s2[0] += t[k][i];
                        s2[1] = fmaf(t[k][i], y[k][i], s2[1]);
                    }
                }
                if (LAYER) {
                    sum(s2, at);
                } else {
                    float s1[1] = {s2[1]};
                    sum(s1, at);
                    s2[1] = s1[0];
                }
                const float m0 = LAYER ? s2[0] * inv_c : 0.f, m1 = s2[1] * inv_c;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    unpack16<T>(now.d[k], d[k]);        // held as loaded until here: registers are what limits the waves in flight
#pragma unroll
                    for (int i = 0; i < V; ++i) d[k][i] = fmaf(r_y, fmaf(-m1, y[k][i], LAYER ? t[k][i] - m0 : t[k][i]), d[k][i]);
                }
            }
            if (!full) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) d[k][i] = i < left[k] ? d[k][i] : 0.f;
            }
            if (a.dx) {
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (here && left[k] > 0) store_chunk<T>(gptr<T>(a.dx) + row * (long long)C + col[k], left[k], d[k]);
            }
            if (branch_grads) {
                float s3[3] = {0.f, 0.f, 0.f};       // sums of q, q z and, per row, d B; q = d W, with the row's f put in after the sums
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    float wo[4], bo[4];
                    if (GM == GM_VECTOR) {
                        float(&fk)[V] = f[GM == GM_VECTOR ? k : 0];
                        if (a.dgate) {
                            float g[V];
                            load_param_or<T, S::TINY>(a.gate, row * a.gate_stride + col[k], gf, here ? left[k] : 0, 0.f, g);
                            gate_slopes<V>(g, a.gate_act, gf);
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                if (i % 4 == 0) {
                                    get(W_O, k, i / 4, wo);
                                    if (BIAS) get(W_B, k, i / 4, bo);
                                }
                                g[i] *= d[k][i] * (BIAS ? fmaf(wo[i % 4], z[k][i], bo[i % 4]) : wo[i % 4] * z[k][i]);
                            }
                            if (here && left[k] > 0) store_param<T>(a.dgate, row * (long long)C + col[k], gf, left[k], g);
                        }
#pragma unroll
                        for (int i = 0; i < V; ++i) d[k][i] *= fk[i];
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        if (i % 4 == 0) {
                            if (i) __builtin_amdgcn_sched_barrier(0);
                            get(W_O, k, i / 4, wo);
                            if (BIAS) get(W_B, k, i / 4, bo);
                        }
                        const float fd = GM == GM_ROW ? ft * d[k][i] : d[k][i];
                        ao[k][i] = fmaf(fd, z[k][i], ao[k][i]);
                        if (BIAS) ao0[BIAS ? k : 0][i] += fd;
                        if (GM == GM_ROW && BIAS) s3[2] = fmaf(d[k][i], bo[i % 4], s3[2]);
                        d[k][i] *= wo[i % 4];
                        if (LAYER) s3[0] += d[k][i];
                        s3[1] = fmaf(d[k][i], z[k][i], s3[1]);
                    }
                }
                if (post || GM == GM_ROW) sum(s3, at);
                if (GM == GM_ROW && a.dgate && here && at.lane == 0) {
                    const float dg = gate_slope(gt, a.gate_act, true) * (s3[1] + s3[2]);
                    if (gf) gptr<float>(a.dgate)[row] = dg;
                    else gptr<T>(a.dgate)[row] = f_to_elem<T>(dg);
                }
                if (a.dbranch) {
                    const float m0 = LAYER ? s3[0] * inv_c : 0.f, m1 = s3[1] * inv_c, r = r_o * ft;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        if (post) {
#pragma unroll
                            for (int i = 0; i < V; ++i) d[k][i] = r * fmaf(-m1, z[k][i], LAYER ? d[k][i] - m0 : d[k][i]);
                        } else if (GM == GM_ROW) {
#pragma unroll
                            for (int i = 0; i < V; ++i) d[k][i] *= ft;
                        }
                        if (here && left[k] > 0) store_chunk<T>(gptr<T>(a.dbranch) + row * (long long)C + col[k], left[k], d[k]);
                    }
                }
            }
        }
        leave_branch_sums(seg, sample_gate);
        clear(ao);
        clear(ao0);
    }
    if (plan.dst[SUM_PRE_W] || plan.dst[SUM_PRE_B]) {
        __syncthreads();
        collect(ay, W_O);
        if (BIAS) collect(ay0, W_B);
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += blockDim.x) {
            if (plan.dst[SUM_PRE_W]) leave(SUM_PRE_W, blockIdx.x, c, weights[W_O * pitch + c], pf);
            if (BIAS && plan.dst[SUM_PRE_B]) leave(SUM_PRE_B, blockIdx.x, c, weights[W_B * pitch + c], pf);
        }
    }
}

}  // namespace

template <typename T, int L, int E>
const void* bwd_kernel(int gm, bool layer, bool bias) {
#define FNET_BWD(GM)                                                                                                                 \
    (layer ? (bias ? (const void*)k_block_norm_bwd<T, L, E, GM, true, true> : (const void*)k_block_norm_bwd<T, L, E, GM, true, false>) \
           : (bias ? (const void*)k_block_norm_bwd<T, L, E, GM, false, true> : (const void*)k_block_norm_bwd<T, L, E, GM, false, false>))
    return gm == GM_CONST ? FNET_BWD(GM_CONST) : gm == GM_ROW ? FNET_BWD(GM_ROW) : FNET_BWD(GM_VECTOR);
#undef FNET_BWD
}
inline int bwd_lds_bytes(int L, int E, const RowLaunch& rl, bool bias) { return bwd_lds_arrays(E, bias) * (L >= 8 ? L : 64 * rl.waves) * E * 4; }

template <typename T, int L, int E>
int fnet_block_norm_bwd_resident(const RowLaunch& rl, int gm, bool bias, bool layer) {
    return fnet_resident_blocks(bwd_kernel<T, L, E>(gm, layer, bias), rl.threads, bwd_lds_bytes(L, E, rl, bias), 256 * 1024 / rl.threads);
}
template <typename T, int L, int E>
int fnet_block_norm_bwd_launch(const FnetBlockNorm& a, const BwdPlan& plan, const RowLaunch& rl, int blocks, int gm, bool bias, hipStream_t st) {
    const void* kernel = bwd_kernel<T, L, E>(gm, a.kind == FNET_NORM_LAYER, bias);
    const int lds = bwd_lds_bytes(L, E, rl, bias);
    hipError_t e = hipSuccess;
    if (lds > 32768)                                 // with the kernel's static LDS this may pass what is granted without asking
        e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    FnetBlockNorm arg = a;
    BwdPlan p = plan;
    RowLaunch r = rl;
    void* args[] = {&arg, &p, &r};
    if (e == hipSuccess) e = hipLaunchKernel(kernel, dim3(blocks), dim3(rl.threads), args, lds, st);
    if (e != hipSuccess) { g_fnet_last_hip_error = (int)e; return FNET_E_HIP; }
    return FNET_OK;
}
#define FNET_BLOCK_NORM_BWD_INSTANCE(T, L, E)                                                                                          \
    template int fnet_block_norm_bwd_resident<T, L, E>(const RowLaunch&, int, bool, bool);                                            \
    template int fnet_block_norm_bwd_launch<T, L, E>(const FnetBlockNorm&, const BwdPlan&, const RowLaunch&, int, int, bool, hipStream_t);
#endif
