// Backward of the norms around a residual block (formulas at FnetBlockNorm in include/fluidnet_hip.h): one pass over x, branch, gate, dy
// and dh gives dx, dbranch and dgate; the gradients of everything that a row shares with others are summed per block on the way and over
// the blocks by a second, small launch.
#include "fnet_block_norm.h"

namespace {

// what is summed over rows; the weights come first, so that a norm without biases, gate and scale sums two of them only
enum { SUM_PRE_W = 0, SUM_POST_W, SUM_PRE_B, SUM_POST_B, SUM_SCALE, SUM_GATE, SUM_COUNT };

struct BwdPlan {
    uint64_t dst[SUM_COUNT];     // where a block leaves a sum: its row of the partial sums, or (direct) the gradient itself; 0: nowhere
    int direct;                  // bit i: dst[i] is the gradient, in its own type
    int samples, parts;          // segments = samples * parts: part p of a sample is its rows [p * part_rows, (p + 1) * part_rows)
    long long sample_rows, part_rows;
};

// The sums of a block's row groups into one row of `dst`.  Rows inside waves (L <= 64): through LDS, group by group in order.
template <typename T, int L, int E>
__device__ __forceinline__ void leave_sum(const float (&acc)[RowShape<T, L, E>::K][RowShape<T, L, E>::V], uint64_t dst, long long row, int C,
                                          bool direct, bool f32, float* sm) {
    using S = RowShape<T, L, E>;
    constexpr int V = S::V, K = S::K;
    const int lane = threadIdx.x % L;
    if (L > 64) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * L + lane) * V, n = min(C - c, V);
            if (n <= 0) continue;
            if (direct) {
                store_param<T>(dst, row * C + c, f32, n, acc[k]);
            } else {
                float* q = gptr<float>(dst) + row * C + c;
#pragma unroll
                for (int i = 0; i < V; i += 4)
                    if (n > i) store_chunk<float>(q + i, min(n - i, 4), &acc[k][i]);
            }
        }
    } else {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) sm[(threadIdx.x / L) * (L * E) + (k * L + lane) * V + i] = acc[k][i];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += S::THREADS) {
            float s = 0.f;
            for (int g = 0; g < S::RPB; ++g) s += sm[g * (L * E) + c];
            if (direct && !f32) gptr<T>(dst)[row * C + c] = f_to_elem<T>(s);
            else gptr<float>(dst)[row * C + c] = s;
        }
    }
}

// NS: how many of the sums are kept (0, 2 or all).  A sum costs E registers per lane.
template <typename T, int L, int E, int NS>
__global__ __launch_bounds__((RowShape<T, L, E>::THREADS)) void k_block_norm_bwd(FnetBlockNorm a, BwdPlan plan) {
    using S = RowShape<T, L, E>;
    constexpr int V = S::V, K = S::K;
    __shared__ float red[2 * 3 * RowSum<L, 3>::W];
    __shared__ float sm[L <= 64 && NS > 0 ? 256 * E : 1];
    RowSum<L, 3> sum(red);
    const int C = a.width, lane = threadIdx.x % L;
    const bool pf = a.param_dtype == FNET_F32, gf = a.gate_dtype == FNET_F32, layer = a.kind == FNET_NORM_LAYER;
    const float inv_c = 1.f / (float)C;
    const bool post = a.post != 0, pre = a.dh != 0;
    // the branch's side is needed for y (through the second norm) and for the gradients on its side
    const bool branch_grads = a.branch != 0 && (a.dbranch || a.dgate || a.dscale || a.dpost_weight || a.dpost_bias);
    const bool need_u = a.branch != 0 && (pre || branch_grads);

    int left[K];
#pragma unroll
    for (int k = 0; k < K; ++k) left[k] = min(max(C - (k * L + lane) * V, 0), V);
    float acc[NS > 0 ? NS : 1][K][V];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[s][k][i] = 0.f;

    const int segments = plan.samples * plan.parts;
    for (int seg = blockIdx.x; seg < segments; seg += gridDim.x) {
        const int sample = seg / plan.parts;
        const long long first = sample * plan.sample_rows + (seg - sample * plan.parts) * plan.part_rows;
        const long long end = min(first + plan.part_rows, (sample + 1) * plan.sample_rows);
        for (long long row = first + threadIdx.x / L; row < end; row += S::RPB) {
            float y[K][V], o[K][V], d[K][V], g[K][V];       // y: x, then y; o: branch, then its norm; d: the gradient of y; g: the gate
            float mu_o = 0.f, r_o = 1.f, mu_y = 0.f, r_y = 1.f, gt = 0.f;
            const long long gate_at = a.gate_kind == FNET_GATE_ELEMENT || a.gate_kind == FNET_GATE_TOKEN ? row * a.gate_stride
                                      : a.gate_kind == FNET_GATE_SAMPLE ? (long long)sample * a.gate_stride : 0;
            const bool gate_row = a.gate_kind != FNET_GATE_NONE && a.gate_kind != FNET_GATE_TOKEN && need_u;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * L + lane) * V;
#pragma unroll
                for (int i = 0; i < V; ++i) { y[k][i] = 0.f; o[k][i] = 0.f; d[k][i] = 0.f; g[k][i] = 1.f; }
                if (left[k] > 0) {
                    if (pre) load_chunk<T>(gptr<const T>(a.x) + row * a.x_stride + c, left[k], y[k]);
                    if (need_u) load_chunk<T>(gptr<const T>(a.branch) + row * a.branch_stride + c, left[k], o[k]);
                    if (a.dy) load_chunk<T>(gptr<const T>(a.dy) + row * a.dy_stride + c, left[k], d[k]);
                    if (gate_row) load_param<T>(a.gate, gate_at + c, gf, left[k], g[k]);
                }
            }
            if (post) { mu_o = gptr<const float>(a.stats)[row]; r_o = gptr<const float>(a.stats)[a.rows + row]; }
            if (pre) { mu_y = gptr<const float>(a.stats)[2 * a.rows + row]; r_y = gptr<const float>(a.stats)[3 * a.rows + row]; }
            if (a.gate_kind == FNET_GATE_TOKEN && need_u) gt = load_param1<T>(a.gate, gate_at, gf);
            const float pt = gate_value(gt, a.gate_act);

            // u of chunk k, and residual_scale * scale * act(gate) without (sc) and with (sp) the gate
            auto branch_side = [&](int k, float (&u)[V], float (&sc)[V], float (&sp)[V]) {
                const int c = (k * L + lane) * V;
                float w[V], b[V];
#pragma unroll
                for (int i = 0; i < V; ++i) { w[i] = 1.f; b[i] = 0.f; sc[i] = a.residual_scale; }
                if (left[k] > 0) {
                    if (a.post_weight) load_param<T>(a.post_weight, c, pf, left[k], w);
                    if (a.post_bias) load_param<T>(a.post_bias, c, pf, left[k], b);
                    if (a.scale) {
                        load_param<T>(a.scale, c, pf, left[k], sc);
#pragma unroll
                        for (int i = 0; i < V; ++i) sc[i] *= a.residual_scale;
                    }
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    u[i] = fmaf(o[k][i], w[i], b[i]);
                    const float phi = a.gate_kind == FNET_GATE_NONE ? 1.f : a.gate_kind == FNET_GATE_TOKEN ? pt : gate_value(g[k][i], a.gate_act);
                    sp[i] = sc[i] * phi;
                }
            };
            if (need_u) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int i = 0; i < V; ++i) o[k][i] = (o[k][i] - mu_o) * r_o;
                    float u[V], sc[V], sp[V];
                    branch_side(k, u, sc, sp);
#pragma unroll
                    for (int i = 0; i < V; ++i) y[k][i] = fmaf(sp[i], u[i], y[k][i]);
                }
            }
            if (pre) {
                float t[K][V], s2[2] = {0.f, 0.f};
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = (k * L + lane) * V;
                    float w[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) { t[k][i] = 0.f; w[i] = 1.f; }
                    if (left[k] > 0) {
                        load_chunk<T>(gptr<const T>(a.dh) + row * a.dh_stride + c, left[k], t[k]);
                        if (a.pre_weight) load_param<T>(a.pre_weight, c, pf, left[k], w);
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        y[k][i] = (y[k][i] - mu_y) * r_y;
                        if (NS > SUM_PRE_W) acc[SUM_PRE_W][k][i] = fmaf(t[k][i], y[k][i], acc[SUM_PRE_W][k][i]);
                        if (NS > SUM_PRE_B) acc[NS > SUM_PRE_B ? SUM_PRE_B : 0][k][i] += t[k][i];
                        t[k][i] *= w[i];
                        s2[0] += t[k][i];
                        s2[1] = fmaf(t[k][i], y[k][i], s2[1]);
                    }
                }
                sum(s2);
                const float m0 = layer ? s2[0] * inv_c : 0.f, m1 = s2[1] * inv_c;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i < left[k]) d[k][i] = fmaf(r_y, t[k][i] - m0 - y[k][i] * m1, d[k][i]);
            }
            if (a.dx) {
                T* p = gptr<T>(a.dx) + row * (long long)C;
#pragma unroll
                for (int k = 0; k < K; ++k)
                    if (left[k] > 0) store_chunk<T>(p + (k * L + lane) * V, left[k], d[k]);
            }
            if (branch_grads) {
                float s3[3] = {0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = (k * L + lane) * V;
                    float u[V], sc[V], sp[V], w[V];
                    branch_side(k, u, sc, sp);
#pragma unroll
                    for (int i = 0; i < V; ++i) w[i] = 1.f;
                    if (a.post_weight && left[k] > 0) load_param<T>(a.post_weight, c, pf, left[k], w);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float gi = a.gate_kind == FNET_GATE_TOKEN ? gt : g[k][i];
                        const float phi = a.gate_kind == FNET_GATE_NONE ? 1.f : a.gate_kind == FNET_GATE_TOKEN ? pt : gate_value(gi, a.gate_act);
                        const float dg = d[k][i] * sc[i] * u[i] * gate_slope(gi, a.gate_act), du = d[k][i] * sp[i];
                        s3[2] += dg;
                        g[k][i] = dg;
                        if (NS > SUM_SCALE) acc[NS > SUM_SCALE ? SUM_SCALE : 0][k][i] = fmaf(d[k][i] * a.residual_scale, phi * u[i], acc[NS > SUM_SCALE ? SUM_SCALE : 0][k][i]);
                        if (NS > SUM_GATE) acc[NS > SUM_GATE ? SUM_GATE : 0][k][i] += dg;
                        if (NS > SUM_POST_W) acc[NS > SUM_POST_W ? SUM_POST_W : 0][k][i] = fmaf(du, o[k][i], acc[NS > SUM_POST_W ? SUM_POST_W : 0][k][i]);
                        if (NS > SUM_POST_B) acc[NS > SUM_POST_B ? SUM_POST_B : 0][k][i] += du;
                        d[k][i] = du * w[i];
                        s3[0] += d[k][i];
                        s3[1] = fmaf(d[k][i], o[k][i], s3[1]);
                    }
                }
                if (post || a.gate_kind == FNET_GATE_TOKEN) sum(s3);
                if (a.gate_kind == FNET_GATE_TOKEN && a.dgate && lane == 0) {
                    if (gf) gptr<float>(a.dgate)[row] = s3[2];
                    else gptr<T>(a.dgate)[row] = f_to_elem<T>(s3[2]);
                }
                const float m0 = layer ? s3[0] * inv_c : 0.f, m1 = s3[1] * inv_c;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (left[k] <= 0) continue;
                    const long long at = row * (long long)C + (k * L + lane) * V;
                    if (a.gate_kind == FNET_GATE_ELEMENT && a.dgate) store_param<T>(a.dgate, at, gf, left[k], g[k]);
                    if (a.dbranch) {
                        if (post) {
#pragma unroll
                            for (int i = 0; i < V; ++i) d[k][i] = r_o * (d[k][i] - m0 - o[k][i] * m1);
                        }
                        store_chunk<T>(gptr<T>(a.dbranch) + at, left[k], d[k]);
                    }
                }
            }
        }
        if (NS > SUM_GATE && a.gate_kind == FNET_GATE_SAMPLE && plan.dst[SUM_GATE]) {
            constexpr int G = NS > SUM_GATE ? SUM_GATE : 0;
            leave_sum<T, L, E>(acc[G], plan.dst[SUM_GATE], seg, C, (plan.direct >> SUM_GATE) & 1, gf, sm);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[G][k][i] = 0.f;
        }
    }
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (plan.dst[s] && !(s == SUM_GATE && a.gate_kind == FNET_GATE_SAMPLE))
            leave_sum<T, L, E>(acc[s], plan.dst[s], blockIdx.x, C, (plan.direct >> s) & 1, s == SUM_GATE ? gf : pf, sm);
}

// out[group][c] = sum over the group's partial rows, in order: 32 columns by 32 lanes of rows per block
struct ColSums {
    uint64_t src[SUM_COUNT], dst[SUM_COUNT];
    int groups[SUM_COUNT], slots[SUM_COUNT], f32[SUM_COUNT];
    int count, width;
};
template <typename T>
__global__ __launch_bounds__(1024) void k_block_norm_cols(ColSums a) {
    __shared__ float sm[32][33];
    int e = 0, g = blockIdx.y;
    while (e + 1 < a.count && g >= a.groups[e]) g -= a.groups[e++];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx, C = a.width;
    float s = 0.f;
    if (c < C) {
        const float* p = gptr<const float>(a.src[e]) + (long long)g * a.slots[e] * C + c;
        for (int r = ry; r < a.slots[e]; r += 32) s += p[(long long)r * C];
    }
    sm[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && c < C) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) t += sm[r][cx];
        if (a.f32[e]) gptr<float>(a.dst[e])[(long long)g * C + c] = t;
        else gptr<T>(a.dst[e])[(long long)g * C + c] = f_to_elem<T>(t);
    }
}

struct BwdShape {
    BwdPlan plan;
    int blocks, ns;
    long long bytes;             // of partial sums
};
constexpr int kMinSteps = 4;     // steps of a block's rows at least, where there are that many: a block's partial sums cost as much as a row

// How the rows are cut: blocks that fill the chip once, each with a run of rows; with a gate per sample a run ends with its sample, so that
// the gate's gradient is summed with the others.
int bwd_shape(const FnetBlockNorm& a, int threads, int rpb, BwdShape* out) {
    BwdPlan p{};
    const bool by_sample = a.gate_kind == FNET_GATE_SAMPLE;
    p.samples = by_sample ? (int)(a.rows / a.tokens) : 1;
    p.sample_rows = by_sample ? a.tokens : a.rows;
    const long long target = 256 * (1024 / threads);
    const long long steps = (p.sample_rows + rpb - 1) / rpb;
    long long parts = target / p.samples;
    if (parts > steps / kMinSteps) parts = steps / kMinSteps;
    if (parts < 1) parts = 1;
    p.part_rows = ((steps + parts - 1) / parts) * rpb;
    p.parts = (int)((p.sample_rows + p.part_rows - 1) / p.part_rows);
    const long long segments = (long long)p.samples * p.parts;
    out->blocks = (int)(segments < target ? segments : target);
    out->ns = 0;
    out->bytes = 0;
    const uint64_t want[SUM_COUNT] = {a.dpre_weight, a.dpost_weight, a.dpre_bias, a.dpost_bias, a.dscale,
                                      a.gate_kind == FNET_GATE_SAMPLE || a.gate_kind == FNET_GATE_CHANNEL ? a.dgate : 0};
    for (int s = 0; s < SUM_COUNT; ++s) {
        if (!want[s]) continue;
        out->ns = s < 2 && out->ns <= 2 ? 2 : SUM_COUNT;
        const bool gate_rows = s == SUM_GATE && by_sample;
        const long long rows = gate_rows ? segments : out->blocks;
        if (gate_rows ? p.parts == 1 : out->blocks == 1) {
            p.direct |= 1 << s;
            p.dst[s] = want[s];
        } else {
            p.dst[s] = a.workspace + out->bytes;
            out->bytes += (rows * a.width * 4 + 15) / 16 * 16;
        }
    }
    out->plan = p;
    return FNET_OK;
}

int bwd_check(const FnetBlockNorm* a) {
    const int rc = fnet_block_norm_check(a);
    if (rc != FNET_OK) return rc;
    FNET_CHECK_ARG(a->branch != 0 || (!a->dbranch && !a->dgate && !a->dscale));
    FNET_CHECK_ARG(a->post || (!a->dpost_weight && !a->dpost_bias));
    FNET_CHECK_ARG(a->gate_kind != FNET_GATE_NONE || !a->dgate);
    const auto ok = [](uint64_t p, int dtype) { return p % (dtype == FNET_F32 ? 4 : 2) == 0; };
    FNET_CHECK_ARG(ok(a->dy | a->dh | a->dx | a->dbranch, a->dtype) && ok(a->dgate, a->gate_dtype));
    FNET_CHECK_ARG(ok(a->dscale | a->dpost_weight | a->dpost_bias | a->dpre_weight | a->dpre_bias, a->param_dtype));
    return FNET_OK;
}

template <typename T, int L, int E>
int run_bwd(const FnetBlockNorm& a, hipStream_t st) {
    using S = RowShape<T, L, E>;
    BwdShape s;
    bwd_shape(a, S::THREADS, S::RPB, &s);
    FNET_CHECK_ARG(s.bytes == 0 || (a.workspace != 0 && a.workspace % 16 == 0 && a.workspace_bytes >= s.bytes));
    const dim3 grid(s.blocks), block(S::THREADS);
    if (s.ns == 0) hipLaunchKernelGGL((k_block_norm_bwd<T, L, E, 0>), grid, block, 0, st, a, s.plan);
    else if (s.ns == 2) hipLaunchKernelGGL((k_block_norm_bwd<T, L, E, 2>), grid, block, 0, st, a, s.plan);
    else hipLaunchKernelGGL((k_block_norm_bwd<T, L, E, SUM_COUNT>), grid, block, 0, st, a, s.plan);
    FNET_LAUNCH_CHECK();
    if (s.bytes == 0) return FNET_OK;
    ColSums c{};
    c.width = a.width;
    const uint64_t out[SUM_COUNT] = {a.dpre_weight, a.dpost_weight, a.dpre_bias, a.dpost_bias, a.dscale, a.dgate};
    int groups = 0;
    for (int i = 0; i < SUM_COUNT; ++i) {
        if (!s.plan.dst[i] || (s.plan.direct >> i) & 1) continue;
        const bool by_sample = i == SUM_GATE && a.gate_kind == FNET_GATE_SAMPLE;
        c.src[c.count] = s.plan.dst[i];
        c.dst[c.count] = out[i];
        c.groups[c.count] = by_sample ? s.plan.samples : 1;
        c.slots[c.count] = by_sample ? s.plan.parts : s.blocks;
        c.f32[c.count] = (i == SUM_GATE ? a.gate_dtype : a.param_dtype) == FNET_F32;
        groups += c.groups[c.count++];
    }
    hipLaunchKernelGGL(k_block_norm_cols<T>, dim3((a.width + 31) / 32, groups), dim3(1024), 0, st, c);
    FNET_LAUNCH_CHECK();
    return FNET_OK;
}

}  // namespace

int fnet_block_norm_workspace(const FnetBlockNorm* host_args, int64_t* bytes) {
    FNET_CHECK_ARG(bytes);
    const int rc = bwd_check(host_args);
    if (rc != FNET_OK) return rc;
    *bytes = 0;
    if (host_args->rows == 0) return FNET_OK;
    BwdShape s;
    DISPATCH_T3(host_args->dtype, DISPATCH_ROW(host_args->width, { using S = RowShape<T, L, E>; bwd_shape(*host_args, S::THREADS, S::RPB, &s); }));
    *bytes = s.bytes;
    return FNET_OK;
}

int fnet_block_norm_bwd(const FnetBlockNorm* host_args, void* stream) {
    const int rc = bwd_check(host_args);
    if (rc != FNET_OK) return rc;
    const FnetBlockNorm& a = *host_args;
    if (a.rows == 0) return FNET_OK;
    FNET_CHECK_ARG((!a.post && !a.dh) || a.stats != 0);
    FNET_CHECK_ARG(a.dh != 0 || (!a.dpre_weight && !a.dpre_bias));
    int out = FNET_OK;
    DISPATCH_T3(a.dtype, DISPATCH_ROW(a.width, { out = run_bwd<T, L, E>(a, (hipStream_t)stream); }));
    return out;
}
