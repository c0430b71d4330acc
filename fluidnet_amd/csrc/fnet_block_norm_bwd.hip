// Backward of the norms around a residual block (formulas at FnetBlockNorm in include/fluidnet_hip.h): one pass over x, branch, gate, dy
// and dh gives dx, dbranch and dgate; the gradients of everything that a row shares with others are summed per block on the way and over
// the blocks by a second, small launch.
#include "fnet_block_norm_bwd.h"

namespace {

// out[group][c] = sum over the group's partial rows, in a fixed order: 16 columns by 64 lanes of rows per block
struct ColSums {
    uint64_t src[SUM_COUNT], dst[SUM_COUNT];
    int groups[SUM_COUNT], slots[SUM_COUNT], f32[SUM_COUNT];
    int count, width;
};
template <typename T>
__global__ __launch_bounds__(1024) void k_block_norm_cols(ColSums a) {
    __shared__ float sm[64][17];
    int e = 0, g = blockIdx.y;
    while (e + 1 < a.count && g >= a.groups[e]) g -= a.groups[e++];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4, c = blockIdx.x * 16 + cx, C = a.width, slots = a.slots[e];
    float s = 0.f;
    if (c < C) {
        const float* p = gptr<const float>(a.src[e]) + (long long)g * slots * C + c;
        int r = ry;
        for (; r + 192 < slots; r += 256) {          // four loads under way
            const float v0 = p[(long long)r * C], v1 = p[(long long)(r + 64) * C], v2 = p[(long long)(r + 128) * C], v3 = p[(long long)(r + 192) * C];
            s += (v0 + v1) + (v2 + v3);
        }
        for (; r < slots; r += 64) s += p[(long long)r * C];
    }
    sm[ry][cx] = s;
    __syncthreads();
    if (ry < 16) {                                   // 16 columns by 16 lanes, four rows each, then over the 16 lanes of a column
        const int col = threadIdx.x >> 4, l = threadIdx.x & 15;
        float t = (sm[l][col] + sm[l + 16][col]) + (sm[l + 32][col] + sm[l + 48][col]);
        t = lane_sum<16>(t);
        const int o = blockIdx.x * 16 + col;
        if (l == 0 && o < C) {
            if (a.f32[e]) gptr<float>(a.dst[e])[(long long)g * C + o] = t;
            else gptr<T>(a.dst[e])[(long long)g * C + o] = f_to_elem<T>(t);
        }
    }
}

struct BwdShape {
    BwdPlan plan;
    RowLaunch rl;
    int blocks, gm;
    bool bias;
    long long bytes;             // of partial sums
};
constexpr int kMinSteps = 4;     // steps of a block's rows at least, where there are that many: a block's partial sums cost as much as a row

// How the rows are cut: blocks that fill the chip once, each with a run of rows; with a gate per sample a run ends with its sample, so that
// what the gate multiplies is constant over it.
void bwd_shape(const FnetBlockNorm& a, int L, int E, BwdShape* out) {
    BwdPlan p{};
    out->rl = row_launch(L, E, a.width);
    const int rpb = out->rl.rpb;
    const bool by_sample = a.gate_kind == FNET_GATE_SAMPLE;
    p.samples = by_sample ? (int)(a.rows / a.tokens) : 1;
    p.sample_rows = by_sample ? a.tokens : a.rows;
    out->gm = a.gate_kind == FNET_GATE_TOKEN ? GM_ROW : a.gate_kind == FNET_GATE_ELEMENT ? GM_VECTOR : GM_CONST;
    out->bias = a.post_bias || a.dpost_bias || a.dpre_bias;
    const int per_cu = (bwd_waves(L, out->gm, out->bias) * 256) / out->rl.threads;
    const long long target = 256 * (per_cu > 1 ? per_cu : 1);
    const long long steps = (p.sample_rows + rpb - 1) / rpb;
    long long parts = target / p.samples;
    if (parts > steps / kMinSteps) parts = steps / kMinSteps;
    if (parts < 1) parts = 1;
    p.part_rows = ((steps + parts - 1) / parts) * rpb;
    p.parts = (int)((p.sample_rows + p.part_rows - 1) / p.part_rows);
    const long long segments = (long long)p.samples * p.parts;
    out->blocks = (int)(segments < target ? segments : target);
    out->bytes = 0;
    const uint64_t want[SUM_COUNT] = {a.dpre_weight, a.dpre_bias, a.dpost_weight, a.dpost_bias, a.dscale, out->gm == GM_CONST ? a.dgate : 0};
    for (int s = 0; s < SUM_COUNT; ++s) {
        if (!want[s]) continue;
        const long long rows = s >= SUM_POST_W ? segments : out->blocks;
        if (s == SUM_GATE && by_sample ? p.parts == 1 : rows == 1) {
            p.direct |= 1 << s;
            p.dst[s] = want[s];
        } else {
            p.dst[s] = a.workspace + out->bytes;
            out->bytes += (rows * a.width * 4 + 15) / 16 * 16;
        }
    }
    out->plan = p;
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
    BwdShape s;
    bwd_shape(a, L, E, &s);
    FNET_CHECK_ARG(s.bytes == 0 || (a.workspace != 0 && a.workspace % 16 == 0 && a.workspace_bytes >= s.bytes));
    fnet_block_norm_bwd_launch<T, L, E>(a, s.plan, s.rl, s.blocks, s.gm, s.bias, st);
    FNET_LAUNCH_CHECK();
    if (s.bytes == 0) return FNET_OK;
    ColSums c{};
    c.width = a.width;
    const uint64_t out[SUM_COUNT] = {a.dpre_weight, a.dpre_bias, a.dpost_weight, a.dpost_bias, a.dscale, a.dgate};
    int groups = 0;
    for (int i = 0; i < SUM_COUNT; ++i) {
        if (!s.plan.dst[i] || (s.plan.direct >> i) & 1) continue;
        const bool by_sample = i == SUM_GATE && a.gate_kind == FNET_GATE_SAMPLE;
        c.src[c.count] = s.plan.dst[i];
        c.dst[c.count] = out[i];
        c.groups[c.count] = by_sample ? s.plan.samples : 1;
        c.slots[c.count] = by_sample ? s.plan.parts : i >= SUM_POST_W ? s.plan.samples * s.plan.parts : s.blocks;
        c.f32[c.count] = (i == SUM_GATE ? a.gate_dtype : a.param_dtype) == FNET_F32;
        groups += c.groups[c.count++];
    }
    hipLaunchKernelGGL(k_block_norm_cols<T>, dim3((a.width + 15) / 16, groups), dim3(1024), 0, st, c);
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
    DISPATCH_ROW(host_args->width, { bwd_shape(*host_args, L, E, &s); });
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
