// Norms around a residual block: argument checks, the cut of the rows, the sum of a backward's partial sums and the C entries.  The two large
// kernels are in fnet_block_norm_fwd.h / fnet_block_norm_bwd.h, compiled once per operand type (fnet_block_norm_{f32,bf16,f16}.hip).
#include <algorithm>
#include <mutex>

#include "fnet_block_norm_bwd.h"

namespace {

bool type_ok(int d, int operand) { return d == FNET_F32 || d == operand; }
bool aligned(uint64_t p, int dtype) { return p % (dtype == FNET_F32 ? 4 : 2) == 0; }

// The arguments as the kernels take them: a gate per sample of one token is a row of values per row.  (Samples of two tokens and more are at
// most 2^30, so the kernels' 32-bit count of segments stays below 2^31 when a grid is added to it; samples of one row may be 2^31 - 1.)
FnetBlockNorm as_launched(const FnetBlockNorm& given) {
    FnetBlockNorm a = given;
    if (a.gate_kind == FNET_GATE_SAMPLE && a.tokens == 1) a.gate_kind = FNET_GATE_ELEMENT;
    return a;
}

}  // namespace

int fnet_resident_blocks(const void* kernel, int threads, size_t lds, int otherwise) {
    struct Known { const void* kernel; int threads, device; size_t lds; int blocks; };
    static std::mutex mu;
    static Known known[1024];
    static int count = 0;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return otherwise;
    std::lock_guard<std::mutex> lock(mu);
    // open addressing: the few shapes of a program are found at once, and a full table only means asking again
    size_t h = ((size_t)kernel >> 4) * 31 + threads + lds * 7 + dev;
    for (int probe = 0; probe < 1024; ++probe, ++h) {
        Known& k = known[h & 1023];
        if (k.kernel == kernel && k.threads == threads && k.lds == lds && k.device == dev) return k.blocks;
        if (k.kernel) continue;
        // What a CU holds, from the kernel's registers and LDS: hipOccupancyMaxActiveBlocksPerMultiprocessor names more where the waves of a block
        // are no multiple of four, and blocks too many run one after the rest.  Measured, 5 waves take the room of 8 (bf16 backward, 13020 x
        // 2304: 112 us with three blocks a CU, 90 with two; forward, 10653 x 2816 with a gate per token: 67 and 54).  Three waves a block pack
        // better in some kernels: 25000 x 1200 layer norms with biases 149 -> 113, with a gate per element and no biases 144 -> 168.
        hipFuncAttributes attr;
        int cus = 0, shared = 0;
        if (hipFuncGetAttributes(&attr, kernel) != hipSuccess || attr.numRegs < 1 ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1 ||
            hipDeviceGetAttribute(&shared, hipDeviceAttributeMaxSharedMemoryPerMultiprocessor, dev) != hipSuccess || shared < 1) {
            (void)hipGetLastError();
            return otherwise;
        }
        const int waves = std::min(8, 512 / ((attr.numRegs + 7) / 8 * 8)), per_simd = (threads / 64 + 3) / 4;
        const size_t bytes = attr.sharedSizeBytes + lds;
        int per_cu = waves / per_simd;
        if (bytes) per_cu = std::min(per_cu, (int)(shared / bytes));
        per_cu = std::max(per_cu, 1);
        if (count < 1000) {
            ++count;
            k = Known{kernel, threads, dev, lds, per_cu * cus};
        }
        return per_cu * cus;
    }
    return otherwise;
}

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
    const FnetBlockNorm a = as_launched(*host_args);
    if (a.rows == 0) return FNET_OK;
    FNET_CHECK_ARG((a.branch != 0) == (a.y != 0) && (a.y != 0 || a.h != 0) && (a.h != 0 || (a.pre_weight == 0 && a.pre_bias == 0)));
    FNET_CHECK_ARG(aligned(a.y | a.h, a.dtype));
    int out = FNET_OK;
    DISPATCH_T3(a.dtype, DISPATCH_ROW(a.width, { out = fnet_block_norm_fwd_launch<T, L, E>(a, (hipStream_t)stream); }));
    return out;
}

// ---- backward
namespace {

// out[group][c] = sum over the group's partial rows, in a fixed order: 64 columns by 64 lanes of rows per block, 16 bytes a lane
struct ColSums {
    uint64_t src[SUM_COUNT], dst[SUM_COUNT];
    int groups[SUM_COUNT], slots[SUM_COUNT], f32[SUM_COUNT];
    int count, width;
};
template <typename T>
__global__ __launch_bounds__(1024) void k_block_norm_cols(ColSums a) {
    __shared__ float sm[64][65];
    int e = 0, g = blockIdx.y;
    while (e + 1 < a.count && g >= a.groups[e]) g -= a.groups[e++];
    const int cx = (threadIdx.x & 15) * 4, ry = threadIdx.x >> 4, c = blockIdx.x * 64 + cx, C = a.width, slots = a.slots[e], n = C - c;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (n > 0) {
        const float* p = gptr<const float>(a.src[e]) + (long long)g * slots * C + c;
        int r = ry;
        for (; r + 192 < slots; r += 256) {          // four loads under way
            float v[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) load_chunk<float>(p + (long long)(r + 64 * k) * C, n, v[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] += v[k][i];
        }
        for (; r < slots; r += 64) {
            float v[4];
            load_chunk<float>(p + (long long)r * C, n, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sm[ry][cx + i] = s[i];
    __syncthreads();
    const int col = threadIdx.x >> 4, l = threadIdx.x & 15, o = blockIdx.x * 64 + col;
    const float t = lane_sum<16>((sm[l][col] + sm[l + 16][col]) + (sm[l + 32][col] + sm[l + 48][col]));
    if (l == 0 && o < C) {
        if (a.f32[e]) gptr<float>(a.dst[e])[(long long)g * C + o] = t;
        else gptr<T>(a.dst[e])[(long long)g * C + o] = f_to_elem<T>(t);
    }
}

struct BwdShape {
    BwdPlan plan;
    RowLaunch rl;
    int blocks, gm;
    bool bias;
    long long bytes;             // of partial sums
};
// Steps of a block's rows at least, once every CU has a block: a block's partial sums cost as much as a row.  2031 x 1001 fp32 with every
// operand: 36 us with 4, 32 with 2 or 1; 2000 x 2048 bf16: 24, 25, 25; 512 x 4096: 23, 22, 24; 128 x 4096, a step per block: 21 -> 16.
constexpr int kMinSteps = 2;

// Blocks that fill the chip once, and where each leaves its sums.  most: blocks that the GPU holds at once, as far as that is known (the
// workspace is of the most that there may be).
void bwd_shape(const FnetBlockNorm& a, int L, int E, int most, BwdShape* out) {
    BwdPlan p{};
    out->rl = row_launch(L, E, a.width);
    const int rpb = out->rl.rpb;
    const bool by_sample = a.gate_kind == FNET_GATE_SAMPLE;
    out->gm = a.gate_kind == FNET_GATE_TOKEN ? GM_ROW : a.gate_kind == FNET_GATE_ELEMENT ? GM_VECTOR : GM_CONST;
    out->bias = a.post_bias || a.dpost_bias || a.dpre_bias;
    const int per_cu = 1024 / out->rl.threads, chip = 256 * (per_cu > 1 ? per_cu : 1);     // 16 waves of 128 registers on a CU
    const long long target = most > 0 && most < chip ? most : chip;
    p.cut = cut_rows(a, rpb, target, kMinSteps);
    // Neighbouring rows at a time keep the memory channels evenly busy (8192 x 4096 bf16: 97 us in runs, 90 in turn), but rows that share cache
    // lines then share them across blocks (7000 x 4507: 143 and 150), and with a gate per sample runs are faster (16 x 1024 x 2048: 105 and 110).
    p.in_turn = !by_sample && (long long)a.width * (a.dtype == FNET_F32 ? 4 : 2) % 128 == 0;
    const long long segments = (long long)p.cut.samples * p.cut.parts;
    out->blocks = (int)(segments < target ? segments : target);
    out->bytes = 0;
    const uint64_t want[SUM_COUNT] = {a.dpre_weight, a.dpre_bias, a.dpost_weight, a.dpost_bias, a.dscale, out->gm == GM_CONST ? a.dgate : 0};
    for (int s = 0; s < SUM_COUNT; ++s) {
        if (!want[s]) continue;
        const long long rows = s == SUM_GATE ? segments : out->blocks;
        if (s == SUM_GATE && by_sample ? p.cut.parts == 1 : rows == 1) {
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
    bwd_shape(a, L, E, 0, &s);
    FNET_CHECK_ARG(s.bytes == 0 || (a.workspace != 0 && a.workspace % 16 == 0 && a.workspace_bytes >= s.bytes));
    const int most = fnet_block_norm_bwd_resident<T, L, E>(s.rl, s.gm, s.bias, a.kind == FNET_NORM_LAYER);
    if (most < s.blocks) bwd_shape(a, L, E, most, &s);
    const int rc = fnet_block_norm_bwd_launch<T, L, E>(a, s.plan, s.rl, s.blocks, s.gm, s.bias, st);
    if (rc != FNET_OK) return rc;
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
        c.groups[c.count] = by_sample ? s.plan.cut.samples : 1;
        c.slots[c.count] = by_sample ? s.plan.cut.parts : s.blocks;
        c.f32[c.count] = (i == SUM_GATE ? a.gate_dtype : a.param_dtype) == FNET_F32;
        groups += c.groups[c.count++];
    }
    hipLaunchKernelGGL(k_block_norm_cols<T>, dim3((a.width + 63) / 64, groups), dim3(1024), 0, st, c);
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
    DISPATCH_ROW(host_args->width, { bwd_shape(as_launched(*host_args), L, E, 0, &s); });
    *bytes = s.bytes;
    return FNET_OK;
}

int fnet_block_norm_bwd(const FnetBlockNorm* host_args, void* stream) {
    const int rc = bwd_check(host_args);
    if (rc != FNET_OK) return rc;
    const FnetBlockNorm a = as_launched(*host_args);
    if (a.rows == 0) return FNET_OK;
    FNET_CHECK_ARG((!a.post && !a.dh) || a.stats != 0);
    FNET_CHECK_ARG(a.dh != 0 || (!a.dpre_weight && !a.dpre_bias));
    int out = FNET_OK;
    DISPATCH_T3(a.dtype, DISPATCH_ROW(a.width, { out = run_bwd<T, L, E>(a, (hipStream_t)stream); }));
    return out;
}
