// Shared by the forward and the backward of the norms around a residual block (fnet_block_norm*.hip).
#pragma once
#include <algorithm>

#include "fnet_vec.h"

// How rows lie on lanes.  A row is held in registers from its one load to its last store, E elements a lane in chunks of 16 bytes: lane l of
// a row holds chunks l, l + lanes, ...
//   L = 8 .. 64  that many lanes of one wave: sums stay inside the wave, no barrier, 256 / L rows per block at a time
//   L = 1        whole waves, as many as the row needs (2 .. 4, a number of the launch: a wide odd row leaves less than one wave idle), blocks
//                of 4 waves at most, so that the compiler may give a wave more than 128 registers
//   L = 0        the same with 5 .. 16 waves, one row to a block
// E = 8 covers 8192 elements with the 1024 lanes that a block has at most; wider rows take E = 16.
template <typename T, int L, int E>
struct RowShape {
    static constexpr int V = VecOf<T>::V;                       // elements per chunk
    static constexpr int K = E / V;                             // chunks per lane
    static constexpr int MAX_THREADS = L ? 256 : 1024;
    static constexpr bool WAVES = L < 8;
    static constexpr bool TINY = L == 8;                        // rows shorter than a chunk
    // rows of whole waves are the same for all lanes of a wave: their addresses stay in scalar registers
    static __device__ __forceinline__ long long row(long long r) {
        if (!WAVES && L != 64) return r;
        // r < 2^31 + 4: a block's last groups may lie behind the last row, so the 32 bits that are carried over are unsigned
        return (long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)r);
    }
    // a value per row, likewise (16 elements a lane: they spill as it is, and 4 to 27 registers go if a wide row's gate becomes a scalar)
    static __device__ __forceinline__ float row_value(float v) {
        if ((!WAVES && L != 64) || E > 8) return v;
        return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v)));
    }
};
struct RowLaunch {
    int waves;                   // per row (L = 0)
    int rpb;                     // rows per block and step
    int threads;
};
inline RowLaunch row_launch(int L, int E, int width) {
    if (L >= 8) return RowLaunch{1, 256 / L, 256};
    const int w = (width + 64 * E - 1) / (64 * E), r = w < 4 ? 4 / w : 1;
    return RowLaunch{w, r, 64 * w * r};
}

// How the rows are cut: segments = samples * parts, part p of a sample its rows [p * part_rows, (p + 1) * part_rows).  With a gate per sample
// a segment ends with its sample, so that what the gate multiplies is constant over it; otherwise all rows are one "sample".
struct RowCut {
    int samples, parts;          // their product: segments, at most 2^30 and the target
    long long sample_rows, part_rows;
};
// about `target` segments, each of at least min_steps steps of rpb rows where there are that many for 256 of them
inline RowCut cut_rows(const FnetBlockNorm& a, int rpb, long long target, int min_steps) {
    RowCut c;
    const bool by_sample = a.gate_kind == FNET_GATE_SAMPLE;
    c.samples = by_sample ? (int)(a.rows / a.tokens) : 1;
    c.sample_rows = by_sample ? a.tokens : a.rows;
    const long long steps = (c.sample_rows + rpb - 1) / rpb;
    long long parts = target / c.samples;
    const long long fill = std::min(steps, (255ll + c.samples) / c.samples);
    parts = std::min(parts, std::max(steps / min_steps, fill));
    if (parts < 1) parts = 1;
    c.part_rows = ((steps + parts - 1) / parts) * rpb;
    c.parts = (int)((c.sample_rows + c.part_rows - 1) / c.part_rows);
    return c;
}

// This thread's place: `lane` of row group `group`
template <int L>
struct RowPlace {
    int lane, group, lanes, waves;
    __device__ __forceinline__ RowPlace(const RowLaunch& r) {
        if (L >= 8) {
            lane = threadIdx.x % (L >= 8 ? L : 8);
            group = threadIdx.x / (L >= 8 ? L : 8);
            if (L == 64) group = __builtin_amdgcn_readfirstlane(group);
            lanes = L;
            waves = 1;
        } else {
            waves = r.waves;
            lanes = 64 * waves;
            group = __builtin_amdgcn_readfirstlane((int)threadIdx.x / lanes);
            lane = (int)threadIdx.x - group * lanes;
        }
    }
};

// Sums of up to N values at once over the lanes of a row, in every one of them.  With several waves to a row: each leaves its sums in the
// LDS and after one barrier every wave adds them up, 16 lanes reading 16 places.  `red` (SIZE floats) has room for two rounds: a
// wave can be one round ahead of another, never two, so one barrier a round is enough.  All threads of the block call it together.
template <int L, int N>
struct RowSum {
    static constexpr int PITCH = 16;                            // places per value: waves of a row times rows of a block
    static constexpr int SIZE = L < 8 ? 2 * N * PITCH : 1;
    float* red;
    int turn;
    __device__ __forceinline__ RowSum(float* r) : red(r), turn(0) {}
    template <int M>
    __device__ __forceinline__ void operator()(float (&v)[M], const RowPlace<L>& at) {
        static_assert(M <= N, "the buffer holds N values");
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] = lane_sum<(L < 8 ? 64 : L)>(v[i]);
        if (L < 8) {
            float* b = red + turn * (N * PITCH) + at.group * at.waves;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < M; ++i) b[i * PITCH + (at.lane >> 6)] = v[i];
            }
            __syncthreads();
            const int k = threadIdx.x & 15;
#pragma unroll
            for (int i = 0; i < M; ++i) v[i] = lane_sum<16>(k < at.waves ? b[i * PITCH + k] : 0.f);
        }
    }
};

// Mean and sum of squares about it of a row, for several waves to a row behind ONE barrier: each wave takes its own mean and its squares about
// that, and the waves' are joined as n_w (mean_w - mean)^2 + squares_w.  No difference of large numbers anywhere.  n: elements of wave
// (threadIdx.x & 15) of this row.  `red` as RowSum<L, 2>.
template <int L>
struct RowMoments {
    RowSum<L, 2>& sum;
    float inv_c, n_wave, inv_wave, n;
    __device__ __forceinline__ RowMoments(RowSum<L, 2>& s, const RowPlace<L>& at, int width, int V, int K) : sum(s), inv_c(1.f / (float)width) {
        auto elements = [&](int wave) {
            int c = 0;
            for (int k = 0; k < K; ++k) c += min(max(width - (k * at.lanes + 64 * wave) * V, 0), 64 * V);
            return (float)c;
        };
        n_wave = elements(at.lane >> 6);
        inv_wave = n_wave > 0.f ? 1.f / n_wave : 0.f;
        n = (int)(threadIdx.x & 15) < at.waves ? elements(threadIdx.x & 15) : 0.f;
    }
    // s: this lane's plain sum; squares(mean): this lane's sum of squares about a mean.  Returns the row's, in every lane.
    template <typename F>
    __device__ __forceinline__ float operator()(float s, F squares, float& mean, const RowPlace<L>& at) {
        if (L >= 8) {
            mean = lane_sum<(L >= 8 ? L : 64)>(s) * inv_c;
            return lane_sum<(L >= 8 ? L : 64)>(squares(mean));
        }
        const float m = lane_sum<64>(s) * inv_wave, q = lane_sum<64>(squares(m));
        float* b = sum.red + sum.turn * (2 * RowSum<L, 2>::PITCH) + at.group * at.waves;
        sum.turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
            b[at.lane >> 6] = m;
            b[RowSum<L, 2>::PITCH + (at.lane >> 6)] = q;
        }
        __syncthreads();
        const int k = threadIdx.x & 15;
        const float mk = k < at.waves ? b[k] : 0.f, qk = k < at.waves ? b[RowSum<L, 2>::PITCH + k] : 0.f;
        mean = lane_sum<16>(n * mk) * inv_c;
        const float d = mk - mean;
        return lane_sum<16>(fmaf(n * d, d, qk));
    }
};

// one chunk of a row, n elements of it (n > 0); TINY: the row may be shorter than a chunk.  align_row completes it.
template <typename T, bool TINY>
__device__ __forceinline__ u32x4 load_row(const T* p, int n) {
    return TINY ? load_raw<T>(p, n) : load_row_end<T>(p, n);
}
template <typename T, bool TINY>
__device__ __forceinline__ void align_row(u32x4& w, int n) {
    if (!TINY && n > 0) shift_row<T>(w, n);
}
// one chunk of a parameter (or gate) that is fp32 or of the operands' type
template <typename T, bool TINY>
__device__ __forceinline__ void load_param(uint64_t p, long long at, bool f32, int n, float* v) {
    if (f32 && VecOf<T>::V == 8) {
        const float* q = gptr<const float>(p) + at;
        u32x4 lo = load_row<float, TINY>(q, min(n, 4)), hi = {0u, 0u, 0u, 0u};
        if (n > 4) hi = load_row<float, TINY>(q + 4, n - 4);
        if (n < 8) {
            align_row<float, TINY>(lo, min(n, 4));
            align_row<float, TINY>(hi, n - 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(lo[i]);
            v[VecOf<T>::V - 4 + i] = __uint_as_float(hi[i]);
        }
    } else {
        u32x4 w = load_row<T, TINY>(gptr<const T>(p) + at, n);
        if (n < VecOf<T>::V) align_row<T, TINY>(w, n);
        unpack16<T>(w, v);
    }
}
// the same of a parameter that may be absent (then `absent`), and of a chunk that may lie behind the row (then zero)
template <typename T, bool TINY>
__device__ __forceinline__ void load_param_or(uint64_t p, long long at, bool f32, int n, float absent, float* v) {
#pragma unroll
    for (int i = 0; i < VecOf<T>::V; ++i) v[i] = p ? 0.f : absent;
    if (p && n > 0) load_param<T, TINY>(p, at, f32, n, v);
}
template <typename T>
__device__ __forceinline__ float load_param1(uint64_t p, long long at, bool f32) {
    return f32 ? gptr<const float>(p)[at] : elem_to_f<T>(gptr<const T>(p)[at]);
}
template <typename T>
__device__ __forceinline__ void store_param(uint64_t p, long long at, bool f32, int n, const float* v) {
    if (f32 && VecOf<T>::V == 8) {
        float* q = gptr<float>(p) + at;
        store_chunk<float>(q, n, v);
        if (n > 4) store_chunk<float>(q + 4, n - 4, v + 4);
    } else {
        store_chunk<T>(gptr<T>(p) + at, n, v);
    }
}

// act(g) and its derivative; the choices are uniform, so they stand outside the loops.  Both derivatives are written with e = exp(-|g|) (or its
// square), which keeps them exact where act(g) is within a rounding of 1.
// exp(v), v <= 0, in 32 bits: 2^n with n the rounded v / ln 2, and 1 + t for the rest t = v - n ln 2, with ln 2 in two parts (Cody and Waite's
// reduction, without the rounding to a whole n).  v_exp_f32 is good for one unit in the last place.  Below -200 the result is 0 all the same,
// and an infinity must not meet itself in t; a NaN passes the comparison.
__device__ __forceinline__ float gate_exp(float v) {
    v = v < -200.f ? -200.f : v;
    const float n = v * 1.44269504f, p = __builtin_amdgcn_exp2f(n), t = fmaf(n, 1.90465421e-9f, fmaf(n, -0.693147182f, v));
    return fmaf(p, t, p);
}
// 1 / d for d in 1 .. 4, one Newton step behind v_rcp_f32
__device__ __forceinline__ float gate_rcp(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.f), r, r);
}
// fp32 gates take these, and so do all gates per row (one value a row costs nothing).  Other 16-bit gates take the GPU's own power of two and
// reciprocal alone, whose rounded exponent is off by |g| 2^-24 (1e-6 of a sigmoid at -16): their gradient and the 16-bit outputs round that away,
// and a gate per element would pay for more (16 M bf16 elements with an fp32 gate each: backward 4 to 7 % slower this way).
__device__ __forceinline__ float gate_value(float g, int act, bool f32) {
    if (act == FNET_GATE_SIGMOID) {
        if (!f32) return __builtin_amdgcn_rcpf(1.f + __expf(-g));
        const float e = gate_exp(-fabsf(g)), r = gate_rcp(1.f + e);
        return g < 0.f ? e * r : r;
    }
    if (act == FNET_GATE_TANH) return tanhf(g);
    return g;
}
__device__ __forceinline__ float gate_slope(float g, int act, bool f32) {
    if (act == FNET_GATE_IDENTITY) return 1.f;
    const float v = act == FNET_GATE_SIGMOID ? -fabsf(g) : -2.f * fabsf(g), e = f32 ? gate_exp(v) : __expf(v), n = act == FNET_GATE_SIGMOID ? e : 4.f * e, d = 1.f + e;
    if (f32) return n * gate_rcp(d * d);
    const float r = __builtin_amdgcn_rcpf(d);
    return n * r * r;
}
// of a chunk
template <int V, bool F32>
__device__ __forceinline__ void gate_values_of(float* g, int act) {
    if (act == FNET_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = gate_value(g[i], FNET_GATE_SIGMOID, F32);
    } else if (act == FNET_GATE_TANH) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = gate_value(g[i], FNET_GATE_TANH, F32);
    }
}
template <int V, bool F32>
__device__ __forceinline__ void gate_slopes_of(float* g, int act) {
    if (act == FNET_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = gate_slope(g[i], FNET_GATE_SIGMOID, F32);
    } else if (act == FNET_GATE_TANH) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = gate_slope(g[i], FNET_GATE_TANH, F32);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = 1.f;
    }
}
// V = 4: the operands are fp32 and so is the gate
template <int V>
__device__ __forceinline__ void gate_values(float* g, int act, bool f32) {
    if (V == 4 || f32) gate_values_of<V, true>(g, act);
    else gate_values_of<V, false>(g, act);
}
template <int V>
__device__ __forceinline__ void gate_slopes(float* g, int act, bool f32) {
    if (V == 4 || f32) gate_slopes_of<V, true>(g, act);
    else gate_slopes_of<V, false>(g, act);
}

// How the gate enters a kernel: constant over a segment's rows (none, per channel, per sample: part of the weights), one value per row, or a
// row of values per row.  (The forward has a gate per sample in an instance of its own: weights that change on the way cost it registers
// that its waves in flight need.)
enum { GM_CONST = 0, GM_ROW = 1, GM_VECTOR = 2, GM_SAMPLE = 3 };

template <typename T, int L, int E>
int fnet_block_norm_fwd_launch(const FnetBlockNorm& a, hipStream_t st);

// Blocks of a kernel that the GPU holds at once, asked once per kernel, block and LDS size; what the kernel was compiled for if it cannot say
int fnet_resident_blocks(const void* kernel, int threads, size_t lds, int otherwise);
int fnet_block_norm_check(const FnetBlockNorm* a);        // the checks that both directions share

#define DISPATCH_ROW(width, ...)                                                   \
    if ((width) <= 64) { constexpr int L = 8, E = 8; __VA_ARGS__; }                 \
    else if ((width) <= 128) { constexpr int L = 16, E = 8; __VA_ARGS__; }          \
    else if ((width) <= 256) { constexpr int L = 32, E = 8; __VA_ARGS__; }          \
    else if ((width) <= 512) { constexpr int L = 64, E = 8; __VA_ARGS__; }          \
    else if ((width) <= 2048) { constexpr int L = 1, E = 8; __VA_ARGS__; }         \
    else if ((width) <= 8192) { constexpr int L = 0, E = 8; __VA_ARGS__; }          \
    else { constexpr int L = 0, E = 16; __VA_ARGS__; }
// the same list, for the instances
#define FNET_BLOCK_NORM_INSTANCES_OF(X, T) X(T, 8, 8) X(T, 16, 8) X(T, 32, 8) X(T, 64, 8) X(T, 1, 8) X(T, 0, 8) X(T, 0, 16)
#define FNET_BLOCK_NORM_INSTANCES(T)                              \
    FNET_BLOCK_NORM_INSTANCES_OF(FNET_BLOCK_NORM_FWD_INSTANCE, T) \
    FNET_BLOCK_NORM_INSTANCES_OF(FNET_BLOCK_NORM_BWD_INSTANCE, T)
