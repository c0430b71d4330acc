// Shared by the forward and the backward of the norms around a residual block (fnet_block_norm.hip, fnet_block_norm_bwd.hip).
#pragma once
#include "fnet_vec.h"

// How rows lie on lanes.  A row belongs to L lanes (8 .. 1024) that hold it in registers from its one load to its last store, E elements
// each, in chunks of 16 bytes: lane l of a row holds chunks l, l + L, ...  Up to 64 lanes a row lies inside a wave (DPP sums, no barrier,
// 256 / L rows per block at a time); above that a block is one row.
template <typename T, int L, int E>
struct RowShape {
    static constexpr int V = VecOf<T>::V;                       // elements per chunk
    static constexpr int K = E / V;                             // chunks per lane
    static constexpr int THREADS = L > 64 ? L : 256;
    static constexpr int RPB = THREADS / L;                     // rows per block and step
};

// Sums of up to N values at once over the lanes of a row, in every one of them.  `red` (2 * N * W floats) has room for two rounds: a wave
// can be one round ahead of another, never two, so one barrier a round is enough.
template <int L, int N>
struct RowSum {
    static constexpr int W = L > 64 ? L / 64 : 1;
    float* red;
    int turn;
    __device__ __forceinline__ RowSum(float* r) : red(r), turn(0) {}
    template <int M>
    __device__ __forceinline__ void operator()(float (&v)[M]) {
        static_assert(M <= N, "the buffer holds N values");
#pragma unroll
        for (int i = 0; i < M; ++i) v[i] = lane_sum<(L > 64 ? 64 : L)>(v[i]);
        if (L > 64) {
            float* b = red + turn * (N * W);
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < M; ++i) b[i * W + (threadIdx.x >> 6)] = v[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < M; ++i) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < W; ++k) s += b[i * W + k];
                v[i] = s;
            }
        }
    }
};

// one chunk of a parameter (or gate) that is fp32 or of the operands' type
template <typename T>
__device__ __forceinline__ void load_param(uint64_t p, long long at, bool f32, int n, float* v) {
    constexpr int V = VecOf<T>::V;
    if (f32 && V == 8) {
        const float* q = gptr<const float>(p) + at;
        load_chunk<float>(q, n < 4 ? n : 4, v);
        if (n > 4) load_chunk<float>(q + 4, n - 4, v + 4);
        else v[4] = v[5] = v[6] = v[7] = 0.f;
    } else {
        load_chunk<T>(gptr<const T>(p) + at, n, v);
    }
}
template <typename T>
__device__ __forceinline__ float load_param1(uint64_t p, long long at, bool f32) {
    return f32 ? gptr<const float>(p)[at] : elem_to_f<T>(gptr<const T>(p)[at]);
}
template <typename T>
__device__ __forceinline__ void store_param(uint64_t p, long long at, bool f32, int n, const float* v) {
    if (f32 && VecOf<T>::V == 8) {
        float* q = gptr<float>(p) + at;
        store_chunk<float>(q, n < 4 ? n : 4, v);
        if (n > 4) store_chunk<float>(q + 4, n - 4, v + 4);
    } else {
        store_chunk<T>(gptr<T>(p) + at, n, v);
    }
}

// act(g) and its derivative.  Both derivatives are written with e = exp(-|g|) (or its square), which keeps them exact where act(g) is
// within a rounding of 1.
__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == FNET_GATE_SIGMOID) return 1.f / (1.f + __expf(-g));
    if (act == FNET_GATE_TANH) return tanhf(g);
    return g;
}
__device__ __forceinline__ float gate_slope(float g, int act) {
    if (act == FNET_GATE_SIGMOID) {
        const float e = __expf(-fabsf(g)), d = 1.f + e;
        return e / (d * d);
    }
    if (act == FNET_GATE_TANH) {
        const float e = __expf(-2.f * fabsf(g)), d = 1.f + e;
        return 4.f * e / (d * d);
    }
    return 1.f;
}

int fnet_block_norm_check(const FnetBlockNorm* a);        // the checks that both directions share

// L and E by the width: E = 8 elements per lane as long as a block of at most 1024 lanes covers the row, then 16.
#define DISPATCH_ROW(width, ...)                                                           \
    if ((width) <= 64) { constexpr int L = 8, E = 8; __VA_ARGS__; }                         \
    else if ((width) <= 128) { constexpr int L = 16, E = 8; __VA_ARGS__; }                  \
    else if ((width) <= 256) { constexpr int L = 32, E = 8; __VA_ARGS__; }                  \
    else if ((width) <= 512) { constexpr int L = 64, E = 8; __VA_ARGS__; }                  \
    else if ((width) <= 1024) { constexpr int L = 128, E = 8; __VA_ARGS__; }                \
    else if ((width) <= 2048) { constexpr int L = 256, E = 8; __VA_ARGS__; }                \
    else if ((width) <= 4096) { constexpr int L = 512, E = 8; __VA_ARGS__; }                \
    else if ((width) <= 8192) { constexpr int L = 1024, E = 8; __VA_ARGS__; }               \
    else { constexpr int L = 1024, E = 16; __VA_ARGS__; }
