// Vector access at any alignment and lane reductions for the row / list kernels (fnet_block_norm*.hip, fnet_tensor_list.hip).
#pragma once
#include <hip/hip_fp16.h>

#include "fnet_common.h"

// 16 bytes at a time whatever the address: rows of an odd width and gradients packed into one bucket start at any multiple of the element
// size.  The global memory path of gfx950 takes such addresses (the HSA target runs in unaligned-access mode), and with the element's own
// alignment declared here the compiler still emits one global_load_dwordx4 / global_store_dwordx4, so there is one code path for aligned
// and unaligned operands.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));

// An address that came as an integer, as a pointer to global memory: without the named address space every access through it would be a
// flat one, which also occupies the LDS counter.
template <typename T>
__device__ __forceinline__ T* gptr(uint64_t a) {
    return (T*)(__attribute__((address_space(1))) T*)a;
}

struct f16_t { uint16_t b; };      // raw fp16 bits (bf16_t is a plain uint16_t: the two must be different types)

template <typename T> struct VecOf;
template <> struct VecOf<float> { static constexpr int V = 4; typedef u32x4_a4 vec; };
template <> struct VecOf<bf16_t> { static constexpr int V = 8; typedef u32x4_a2 vec; };
template <> struct VecOf<f16_t> { static constexpr int V = 8; typedef u32x4_a2 vec; };

template <typename T> __device__ __forceinline__ float elem_to_f(T v);
template <> __device__ __forceinline__ float elem_to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float elem_to_f<bf16_t>(bf16_t v) { return bf2f(v); }
template <> __device__ __forceinline__ float elem_to_f<f16_t>(f16_t v) { return (float)__builtin_bit_cast(_Float16, v.b); }
template <typename T> __device__ __forceinline__ T f_to_elem(float v);          // round to nearest even
template <> __device__ __forceinline__ float f_to_elem<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t f_to_elem<bf16_t>(float v) { return f2bf(v); }
template <> __device__ __forceinline__ f16_t f_to_elem<f16_t>(float v) { return f16_t{__builtin_bit_cast(uint16_t, (_Float16)v)}; }

// the 16 bytes as loaded -> V floats, and back
template <typename T> __device__ __forceinline__ void unpack16(const u32x4& w, float* v);
template <> __device__ __forceinline__ void unpack16<float>(const u32x4& w, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
}
template <> __device__ __forceinline__ void unpack16<bf16_t>(const u32x4& w, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void unpack16<f16_t>(const u32x4& w, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[k] & 0xffffu));
        v[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[k] >> 16));
    }
}
template <typename T> __device__ __forceinline__ u32x4 pack16(const float* v);
template <> __device__ __forceinline__ u32x4 pack16<float>(const float* v) {
    return (u32x4){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <> __device__ __forceinline__ u32x4 pack16<bf16_t>(const float* v) {
    return (u32x4){f2bf_pk(v[0], v[1]), f2bf_pk(v[2], v[3]), f2bf_pk(v[4], v[5]), f2bf_pk(v[6], v[7])};
}
template <> __device__ __forceinline__ u32x4 pack16<f16_t>(const float* v) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * k + 1]) << 16);
    return w;
}

// n (1 .. V) leading elements of the 16-byte chunk at p; the rest reads as zero / is left alone
template <typename T>
__device__ __forceinline__ u32x4 load_raw(const T* p, int n) {
    constexpr int V = VecOf<T>::V;
    if (n >= V) return *reinterpret_cast<const typename VecOf<T>::vec*>(p);
    u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if (k >= n) break;
        if (V == 4) w[k] = reinterpret_cast<const uint32_t*>(p)[k];
        else w[k / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[k] << (16 * (k & 1));
    }
    return w;
}
template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, int n, float* v) { unpack16<T>(load_raw<T>(p, n), v); }
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, int n, const float* v) {
    constexpr int V = VecOf<T>::V;
    const u32x4 w = pack16<T>(v);
    if (n >= V) {
        *reinterpret_cast<typename VecOf<T>::vec*>(p) = w;
        return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if (k >= n) break;
        if (V == 4) reinterpret_cast<uint32_t*>(p)[k] = w[k];
        else reinterpret_cast<uint16_t*>(p)[k] = (uint16_t)(w[k / 2] >> (16 * (k & 1)));
    }
}

// The same for a chunk that ends a row of at least V elements: the 16 bytes that end where the row ends, and shift_row to move them down to
// the chunk's own place (one load and a dozen operations instead of a load per element).  Two steps, because the second has to wait for the
// first: a row's loads are all issued before any of them is shifted.
template <typename T>
__device__ __forceinline__ u32x4 load_row_end(const T* p, int n) {
    return *reinterpret_cast<const typename VecOf<T>::vec*>(p - (VecOf<T>::V - n));
}
template <typename T>
__device__ __forceinline__ void shift_row(u32x4& w, int n) {
    constexpr int V = VecOf<T>::V;
    const int s = V - n;                             // 0 for a whole chunk
    if (V == 8) {
        const u32x4 h = {__builtin_amdgcn_alignbit(w[1], w[0], 16), __builtin_amdgcn_alignbit(w[2], w[1], 16),
                         __builtin_amdgcn_alignbit(w[3], w[2], 16), w[3] >> 16};
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = (s & 1) ? h[k] : w[k];
    }
    const int d = V == 8 ? s >> 1 : s;               // in words
    const u32x4 one = {w[1], w[2], w[3], 0u};
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (d & 1) ? one[k] : w[k];
    const u32x4 two = {w[2], w[3], 0u, 0u};
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (d & 2) ? two[k] : w[k];
}

// Sum over groups of L consecutive lanes (L = 8 .. 64, a power of two), the result in every lane of the group.  Inside 16 lanes by DPP:
// quad_perm exchanges neighbours and pairs, and once a group of four (eight) holds one value the half mirror (mirror) exchanges groups.
// Above, row_bcast carries a 16-lane sum on and the group's last lane is read: no trip through the LDS.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp_f(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, ROWS, 0xf, ROWS == 0xf));
}
__device__ __forceinline__ float read_lane(float v, int lane) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
    v += dpp_f<0xB1>(v);                            // quad_perm [1,0,3,2]
    v += dpp_f<0x4E>(v);                            // quad_perm [2,3,0,1]
    v += dpp_f<0x141>(v);                           // row_half_mirror
    if (L >= 16) v += dpp_f<0x140>(v);              // row_mirror
    if (L >= 32) v += dpp_f<0x142, 0xa>(v);         // row_bcast15 into rows 1 and 3
    if (L >= 64) v += dpp_f<0x143, 0xc>(v);         // row_bcast31 into rows 2 and 3
    if (L == 32) return (threadIdx.x & 32) ? read_lane(v, 63) : read_lane(v, 31);
    if (L == 64) return read_lane(v, 63);
    return v;
}

#define DISPATCH_T3(dtype, ...)                                      \
    if ((dtype) == FNET_BF16) { using T = bf16_t; __VA_ARGS__; }      \
    else if ((dtype) == FNET_F32) { using T = float; __VA_ARGS__; }   \
    else if ((dtype) == FNET_F16) { using T = f16_t; __VA_ARGS__; }   \
    else return FNET_E_BADARG;
