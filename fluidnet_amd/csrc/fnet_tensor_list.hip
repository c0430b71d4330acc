// The global norm of a list of tensors, their clipping in place, and one Adam step of a list of parameters on the clipped gradients.
// What k_grad_norm / k_adam (fnet_optim.hip) do for the UNet's one flat fp32 buffer, for any number of separate tensors of three types.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "fnet_vec.h"

namespace {

constexpr int kThreads = 256;
// Every launch carries its part of the list as a kernel argument (below 4 KB): nothing is uploaded, so there is no table whose lifetime a
// captured graph or another stream could outlive.
constexpr int kTab = 240, kAdamTab = 96, kMasterTab = 80;
constexpr long long kMaxEntry = 1ll << 29;       // a longer tensor takes several entries
constexpr int kMaxBlocks = 2048;                 // eight blocks of four waves per CU, and as many partial sums of all dense tensors together

constexpr uint32_t kCount = (1u << 30) - 1;
enum { NORM_2 = 0, NORM_1 = 1, NORM_INF = 2 };

struct ListTab {
    uint64_t p[kTab];
    uint32_t n[kTab];            // elements, and the type from bit 30 on
    uint32_t first[kTab];        // index of the entry's first chunk in this launch
    int count;
    uint32_t chunks;
};
struct AdamTab {                  // of fp32 parameters, which are their own masters
    uint64_t p[kAdamTab], g[kAdamTab], m[kAdamTab], v[kAdamTab];
    uint32_t n[kAdamTab], first[kAdamTab];
    int count;
    uint32_t chunks;
    static constexpr int SIZE = kAdamTab;
    __host__ __device__ uint64_t& master(int j) { return p[j]; }
    __host__ __device__ uint64_t master(int j) const { return p[j]; }
};
struct MasterTab {
    uint64_t p[kMasterTab], g[kMasterTab], m[kMasterTab], v[kMasterTab], w[kMasterTab];
    uint32_t n[kMasterTab], first[kMasterTab];
    int count;
    uint32_t chunks;
    static constexpr int SIZE = kMasterTab;
    __host__ __device__ uint64_t& master(int j) { return w[j]; }
    __host__ __device__ uint64_t master(int j) const { return w[j]; }
};
static_assert(sizeof(ListTab) <= 3904 && sizeof(AdamTab) <= 3904 && sizeof(MasterTab) <= 3904, "the table and the other arguments must fit 4 KB");

// the entry that chunk c belongs to: every lane looks at one entry, 64 per step (a scan by one lane would be a chain of dependent loads)
template <typename TAB>
__device__ __forceinline__ int find_entry(const TAB& t, uint32_t c) {
    const int lane = threadIdx.x & 63;
    int j = 0;
    for (int base = 0; base < t.count; base += 64) {
        const int k = base + lane;
        const bool le = k < t.count && t.first[k < t.count ? k : 0] <= c;
        const int s = __popcll(__ballot(le));
        j += s;
        if (s < 64) break;
    }
    return __builtin_amdgcn_readfirstlane(j - 1);
}

// the last of this block's chunks blockIdx.x, blockIdx.x + gridDim.x, ... (negative if there is none)
__device__ __forceinline__ long long last_chunk(uint32_t chunks) {
    return blockIdx.x < chunks ? (long long)((chunks - 1 - blockIdx.x) / gridDim.x) * gridDim.x + blockIdx.x : -1;
}

// ---- the norm: partial sums in 64 bits (a sum of squares in 32 overflows at |g| = 1.8e19 and loses the small gradients of a long list)
template <int KIND>
__device__ __forceinline__ void norm_add(double& acc, uint32_t& mx, float v) {
    if (KIND == NORM_2) acc = fma((double)v, (double)v, acc);
    else if (KIND == NORM_1) acc += (double)fabsf(v);
    else mx = max(mx, __float_as_uint(v) & 0x7fffffffu);      // as bits, so that a NaN is larger than everything and stays
}
template <int KIND>
__device__ __forceinline__ double norm_join(double a, double b) {
    if (KIND != NORM_INF) return a + b;
    return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b)));
}
// over the block, the result in every thread.  Fixed order: the same list gives the same bits.
template <int KIND>
__device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = norm_join<KIND>(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = norm_join<KIND>(norm_join<KIND>(red[0], red[1]), norm_join<KIND>(red[2], red[3]));
    __syncthreads();
    return v;
}
template <int KIND>
__device__ __forceinline__ double norm_of(double s) { return KIND == NORM_2 ? sqrt(s) : s; }

__device__ __forceinline__ void advance_clock(double* clock, double b1, double b2) {
    clock[0] += 1.0;
    clock[1] *= b1;
    clock[2] *= b2;
}

constexpr int kNormVecs = 8;                      // 16-byte loads per lane and chunk
template <typename T> __host__ __device__ constexpr uint32_t norm_chunk() { return (uint32_t)kThreads * VecOf<T>::V * kNormVecs; }

// f(T()); with T = void for the type of an entry, which is the same for the whole block.  A list of several types goes through kernels of that
// kind, all types in one launch (41 tensors of two types: 27 us with a launch per type, 20 so); a list of one type through its own, which
// are faster (403 M bf16: 395 us and 437).
template <typename T, typename F>
__device__ __forceinline__ void of_type(uint32_t n_and_type, F f) {
    if constexpr (!std::is_void<T>::value) f(T());
    else if (n_and_type >> 30 == FNET_F32) f(float());
    else if (n_and_type >> 30 == FNET_BF16) f(bf16_t());
    else f(f16_t());
}

template <typename LIST, int KIND>
__global__ __launch_bounds__(256) void k_list_norm(ListTab t, double* partials, double* clock, double b1, double b2) {
    __shared__ double red[4];
    if (clock && blockIdx.x == 0 && threadIdx.x == 0) advance_clock(clock, b1, b2);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    uint32_t mx = 0;
    for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int j = find_entry(t, c);
        of_type<LIST>(t.n[j], [&](auto type) {
            using T = decltype(type);
            constexpr int V = VecOf<T>::V;
            const uint32_t n = t.n[j] & kCount, at = (c - t.first[j]) * norm_chunk<T>();
            const T* p = gptr<const T>(t.p[j]) + at;
            const uint32_t left = n - at;
            if (left >= norm_chunk<T>()) {
                u32x4 w[kNormVecs];
#pragma unroll
                for (int k = 0; k < kNormVecs; ++k) w[k] = *reinterpret_cast<const typename VecOf<T>::vec*>(p + (k * kThreads + threadIdx.x) * V);
#pragma unroll
                for (int k = 0; k < kNormVecs; ++k) {
                    float v[V];
                    unpack16<T>(w[k], v);
#pragma unroll
                    for (int i = 0; i < V; ++i) norm_add<KIND>(acc[i & 3], mx, v[i]);
                }
            } else {
                for (uint32_t o = threadIdx.x * V; o < left; o += kThreads * V) {
                    float v[V];
                    load_chunk<T>(p + o, (int)min(left - o, (uint32_t)V), v);
#pragma unroll
                    for (int i = 0; i < V; ++i) norm_add<KIND>(acc[i & 3], mx, v[i]);
                }
            }
        });
    }
    const double mine = KIND == NORM_INF ? (double)__uint_as_float(mx) : (acc[0] + acc[1]) + (acc[2] + acc[3]);
    const double s = block_join<KIND>(mine, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// All partial sums, by every block of the consumer, for one launch less: about 16 KB out of the L2 for dense tensors.  Each strided one adds
// up to 256 (2 KB), and each has a launch of its own whose blocks read them all again: 100 slices of 64 x 100 take 0.8 ms, 1000 take 17.
template <int KIND>
__device__ __forceinline__ double total_norm(const double* partials, int n, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) v = norm_join<KIND>(v, partials[i]);
    return norm_of<KIND>(block_join<KIND>(v, red));
}
// min(1, max_norm / (norm + 1e-6)) as torch computes it: NaN stays NaN, an infinite norm gives 0
__device__ __forceinline__ float clip_coef(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c >= 1.0 ? 1.f : (float)c;
}

template <int KIND>
__global__ __launch_bounds__(256) void k_list_norm_finish(const double* partials, int n, float* out) {
    __shared__ double red[4];
    const double s = total_norm<KIND>(partials, n, red);
    if (threadIdx.x == 0) *out = (float)s;
}

// ---- clipping in place.  A coefficient of 1 leaves every gradient as it is, so nothing is read or written.
struct ClipFrom {
    const double* partials;      // or null:
    const float* norm;           // the norm is given
    int n_partials, kind;
    double max_norm;
    float* norm_out;             // written by the first block of the first launch
};
__device__ __forceinline__ float coef_of(const ClipFrom& f, double* red) {
    double s;
    if (!f.partials) s = (double)*f.norm;
    else if (f.kind == NORM_2) s = total_norm<NORM_2>(f.partials, f.n_partials, red);
    else if (f.kind == NORM_1) s = total_norm<NORM_1>(f.partials, f.n_partials, red);
    else s = total_norm<NORM_INF>(f.partials, f.n_partials, red);
    if (f.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *f.norm_out = (float)s;
    return clip_coef(s, f.max_norm);
}

template <typename LIST>
__global__ __launch_bounds__(256) void k_list_scale(ListTab t, ClipFrom f) {
    __shared__ double red[4];
    const float coef = coef_of(f, red);
    if (coef == 1.f) return;
    // Each block goes back over the chunks that it had in the norm: they are in its own L2 where they fit, and of a longer list what was read
    // last is still in the cache in front of the memory (403 M bf16: 273 us forwards, 271 back, and the next norm 5 us less).
    for (long long c = last_chunk(t.chunks); c >= 0; c -= gridDim.x) {
        const int j = find_entry(t, (uint32_t)c);
        of_type<LIST>(t.n[j], [&](auto type) {
            using T = decltype(type);
            constexpr int V = VecOf<T>::V;
            const uint32_t n = t.n[j] & kCount, at = ((uint32_t)c - t.first[j]) * norm_chunk<T>();
            T* p = gptr<T>(t.p[j]) + at;
            const uint32_t left = n - at;
            if (left >= norm_chunk<T>()) {
                u32x4 w[kNormVecs];
#pragma unroll
                for (int k = 0; k < kNormVecs; ++k) w[k] = *reinterpret_cast<const typename VecOf<T>::vec*>(p + (k * kThreads + threadIdx.x) * V);
#pragma unroll
                for (int k = 0; k < kNormVecs; ++k) {
                    float v[V];
                    unpack16<T>(w[k], v);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] *= coef;        // in 32 bits, rounded once
                    *reinterpret_cast<typename VecOf<T>::vec*>(p + (k * kThreads + threadIdx.x) * V) = pack16<T>(v);
                }
            } else {
                for (uint32_t o = threadIdx.x * V; o < left; o += kThreads * V) {
                    float v[V];
                    const int m = (int)min(left - o, (uint32_t)V);
                    load_chunk<T>(p + o, m, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] *= coef;
                    store_chunk<T>(p + o, m, v);
                }
            }
        });
    }
}

// ---- tensors that are no dense block of memory (a gradient that is a slice of a larger buffer): one launch each, one element per lane, its
// address by a 64-bit division per axis (a 4096 x 1024 fp32 slice of a 4096 x 2560 buffer: 46 us to clip, 15 for a dense one)
struct Strided {
    uint64_t p;
    long long n;
    int ndim;
    long long size[FNET_LIST_MAXDIM], stride[FNET_LIST_MAXDIM];
};
__device__ __forceinline__ long long strided_at(const Strided& s, long long i) {
    long long o = 0;
    for (int d = s.ndim - 1; d > 0; --d) {
        const long long q = i / s.size[d];
        o += (i - q * s.size[d]) * s.stride[d];
        i = q;
    }
    return o + i * s.stride[0];
}
template <typename T, int KIND>
__global__ __launch_bounds__(256) void k_strided_norm(Strided s, double* partials, double* clock, double b1, double b2) {
    __shared__ double red[4];
    if (clock && blockIdx.x == 0 && threadIdx.x == 0) advance_clock(clock, b1, b2);
    double acc = 0.0;
    uint32_t mx = 0;
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < s.n; i += (long long)gridDim.x * kThreads)
        norm_add<KIND>(acc, mx, elem_to_f<T>(gptr<const T>(s.p)[strided_at(s, i)]));
    const double r = block_join<KIND>(KIND == NORM_INF ? (double)__uint_as_float(mx) : acc, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = r;
}
template <typename T>
__global__ __launch_bounds__(256) void k_strided_scale(Strided s, ClipFrom f) {
    __shared__ double red[4];
    const float coef = coef_of(f, red);
    if (coef == 1.f) return;
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < s.n; i += (long long)gridDim.x * kThreads) {
        T* p = gptr<T>(s.p) + strided_at(s, i);
        *p = f_to_elem<T>(elem_to_f<T>(*p) * coef);
    }
}

__global__ void k_clock_advance(double* clock, double b1, double b2) { advance_clock(clock, b1, b2); }

// ---- Adam.  gc = coef g;  m = b1 m + (1 - b1) gc;  v = b2 v + (1 - b2) gc^2;
// w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps).  The clipped gradient is never written.  Moments and the
// updated weight are 32-bit; a 16-bit parameter has a 32-bit master w (an update of lr is lost in a 16-bit weight more than 2^8 (bf16)
// times as large) and p is its rounding.  t and the betas' powers are on the device, so that a captured step goes on counting when replayed.
struct AdamArgs {
    ClipFrom f;
    int clip;
    const double* clock;         // t, b1^t, b2^t
    const double* lr_dev;        // or null: lr
    double lr, wd;
    float b1, b2, omb1, omb2, eps;
};
constexpr int kAdamVecs = 2;                      // groups of eight elements per lane and chunk
constexpr uint32_t kAdamChunk = kThreads * 8 * kAdamVecs;

struct AdamCoef { float coef, step, root, keep; };

__device__ __forceinline__ float adam_elem(const AdamArgs& a, const AdamCoef& k, float g, float& m, float& v, float w) {
    const float gc = g * k.coef;
    m = fmaf(a.b1, m, a.omb1 * gc);
    v = fmaf(a.b2, v, a.omb2 * gc * gc);
    float n = fmaf(w, k.keep, -k.step * m / (sqrtf(v) / k.root + a.eps));
    // a value of its own, so that the parameter is the rounding of the master as stored: the compiler otherwise computes an fp16 parameter
    // a second time with v_fma_mixlo_f16, which rounds the unrounded sum, and the two differ in ties
    asm("" : "+v"(n));
    return n;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
    load_chunk<T>(p, VecOf<T>::V, v);
    if (VecOf<T>::V == 4) load_chunk<T>(p + 4, 4, v + (VecOf<T>::V == 4 ? 4 : 0));
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
    store_chunk<T>(p, VecOf<T>::V, v);
    if (VecOf<T>::V == 4) store_chunk<T>(p + 4, 4, v + (VecOf<T>::V == 4 ? 4 : 0));
}

// MasterTab: w is a buffer of its own and p (type T) its rounding; otherwise T is float and p is the weight
template <typename T, typename TAB>
__global__ __launch_bounds__(256) void k_list_adam(TAB t, AdamArgs a) {
    constexpr bool MASTER = !std::is_same<TAB, AdamTab>::value;
    __shared__ double red[4];
    AdamCoef k;
    k.coef = a.clip ? coef_of(a.f, red) : 1.f;
    {
        const double lr = a.lr_dev ? *a.lr_dev : a.lr;
        k.step = (float)(lr / (1.0 - a.clock[1]));
        k.root = (float)sqrt(1.0 - a.clock[2]);
        k.keep = (float)(1.0 - lr * a.wd);
    }
    for (long long c = last_chunk(t.chunks); c >= 0; c -= gridDim.x) {
        const int j = find_entry(t, (uint32_t)c);
        const uint32_t n = t.n[j], at = ((uint32_t)c - t.first[j]) * kAdamChunk;
        const T* G = gptr<const T>(t.g[j]);
        T* P = gptr<T>(t.p[j]);
        float *M = gptr<float>(t.m[j]), *S = gptr<float>(t.v[j]);
        float* W = gptr<float>(t.master(j));
#pragma unroll
        for (int q = 0; q < kAdamVecs; ++q) {
            const uint32_t o = at + (q * kThreads + threadIdx.x) * 8;
            if (o + 8 <= n) {
                float g[8], m[8], v[8], w[8];
                load8<T>(G + o, g);
                load8<float>(M + o, m);
                load8<float>(S + o, v);
                load8<float>(W + o, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = adam_elem(a, k, g[i], m[i], v[i], w[i]);
                store8<float>(M + o, m);
                store8<float>(S + o, v);
                store8<float>(W + o, w);
                if (MASTER) store8<T>(P + o, w);
            } else {
                for (uint32_t i = o; i < n; ++i) {
                    float m = M[i], v = S[i];
                    const float w = adam_elem(a, k, elem_to_f<T>(G[i]), m, v, W[i]);
                    M[i] = m;
                    S[i] = v;
                    W[i] = w;
                    if (MASTER) P[i] = f_to_elem<T>(w);
                }
            }
        }
    }
}

int elem_size(int dtype) { return dtype == FNET_F32 ? 4 : 2; }
bool dtype_ok(int d) { return d == FNET_F32 || d == FNET_BF16 || d == FNET_F16; }

struct Span { uint64_t lo, hi; };
int apart(Span* s, int m) {
    std::sort(s, s + m, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    for (int k = 1; k < m; ++k)
        if (s[k].lo < s[k - 1].hi) return FNET_E_OVERLAP;
    return FNET_OK;
}
// two dense tensors that share memory would be scaled by two blocks at once
int check_apart(int n, const uint64_t* ptr, const int64_t* numel, const int32_t* dtype) {
    uint64_t end = 0;
    bool sorted = true;
    for (int k = 0; k < n && sorted; ++k) {
        if (numel[k] == 0) continue;
        if (ptr[k] < end) sorted = false;
        end = ptr[k] + (uint64_t)numel[k] * elem_size(dtype[k]);
    }
    if (sorted) return FNET_OK;
    Span* s = (Span*)malloc(sizeof(Span) * (size_t)n);
    if (!s) return FNET_E_HIP;
    int m = 0;
    for (int k = 0; k < n; ++k)
        if (numel[k]) s[m++] = Span{ptr[k], ptr[k] + (uint64_t)numel[k] * elem_size(dtype[k])};
    const int rc = apart(s, m);
    free(s);
    return rc;
}

int check_dense(int n, const uint64_t* ptr, const int64_t* numel, const int32_t* dtype) {
    FNET_CHECK_ARG(n >= 0 && (n == 0 || (ptr && numel && dtype)));
    for (int k = 0; k < n; ++k) {
        FNET_CHECK_ARG(dtype_ok(dtype[k]) && numel[k] >= 0 && numel[k] < (1ll << 46));
        FNET_CHECK_ARG(numel[k] == 0 || (ptr[k] != 0 && ptr[k] % elem_size(dtype[k]) == 0));
    }
    return FNET_OK;
}
int check_strided(int n, const FnetStridedTensor* s) {
    FNET_CHECK_ARG(n >= 0 && (n == 0 || s));
    for (int k = 0; k < n; ++k) {
        FNET_CHECK_ARG(dtype_ok(s[k].dtype) && s[k].ptr && s[k].ptr % elem_size(s[k].dtype) == 0 && s[k].ndim >= 1 && s[k].ndim <= FNET_LIST_MAXDIM);
        for (int d = 0; d < s[k].ndim; ++d) FNET_CHECK_ARG(s[k].size[d] > 0 && s[k].stride[d] > 0);
    }
    return FNET_OK;
}
Strided to_strided(const FnetStridedTensor& s) {
    Strided r;
    r.p = s.ptr;
    r.ndim = s.ndim;
    r.n = 1;
    for (int d = 0; d < FNET_LIST_MAXDIM; ++d) {
        r.size[d] = d < s.ndim ? s.size[d] : 1;
        r.stride[d] = d < s.ndim ? s.stride[d] : 0;
        r.n *= r.size[d];
    }
    return r;
}
unsigned strided_blocks(const Strided& s) { return (unsigned)std::min<long long>((s.n + kThreads - 1) / kThreads, 256); }

uint32_t chunk_of(int dtype) { return dtype == FNET_F32 ? norm_chunk<float>() : norm_chunk<bf16_t>(); }

// calls launch(table) for every table of at most kTab entries; 0 or the first error
template <typename F>
int for_tables(int n, const uint64_t* ptr, const int64_t* numel, const int32_t* dtype, F launch) {
    ListTab t;
    t.count = 0;
    t.chunks = 0;
    for (int k = 0; k < n; ++k) {
        const uint32_t chunk = chunk_of(dtype[k]);
        for (int64_t at = 0; at < numel[k]; at += kMaxEntry) {
            const uint32_t len = (uint32_t)std::min<int64_t>(numel[k] - at, kMaxEntry);
            t.p[t.count] = ptr[k] + (uint64_t)at * elem_size(dtype[k]);
            t.n[t.count] = len | (uint32_t)dtype[k] << 30;
            t.first[t.count] = t.chunks;
            t.chunks += (len + chunk - 1) / chunk;
            if (++t.count == kTab) {
                const int rc = launch(t);
                if (rc != FNET_OK) return rc;
                t.count = 0;
                t.chunks = 0;
            }
        }
    }
    return t.count ? launch(t) : FNET_OK;
}

// the type of a list's tensors, -1 for several
int list_type(int n, const int32_t* dtype) {
    for (int k = 1; k < n; ++k)
        if (dtype[k] != dtype[0]) return -1;
    return n ? dtype[0] : -1;
}
#define DISPATCH_LIST(type, ...)                                       \
    if ((type) < 0) { using LIST = void; __VA_ARGS__; }                \
    else { DISPATCH_T3(type, { using LIST = T; __VA_ARGS__; }) }

#define DISPATCH_KIND(kind, ...)                                                                  \
    if ((kind) == NORM_2) { constexpr int KIND = NORM_2; __VA_ARGS__; }                            \
    else if ((kind) == NORM_1) { constexpr int KIND = NORM_1; __VA_ARGS__; }                       \
    else { constexpr int KIND = NORM_INF; __VA_ARGS__; }

}  // namespace

int fnet_list_norm_partials(int32_t n, const uint64_t* host_ptr, const int64_t* host_numel, const int32_t* host_dtype, int32_t n_strided,
                            const FnetStridedTensor* host_strided, int32_t norm_kind, double* partials, int32_t capacity,
                            int32_t* n_partials, double* clock, double beta1, double beta2, void* stream) {
    int rc = check_dense(n, host_ptr, host_numel, host_dtype);
    if (rc == FNET_OK) rc = check_strided(n_strided, host_strided);
    if (rc != FNET_OK) return rc;
    FNET_CHECK_ARG(norm_kind >= NORM_2 && norm_kind <= NORM_INF && partials && n_partials);
    long long total = 0;
    for (int k = 0; k < n; ++k) total += (host_numel[k] + chunk_of(host_dtype[k]) - 1) / chunk_of(host_dtype[k]);
    hipStream_t st = (hipStream_t)stream;
    // what the launches will use is known before the first of them: nothing is launched if the workspace is too small
    auto blocks_of = [&](const ListTab& t) { return (unsigned)std::max<long long>(1, std::min<long long>(t.chunks, (long long)kMaxBlocks * t.chunks / std::max(total, 1ll))); };
    long long need = 0;
    for_tables(n, host_ptr, host_numel, host_dtype, [&](const ListTab& t) { need += blocks_of(t); return FNET_OK; });
    for (int k = 0; k < n_strided; ++k) need += strided_blocks(to_strided(host_strided[k]));
    FNET_CHECK_ARG(need <= capacity);
    int used = 0;
    const int type = list_type(n, host_dtype);
    rc = for_tables(n, host_ptr, host_numel, host_dtype, [&](const ListTab& t) -> int {
        const unsigned b = blocks_of(t);
        double* clk = used == 0 ? clock : nullptr;
        DISPATCH_LIST(type, DISPATCH_KIND(norm_kind, hipLaunchKernelGGL((k_list_norm<LIST, KIND>), dim3(b), dim3(kThreads), 0, st, t, partials + used, clk, beta1, beta2)));
        FNET_LAUNCH_CHECK();
        used += b;
        return FNET_OK;
    });
    if (rc != FNET_OK) return rc;
    for (int k = 0; k < n_strided; ++k) {
        const Strided s = to_strided(host_strided[k]);
        double* clk = used == 0 ? clock : nullptr;
        DISPATCH_T3(host_strided[k].dtype, DISPATCH_KIND(norm_kind, hipLaunchKernelGGL((k_strided_norm<T, KIND>), dim3(strided_blocks(s)), dim3(kThreads), 0, st, s,
                                                                                        partials + used, clk, beta1, beta2)));
        FNET_LAUNCH_CHECK();
        used += strided_blocks(s);
    }
    if (used == 0 && clock) {
        hipLaunchKernelGGL(k_clock_advance, dim3(1), dim3(1), 0, st, clock, beta1, beta2);
        FNET_LAUNCH_CHECK();
    }
    *n_partials = used;
    return FNET_OK;
}

int fnet_list_clock(double* clock, double beta1, double beta2, void* stream) {
    FNET_CHECK_ARG(clock);
    hipLaunchKernelGGL(k_clock_advance, dim3(1), dim3(1), 0, (hipStream_t)stream, clock, beta1, beta2);
    FNET_LAUNCH_CHECK();
    return FNET_OK;
}

int fnet_list_norm_finish(const double* partials, int32_t n_partials, int32_t norm_kind, float* norm_out, void* stream) {
    FNET_CHECK_ARG(partials && n_partials >= 0 && norm_out && norm_kind >= NORM_2 && norm_kind <= NORM_INF);
    DISPATCH_KIND(norm_kind, hipLaunchKernelGGL(k_list_norm_finish<KIND>, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, partials, n_partials, norm_out));
    FNET_LAUNCH_CHECK();
    return FNET_OK;
}

int fnet_list_scale(int32_t n, const uint64_t* host_ptr, const int64_t* host_numel, const int32_t* host_dtype, int32_t n_strided,
                    const FnetStridedTensor* host_strided, const double* partials, int32_t n_partials, int32_t norm_kind, const float* norm,
                    double max_norm, float* norm_out, void* stream) {
    int rc = check_dense(n, host_ptr, host_numel, host_dtype);
    if (rc == FNET_OK) rc = check_strided(n_strided, host_strided);
    if (rc == FNET_OK) rc = check_apart(n, host_ptr, host_numel, host_dtype);
    if (rc != FNET_OK) return rc;
    FNET_CHECK_ARG((partials != nullptr) != (norm != nullptr) && (!partials || n_partials >= 0));
    FNET_CHECK_ARG(norm_kind >= NORM_2 && norm_kind <= NORM_INF && max_norm >= 0.0);
    ClipFrom f{partials, norm, n_partials, norm_kind, max_norm, norm_out};
    hipStream_t st = (hipStream_t)stream;
    const int type = list_type(n, host_dtype);
    rc = for_tables(n, host_ptr, host_numel, host_dtype, [&](const ListTab& t) -> int {
        DISPATCH_LIST(type, hipLaunchKernelGGL(k_list_scale<LIST>, dim3(std::min<uint32_t>(t.chunks, kMaxBlocks)), dim3(kThreads), 0, st, t, f));
        FNET_LAUNCH_CHECK();
        f.norm_out = nullptr;
        return FNET_OK;
    });
    if (rc != FNET_OK) return rc;
    for (int k = 0; k < n_strided; ++k) {
        const Strided s = to_strided(host_strided[k]);
        DISPATCH_T3(host_strided[k].dtype, hipLaunchKernelGGL(k_strided_scale<T>, dim3(strided_blocks(s)), dim3(kThreads), 0, st, s, f));
        FNET_LAUNCH_CHECK();
        f.norm_out = nullptr;
    }
    if (f.norm_out) {                                // nothing to scale: one block stores the norm
        ListTab t;
        t.count = 0;
        t.chunks = 0;
        hipLaunchKernelGGL(k_list_scale<float>, dim3(1), dim3(kThreads), 0, st, t, f);
        FNET_LAUNCH_CHECK();
    }
    return FNET_OK;
}

int fnet_list_adam(int32_t n, const uint64_t* host_param, const uint64_t* host_grad, const uint64_t* host_exp_avg, const uint64_t* host_exp_avg_sq,
                   const uint64_t* host_master, const int64_t* host_numel, const int32_t* host_dtype, const FnetAdamList* h, void* stream) {
    FNET_CHECK_ARG(h && n > 0 && host_param && host_grad && host_exp_avg && host_exp_avg_sq && host_numel && host_dtype);
    int rc = check_dense(n, host_param, host_numel, host_dtype);
    if (rc == FNET_OK) rc = check_dense(n, host_grad, host_numel, host_dtype);
    if (rc != FNET_OK) return rc;
    FNET_CHECK_ARG(h->clock && (h->max_norm < 0.0 || (h->partials && h->capacity >= 0)));
    FNET_CHECK_ARG(h->beta1 >= 0.0 && h->beta1 < 1.0 && h->beta2 >= 0.0 && h->beta2 < 1.0 && h->eps >= 0.0 && h->weight_decay >= 0.0);
    FNET_CHECK_ARG(std::isfinite(h->lr) && std::isfinite(h->weight_decay) && std::isfinite(h->eps) && !std::isnan(h->max_norm));
    for (int k = 0; k < n; ++k) {
        if (host_numel[k] == 0) continue;
        FNET_CHECK_ARG(host_exp_avg[k] && host_exp_avg_sq[k] && host_exp_avg[k] % 4 == 0 && host_exp_avg_sq[k] % 4 == 0);
        FNET_CHECK_ARG(host_dtype[k] == FNET_F32 || (host_master && host_master[k] && host_master[k] % 4 == 0));
    }
    // everything that is written must lie apart, and no gradient in it (gradients are only read: they may share memory among themselves)
    Span* spans = (Span*)malloc(sizeof(Span) * 4 * (size_t)n);
    if (!spans) return FNET_E_HIP;
    int m = 0;
    for (int k = 0; k < n; ++k) {
        if (host_numel[k] == 0) continue;
        const uint64_t bytes = (uint64_t)host_numel[k] * 4;
        spans[m++] = Span{host_param[k], host_param[k] + (uint64_t)host_numel[k] * elem_size(host_dtype[k])};
        spans[m++] = Span{host_exp_avg[k], host_exp_avg[k] + bytes};
        spans[m++] = Span{host_exp_avg_sq[k], host_exp_avg_sq[k] + bytes};
        if (host_dtype[k] != FNET_F32) spans[m++] = Span{host_master[k], host_master[k] + bytes};
    }
    rc = apart(spans, m);
    for (int k = 0; k < n && rc == FNET_OK; ++k) {
        const uint64_t lo = host_grad[k], hi = lo + (uint64_t)host_numel[k] * elem_size(host_dtype[k]);
        const Span* next = std::lower_bound(spans, spans + m, hi, [](const Span& s, uint64_t end) { return s.lo < end; });
        if (hi > lo && next != spans && next[-1].hi > lo) rc = FNET_E_OVERLAP;
    }
    free(spans);
    if (rc != FNET_OK) return rc;
    // the clock moves with the first launch, so everything that can be refused has been by now
    int32_t used = 0;
    rc = h->max_norm < 0.0 ? fnet_list_clock(h->clock, h->beta1, h->beta2, stream)
                           : fnet_list_norm_partials(n, host_grad, host_numel, host_dtype, 0, nullptr, NORM_2, h->partials, h->capacity, &used,
                                                     h->clock, h->beta1, h->beta2, stream);
    if (rc != FNET_OK) return rc;
    if (used == 0 && h->max_norm >= 0.0 && h->norm_out) return fnet_list_norm_finish(h->partials, 0, NORM_2, h->norm_out, stream);   // no elements at all
    AdamArgs a{};
    a.f = ClipFrom{h->partials, nullptr, used, NORM_2, h->max_norm, h->norm_out};
    a.clip = h->max_norm >= 0.0;
    a.clock = h->clock;
    a.lr_dev = h->lr_device;
    a.lr = h->lr;
    a.wd = h->weight_decay;
    a.b1 = (float)h->beta1;
    a.b2 = (float)h->beta2;
    a.omb1 = (float)(1.0 - h->beta1);
    a.omb2 = (float)(1.0 - h->beta2);
    a.eps = (float)h->eps;
    hipStream_t st = (hipStream_t)stream;
    for (int d = 0; d <= FNET_F16 && rc == FNET_OK; ++d) {
        auto run = [&](auto t, auto kernel) -> int {
            t.count = 0;
            t.chunks = 0;
            auto flush = [&]() -> int {
                hipLaunchKernelGGL(kernel, dim3(std::min<uint32_t>(t.chunks, kMaxBlocks)), dim3(kThreads), 0, st, t, a);
                FNET_LAUNCH_CHECK();
                a.f.norm_out = nullptr;
                t.count = 0;
                t.chunks = 0;
                return FNET_OK;
            };
            for (int k = 0; k < n; ++k) {
                if (host_dtype[k] != d) continue;
                for (int64_t at = 0; at < host_numel[k]; at += kMaxEntry) {
                    const uint32_t len = (uint32_t)std::min<int64_t>(host_numel[k] - at, kMaxEntry);
                    const int i = t.count;
                    t.p[i] = host_param[k] + (uint64_t)at * elem_size(d);
                    t.g[i] = host_grad[k] + (uint64_t)at * elem_size(d);
                    t.m[i] = host_exp_avg[k] + (uint64_t)at * 4;
                    t.v[i] = host_exp_avg_sq[k] + (uint64_t)at * 4;
                    t.master(i) = (d == FNET_F32 ? host_param[k] : host_master[k]) + (uint64_t)at * 4;
                    t.n[i] = len;
                    t.first[i] = t.chunks;
                    t.chunks += (len + kAdamChunk - 1) / kAdamChunk;
                    if (++t.count == t.SIZE) {
                        const int e = flush();
                        if (e != FNET_OK) return e;
                    }
                }
            }
            return t.count ? flush() : FNET_OK;
        };
        if (d == FNET_F32) rc = run(AdamTab(), k_list_adam<float, AdamTab>);
        else if (d == FNET_BF16) rc = run(MasterTab(), k_list_adam<bf16_t, MasterTab>);
        else rc = run(MasterTab(), k_list_adam<f16_t, MasterTab>);
    }
    return rc;
}
