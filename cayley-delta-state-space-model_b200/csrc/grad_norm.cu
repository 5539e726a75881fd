// The 2-norm of many tensors together, and their values scaled down to a bound.
//
// norm = sqrt(sum over all tensors of x^2), c = min(1, max_norm / (norm + 1e-6)), out = c x.
// A block takes one chunk of one tensor, found in a table that travels in the kernel's arguments (nothing of a call outlives it, and a
// captured call keeps its own).  Squares are summed eight at a time in float32 and from there in float64, per thread, warp, block and over
// the blocks in a fixed order: the same bits from run to run, and no length at which small gradients are lost.
// What bounds it: memory.  1.7 GB of float32: sums 237 us, 7.2 TB/s; 291 MB of bf16 into float32: sums 49 us, copy 140 us, 6.2 TB/s.
#include "cdssm_common.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include <type_traits>

namespace cdssm {
namespace gn {

constexpr int kThreads = 256, kChunk = 16384;   // values of a chunk

struct Entry {
    const void* in;
    void* out;
    int64_t n;
    int first;          // chunk of the launch
    unsigned short in_f32, out_f32;
};
template <int kMost> struct Table {
    Entry e[kMost];
    int n;
};

struct Piece {
    const void* in;
    void* out;
    int64_t at;
    int n;
    bool in_f32, out_f32;
};
template <int kMost>
__device__ __forceinline__ Piece piece(const Table<kMost>& t, int chunk) {
    int lo = 0, hi = t.n;   // the last entry that begins at or before the chunk
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.e[mid].first <= chunk) lo = mid;
        else hi = mid;
    }
    const Entry& e = t.e[lo];
    const int64_t at = (int64_t)(chunk - e.first) * kChunk, left = e.n - at;
    return {e.in, e.out, at, (int)(left < kChunk ? left : kChunk), e.in_f32 != 0, e.out_f32 != 0};
}

template <typename T> __device__ __forceinline__ float value(T x) {
    if constexpr (sizeof(T) == 2) return __bfloat162float(x);
    else return x;
}
template <typename T> struct PerVec { static constexpr int k = 16 / sizeof(T); };
template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float (&f)[PerVec<T>::k]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 2) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            f[i] = __uint_as_float(w[i]);
        }
    }
}

// The squares of a few values: in float32 where none of them leaves its range, else in float64.
template <int kE>
__device__ __forceinline__ double squares(const float (&f)[kE]) {
    float s = 0.f, most = 0.f;
#pragma unroll
    for (int i = 0; i < kE; i++) {
        s = fmaf(f[i], f[i], s);
        most = fmaxf(most, fabsf(f[i]));
    }
    if (most > 1e18f || (most < 1e-15f && most > 0.f)) {
        double d = 0.0;
#pragma unroll
        for (int i = 0; i < kE; i++) d += (double)f[i] * (double)f[i];
        return d;
    }
    return (double)s;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* p, int n) {
    constexpr int kE = PerVec<T>::k;
    double sum = 0.0;
    // values before the first 16-byte boundary and behind the last one singly
    const int lead = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T)), vecs = (n - lead) / kE, rest = n - lead - vecs * kE;
    if (threadIdx.x < lead) {
        const float f[1] = {value(p[threadIdx.x])};
        sum += squares(f);
    }
    if (threadIdx.x < rest) {
        const float f[1] = {value(p[n - rest + threadIdx.x])};
        sum += squares(f);
    }
    const uint4* const v = reinterpret_cast<const uint4*>(p + lead);
    constexpr int kAhead = 8;
    for (int i0 = threadIdx.x; i0 < vecs; i0 += kThreads * kAhead) {
        uint4 u[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (i0 + k * kThreads < vecs) u[k] = v[i0 + k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (i0 + k * kThreads < vecs) {
                float f[kE];
                unpack<T>(u[k], f);
                sum += squares(f);
            }
    }
    return sum;
}

__device__ __forceinline__ double block_sum(double x) {   // valid in thread 0
    __shared__ double warp_sum[32];
    for (int o = 16; o; o >>= 1) x += __shfl_down_sync(~0u, x, o);
    if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x < 32) {
        x = threadIdx.x < blockDim.x / 32 ? warp_sum[threadIdx.x] : 0.0;
        for (int o = 16; o; o >>= 1) x += __shfl_down_sync(~0u, x, o);
    }
    return x;
}

template <int kMost>
__global__ void __launch_bounds__(kThreads) squares_kernel(const __grid_constant__ Table<kMost> t, double* sums) {
    const Piece p = piece(t, blockIdx.x);
    grid_launch_dependents();
    grid_dependency_wait();
    const double s = block_sum(p.in_f32 ? chunk_squares(static_cast<const float*>(p.in) + p.at, p.n)
                                        : chunk_squares(static_cast<const __nv_bfloat16*>(p.in) + p.at, p.n));
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// 1 where the norm is within the bound; NaN where it is none
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
    const float c = max_norm / (norm + 1e-6f);
    return c > 1.f ? 1.f : c;
}

__global__ void __launch_bounds__(1024) norm_kernel(const double* sums, int64_t n, float max_norm, float* norm, float* factor) {
    grid_launch_dependents();
    grid_dependency_wait();
    double s = 0.0;
    constexpr int kAhead = 8;
    for (int64_t i = threadIdx.x; i < n; i += 1024 * kAhead) {
        double x[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++) x[k] = i + 1024 * k < n ? __ldcg(sums + i + 1024 * k) : 0.0;
#pragma unroll
        for (int k = 0; k < kAhead; k++) s += x[k];
    }
    s = block_sum(s);
    if (threadIdx.x == 0) {
        const float x = (float)sqrt(s);
        *norm = x;
        if (factor) *factor = clip_factor(x, max_norm);
    }
}

template <typename T, typename O>
__device__ __forceinline__ void chunk_scale(const T* p, O* o, int n, float c) {
    const bool bits = c == 1.f && sizeof(T) == sizeof(O);
    auto one = [&](int i) {
        if constexpr (sizeof(T) == sizeof(O)) {
            if (bits) { o[i] = p[i]; return; }
        }
        if constexpr (sizeof(O) == 2) o[i] = __float2bfloat16_rn(value(p[i]) * c);
        else o[i] = value(p[i]) * c;
    };
    // values up to the first 16-byte boundary of the output and behind the last one singly
    constexpr int kE = 16 / sizeof(O);
    const int lead = min(n, (int)((16 - ((uintptr_t)o & 15)) & 15) / (int)sizeof(O));
    if (((uintptr_t)(p + lead) & (kE * sizeof(T) - 1)) != 0) {   // the two lie at different offsets
        for (int i = threadIdx.x; i < n; i += kThreads) one(i);
        return;
    }
    const int vecs = (n - lead) / kE, rest = n - lead - vecs * kE;
    if (threadIdx.x < lead) one(threadIdx.x);
    if (threadIdx.x < rest) one(n - rest + threadIdx.x);
    using In = std::conditional_t<sizeof(T) == sizeof(O), uint4, uint2>;
    const In* const v = reinterpret_cast<const In*>(p + lead);
    uint4* const to = reinterpret_cast<uint4*>(o + lead);
    constexpr int kAhead = 4;
    for (int i0 = threadIdx.x; i0 < vecs; i0 += kThreads * kAhead) {
        In u[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (i0 + k * kThreads < vecs) u[k] = v[i0 + k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int i = i0 + k * kThreads;
            if (i >= vecs) continue;
            if constexpr (sizeof(T) == sizeof(O)) {
                if (bits) { to[i] = u[k]; continue; }
                const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
                uint32_t r[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (sizeof(T) == 2) {
                        const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(w[e] << 16) * c, __uint_as_float(w[e] & 0xffff0000u) * c);
                        r[e] = reinterpret_cast<const uint32_t&>(b);
                    } else {
                        r[e] = __float_as_uint(__uint_as_float(w[e]) * c);
                    }
                }
                to[i] = make_uint4(r[0], r[1], r[2], r[3]);
            } else {
                const uint32_t w[2] = {u[k].x, u[k].y};
                to[i] = make_uint4(__float_as_uint(__uint_as_float(w[0] << 16) * c), __float_as_uint(__uint_as_float(w[0] & 0xffff0000u) * c),
                                   __float_as_uint(__uint_as_float(w[1] << 16) * c), __float_as_uint(__uint_as_float(w[1] & 0xffff0000u) * c));
            }
        }
    }
}

// The chunks backwards: what the norm has read last is in L2 still.  In place and within the bound there is nothing to do, and the grid is
// small enough to find that out quickly (26 000 blocks: 31 us).
// few > 0: so many sums, few enough for every block to add up (kFewSums), and there was no norm_kernel.
template <int kMost>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ Table<kMost> t, const float* factor, int chunks, int in_place,
                                                         const double* sums, int few, float max_norm, float* norm) {
    grid_launch_dependents();
    grid_dependency_wait();
    float c;
    if (few) {
        __shared__ float shared_factor;
        const double s = block_sum((int)threadIdx.x < few ? sums[threadIdx.x] : 0.0);
        if (threadIdx.x == 0) {
            const float x = (float)sqrt(s);
            shared_factor = clip_factor(x, max_norm);
            if (blockIdx.x == 0) *norm = x;
        }
        __syncthreads();
        c = shared_factor;
    } else {
        c = *factor;
    }
    if (c == 1.f && in_place) return;
    for (int chunk = chunks - 1 - (int)blockIdx.x; chunk >= 0; chunk -= gridDim.x) {
        const Piece p = piece(t, chunk);
        if (c == 1.f && p.in == p.out) continue;
        if (p.in_f32) chunk_scale(static_cast<const float*>(p.in) + p.at, static_cast<float*>(p.out) + p.at, p.n, c);
        else if (p.out_f32) chunk_scale(static_cast<const __nv_bfloat16*>(p.in) + p.at, static_cast<float*>(p.out) + p.at, p.n, c);
        else chunk_scale(static_cast<const __nv_bfloat16*>(p.in) + p.at, static_cast<__nv_bfloat16*>(p.out) + p.at, p.n, c);
    }
}

// Up to this many chunks in one launch, the scaling blocks take the sums themselves: a launch less (135 chunks: 13.8 -> 10.7 us a call).
constexpr int kFewSums = kThreads;
constexpr int kScaleBlocks = 8;              // of an SM
constexpr int kSmall = 48, kLarge = 900;   // tensors of a launch: a table of 2 KB, or of as much as kernel arguments may hold

inline int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// fn(first tensor, tensors, chunks) for every launch's share of the tensors
template <typename F>
int each_launch(const int64_t* sizes, int n, F&& fn) {
    const int most = n <= kSmall ? kSmall : kLarge;
    for (int i = 0; i < n;) {
        int64_t chunks = 0;
        int j = i;
        for (; j < n && j - i < most && chunks + chunks_of(sizes[j]) <= 0x3fffffff; j++) chunks += chunks_of(sizes[j]);
        if (j == i) return CDSSM_ERR_UNSUPPORTED;
        if (chunks)
            if (int rc = fn(i, j - i, chunks)) return rc;
        i = j;
    }
    return CDSSM_OK;
}
template <int kMost>
void fill(Table<kMost>& t, const void* const* in, void* const* out, const int64_t* sizes, const int* in_dt, const int* out_dt, int first, int n) {
    int chunk = 0;
    t.n = 0;
    for (int i = first; i < first + n; i++) {
        if (sizes[i] == 0) continue;
        t.e[t.n++] = {in[i], out ? out[i] : nullptr, sizes[i], chunk, (unsigned short)(in_dt[i] == CDSSM_F32), (unsigned short)(out && out_dt[i] == CDSSM_F32)};
        chunk += (int)chunks_of(sizes[i]);
    }
}
template <int kMost>
int run(const void* const* in, void* const* out, const int64_t* sizes, const int* in_dt, const int* out_dt, int n, float max_norm, float* norm,
        char* ws, cudaStream_t st) {
    double* const sums = reinterpret_cast<double*>(ws + 256);
    float* const factor = out ? reinterpret_cast<float*>(ws) : nullptr;
    int64_t at = 0;
    Table<kMost> t;
    int rc = each_launch(sizes, n, [&](int first, int m, int64_t chunks) {
        fill(t, in, nullptr, sizes, in_dt, nullptr, first, m);
        const int64_t to = at;
        at += chunks;
        return launch_overlapped(squares_kernel<kMost>, dim3((unsigned)chunks), dim3(kThreads), 0, st, t, sums + to);
    });
    if (rc) return rc;
    const int few = out && n <= kMost && at > 0 && at <= kFewSums ? (int)at : 0;
    if (!few)
        if (int e = launch_overlapped(norm_kernel, dim3(1), dim3(1024), 0, st, sums, at, max_norm, norm, factor)) return e;
    if (!out) return CDSSM_OK;
    int sms = 0, in_place = 1;
    if (int e = sm_count(sms)) return e;
    for (int i = 0; i < n; i++) in_place &= in[i] == out[i];
    return each_launch(sizes, n, [&](int first, int m, int64_t chunks) {
        fill(t, in, out, sizes, in_dt, out_dt, first, m);
        return launch_overlapped(scale_kernel<kMost>, dim3((unsigned)std::min<int64_t>(chunks, kScaleBlocks * sms)), dim3(kThreads), 0, st, t, factor,
                                 (int)chunks, in_place, sums, few, max_norm, norm);
    });
}

}  // namespace gn
}  // namespace cdssm

using namespace cdssm;

extern "C" size_t cdssm_b200_grad_clip_workspace_bytes(const int64_t* sizes, int n) {
    if (n < 0 || (n && !sizes)) return 0;
    int64_t chunks = 0;
    for (int i = 0; i < n; i++) {
        if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 42)) return 0;
        chunks += gn::chunks_of(sizes[i]);
    }
    return 256 + 8 * (size_t)chunks;
}

extern "C" int cdssm_b200_grad_clip(const void* const* in, void* const* out, const int64_t* sizes, const int* in_dtypes, const int* out_dtypes, int n,
                                    float max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || !norm || !workspace || (n && (!in || !sizes || !in_dtypes)) || (out && !out_dtypes)) return CDSSM_ERR_BAD_ARG;
    const size_t need = cdssm_b200_grad_clip_workspace_bytes(sizes, n);
    if (need == 0) return CDSSM_ERR_BAD_ARG;
    if (workspace_bytes < need || ((uintptr_t)workspace & 255)) return CDSSM_ERR_WORKSPACE;
    for (int i = 0; i < n; i++) {
        if (sizes[i] == 0) continue;
        const int dt = in_dtypes[i], size = dt == CDSSM_BF16 ? 2 : 4;
        if ((dt != CDSSM_BF16 && dt != CDSSM_F32) || !in[i] || ((uintptr_t)in[i] & (size - 1))) return CDSSM_ERR_BAD_ARG;
        if (out && (!out[i] || (out_dtypes[i] != dt && out_dtypes[i] != CDSSM_F32) || ((uintptr_t)out[i] & (out_dtypes[i] == CDSSM_BF16 ? 1 : 3))))
            return CDSSM_ERR_BAD_ARG;
    }
    char* const ws = static_cast<char*>(workspace);
    const cudaStream_t st = (cudaStream_t)stream;
    return n <= gn::kSmall ? gn::run<gn::kSmall>(in, out, sizes, in_dtypes, out_dtypes, n, max_norm, norm, ws, st)
                           : gn::run<gn::kLarge>(in, out, sizes, in_dtypes, out_dtypes, n, max_norm, norm, ws, st);
}
