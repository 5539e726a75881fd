// Rows of a table for token ids, and the table's gradient by sorted tokens.
//
// out_t = scale * W[id_t];   dW[v] = scale * sum over t with id_t = v of g_t, in the order of t.
// The gradient without atomics: (id, t) pairs are sorted, every kTile of them are summed in their order, and an id that goes on over
// tiles is joined from the tiles' float32 partial sums, again in order: the same bits from run to run.  While one cluster of blocks
// sorts (a few microseconds of latency for a few KB), a second kernel fills dW with the zeros that most of its rows keep.
// What bounds it: memory where there are many rows (32 768 x 2048 float32 of a table of 32 000, forward and backward, 175 us, 6.1 TB/s; rows 56,
// clearing 40, sums 52 on their own), the launches where there are few (16 384 x 768 bf16, 50 257 rows: 41 us on the GPU, bytes 24).
#include "cdssm_common.cuh"
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <algorithm>

namespace cdssm {
namespace emb {

namespace cg = cooperative_groups;

// (No pointer here is __restrict__ and no load a read-only one: a kernel that starts before its predecessors are done reads what they write.)
// ---- values of a 16-byte vector, or single ones where rows are no multiple of it ---------------------
template <typename T, int kE> __device__ __forceinline__ void load(const T* p, float (&f)[kE]) {
    if constexpr (kE == 1) {
        if constexpr (sizeof(T) == 2) f[0] = __bfloat162float(*p);
        else f[0] = *p;
    } else if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float4 u = *reinterpret_cast<const float4*>(p);
        f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
    }
}
template <typename T, int kE> __device__ __forceinline__ void store(T* p, const float (&f)[kE]) {
    if constexpr (kE == 1) {
        if constexpr (sizeof(T) == 2) *p = __float2bfloat16_rn(f[0]);
        else *p = f[0];
    } else if constexpr (sizeof(T) == 2 && kE == 4) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(reinterpret_cast<const uint32_t&>(a), reinterpret_cast<const uint32_t&>(b));
    } else if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = reinterpret_cast<const uint32_t&>(b);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    }
}

// A warp per row; an id that is no row of the table gives NaN.
template <typename T, int kE>
__global__ void __launch_bounds__(256)
embed_kernel(const int64_t* ids, const T* w, int64_t w_stride, T* out, int64_t n, int vocab, int d, float scale) {
    const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    grid_launch_dependents();
    grid_dependency_wait();
    if (t >= n) return;
    const int64_t id = ids[t];
    const bool known = id >= 0 && id < vocab;
    const T* const from = w + (known ? id : 0) * w_stride;
    T* const to = out + t * d;
    constexpr int kAhead = 4;
    for (int c0 = (threadIdx.x & 31) * kE; c0 < d; c0 += 32 * kE * kAhead) {
        float f[kAhead][kE];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (c0 + k * 32 * kE < d) load<T, kE>(from + c0 + k * 32 * kE, f[k]);
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (c0 + k * 32 * kE < d) {
#pragma unroll
                for (int e = 0; e < kE; e++) f[k][e] = known ? f[k][e] * scale : NAN;
                store<T, kE>(to + c0 + k * 32 * kE, f[k]);
            }
    }
}

// ---- sort ------------------------------------------------------------------------------------------
constexpr int kSortThreads = 1024, kItems = 8, kMostBits = 9, kBins = 1 << kMostBits;

struct SortSmem {
    int hist[kBins];              // this block's, read by the others of the cluster
    int base[kBins];              // where this block's next key of a digit goes
    int local[kBins];             // where a digit begins in the sorted sub-tile
    int warp_total[32];
    unsigned short count[32][kBins];   // keys of a digit in a warp's part of the sub-tile, then in the warps before
    unsigned lanes[32][kBins];    // of a warp that have a digit in this round; zero between rounds
    uint2 sorted[kSortThreads * kItems];   // the sub-tile by digit: it leaves in runs (pair by pair, a sector each, 65 536 pairs took 36 us)
};

// Sum of x over the threads before this one (the block's 1024).
__device__ __forceinline__ int block_scan(int x, int* warp_total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int scan = x;
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, scan, o);
        if (lane >= o) scan += y;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    const int before = __reduce_add_sync(~0u, lane < warp ? warp_total[lane] : 0);
    __syncthreads();
    return before + scan - x;
}

// One cluster sorts (key, token) pairs by key, stable, `bits` bits a pass, each block a contiguous part of the pairs.  Ids that take no part
// (no row of the table, `skip`) get the key vocab: behind all others.
__global__ void __launch_bounds__(kSortThreads)
sort_kernel(const int64_t* ids, int n, int vocab, int64_t skip, int bits, int passes, uint2* buf0, uint2* buf1, int* spans) {
    extern __shared__ __align__(16) unsigned char sort_smem[];
    SortSmem& sm = *reinterpret_cast<SortSmem*>(sort_smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < 32 * kBins / 4; i += kSortThreads) reinterpret_cast<uint4*>(sm.lanes)[i] = make_uint4(0, 0, 0, 0);
    grid_dependency_wait();     // first, so that the next kernel may write where those before this one have read
    grid_launch_dependents();
    if (c == 0 && tid == 0) spans[0] = 0;
    const int chunk = (n + C - 1) / C, lo = min(n, c * chunk), hi = min(n, lo + chunk);
    const int bins = 1 << bits;
    const bool once = chunk <= kSortThreads * kItems;      // the block's part is one sub-tile: it is read once a pass
    const int rounds = once ? (chunk + kSortThreads - 1) / kSortThreads : kItems;
    for (int pass = 0; pass < passes; pass++) {
        const uint2* const from = pass & 1 ? buf0 : buf1;
        uint2* const to = pass & 1 ? buf1 : buf0;
        auto pair_at = [&](int i) -> uint2 {
            if (pass) return __ldcg(from + i);
            const int64_t id = ids[i];
            return make_uint2(id >= 0 && id < vocab && id != skip ? (unsigned)id : (unsigned)vocab, (unsigned)i);
        };
        const int shift = pass * bits;
        auto digit_of = [&](unsigned key) { return (int)(key >> shift) & (bins - 1); };
        uint2 pair[kItems];
        int digit[kItems], rank[kItems], here = 0;
        // the sub-tile at s: its pairs, a warp's in a row; their ranks among the warp's of their digit; the digits' counts, of the warps before and in all
        auto count_up = [&](int s) {
            for (int i = tid; i < 32 * kBins / 2; i += kSortThreads) reinterpret_cast<unsigned*>(sm.count)[i] = 0;
#pragma unroll
            for (int k = 0; k < kItems; k++) {
                const int i = s + (warp * rounds + k) * 32 + lane;
                const bool on = k < rounds && i < hi;
                pair[k] = on ? pair_at(i) : make_uint2(0, 0);
                digit[k] = on ? digit_of(pair[k].x) : bins;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kItems; k++) {
                if (k >= rounds) break;
                // (lanes of the same digit find each other in shared memory: 65 536 pairs 34 us by ballots, 40 by the match instruction, this 26)
                const bool on = digit[k] < bins;
                if (on) atomicOr(&sm.lanes[warp][digit[k]], 1u << lane);
                __syncwarp();
                const unsigned same = on ? sm.lanes[warp][digit[k]] : 0u;
                const int old = on ? sm.count[warp][digit[k]] : 0;
                rank[k] = old + __popc(same & ((1u << lane) - 1));
                __syncwarp();
                if (on && lane == __ffs(same) - 1) {
                    sm.lanes[warp][digit[k]] = 0;
                    sm.count[warp][digit[k]] = (unsigned short)(old + __popc(same));
                }
                __syncwarp();
            }
            __syncthreads();
            here = 0;
            if (tid < bins) {
#pragma unroll
                for (int q = 0; q < 32; q++) {
                    const int x = sm.count[q][tid];
                    sm.count[q][tid] = (unsigned short)here;
                    here += x;
                }
            }
        };
        if (once) {
            count_up(lo);
            if (tid < bins) sm.hist[tid] = here;
        } else {
            for (int b = tid; b < bins; b += kSortThreads) sm.hist[b] = 0;
            __syncthreads();
#pragma unroll 4
            for (int i = lo + tid; i < hi; i += kSortThreads) atomicAdd(&sm.hist[digit_of(pair_at(i).x)], 1);
        }
        cluster.sync();
        int before = 0, total = 0;
        if (tid < bins) {
#pragma unroll
            for (int q = 0; q < 8; q++) {
                const int h = q < C ? cluster.map_shared_rank(sm.hist, q)[tid] : 0;
                total += h;
                if (q < c) before += h;
            }
        }
        const int start = block_scan(total, sm.warp_total) + before;
        if (tid < bins) sm.base[tid] = start;
        for (int s = lo; s < hi; s += kSortThreads * kItems) {
            if (!once) count_up(s);
            const int local = block_scan(tid < bins ? here : 0, sm.warp_total);
            if (tid < bins) sm.local[tid] = local;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kItems; k++)
                if (k < rounds && digit[k] < bins) sm.sorted[sm.local[digit[k]] + sm.count[warp][digit[k]] + rank[k]] = pair[k];
            __syncthreads();
            for (int i = tid; i < min(hi - s, kSortThreads * kItems); i += kSortThreads) {
                const uint2 p = sm.sorted[i];
                const int d = digit_of(p.x);
                to[sm.base[d] + i - sm.local[d]] = p;
            }
            __syncthreads();
            if (tid < bins) sm.base[tid] += here;
        }
        __threadfence();
        cluster.sync();
    }
}

// Zeros beside the sort, and no sooner done than it: the sums wait for this kernel alone.  (Clusters of the sort's own launch: 65 us for 262 MB,
// two clusters of eighteen waited for a place; this 40.)
__global__ void __launch_bounds__(kSortThreads) clear_kernel(uint4* to, size_t vecs, unsigned char* tail, int tail_bytes) {
    grid_launch_dependents();
    const size_t i = (size_t)blockIdx.x * kSortThreads + threadIdx.x;
    if (i < vecs) to[i] = make_uint4(0, 0, 0, 0);
    if (blockIdx.x != 0) return;
    if ((int)threadIdx.x < tail_bytes) tail[threadIdx.x] = 0;
    grid_dependency_wait();   // (one block's is enough: the kernel is not done before it)
}

// ---- sums --------------------------------------------------------------------------------------------
// kTile sorted pairs of some columns a block: rows of one id are added up in their order.  An id that lies inside the tile is done; of
// one that came from the tile before the sum goes to head, of one that goes on into the next (and began here) to tail, and the tile is listed
// in spans (their number first).
template <typename T, int kE, int kTile>
__global__ void sum_tiles_kernel(const uint2* pairs, int n, int vocab, const T* grad, T* dw,
                                 float* head, float* tail, int* spans, int d, float scale) {
    __shared__ uint2 tile[kTile + 2];   // with the neighbours of either side
    const int tile_id = blockIdx.x, p0 = tile_id * kTile;
    grid_launch_dependents();
    grid_dependency_wait();
    for (int i = threadIdx.x; i < kTile + 2; i += blockDim.x) {
        const int p = p0 + i - 1;
        tile[i] = p >= 0 && p < n ? pairs[p] : make_uint2((unsigned)vocab, 0);
    }
    __syncthreads();
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * kE;
    if (c >= d) return;
    float sum[kE] = {};
    bool from_before = p0 > 0 && tile[0].x == tile[1].x;
    constexpr int kAhead = kTile < 8 ? kTile : 8;
    for (int i0 = 0; i0 < kTile; i0 += kAhead) {
        if (tile[i0 + 1].x >= (unsigned)vocab) return;
        float g[kAhead][kE];
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            if (tile[i0 + k + 1].x < (unsigned)vocab) load<T, kE>(grad + (size_t)tile[i0 + k + 1].y * d + c, g[k]);
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const unsigned id = tile[i0 + k + 1].x;
            if (id >= (unsigned)vocab) return;
#pragma unroll
            for (int e = 0; e < kE; e++) sum[e] += g[k][e];
            const bool ends = tile[i0 + k + 2].x != id, edge = i0 + k + 1 == kTile;
            if (ends || edge) {
                if (from_before || !ends) {
                    float* const to = (from_before ? head : tail) + (size_t)tile_id * d + c;
#pragma unroll
                    for (int e = 0; e < kE; e++) to[e] = sum[e];
                    if (!ends && !from_before && c == 0) spans[1 + atomicAdd(spans, 1)] = tile_id;   // (their order changes nothing)
                } else {
#pragma unroll
                    for (int e = 0; e < kE; e++) sum[e] *= scale;
                    store<T, kE>(dw + (size_t)id * d + c, sum);
                }
#pragma unroll
                for (int e = 0; e < kE; e++) sum[e] = 0.f;
                from_before = false;
            }
        }
    }
}

// An id that begins in a listed tile and goes on: its tail and the heads of the tiles behind, eight contiguous parts beside each other and
// then those in order; 32 x kE columns at a time.  (A block per tile instead of the list: 29 us for 512 tiles, nearly all of them without one.)
constexpr int kJoinParts = 8;
template <typename T, int kE, int kTile>
__global__ void __launch_bounds__(32 * kJoinParts)
join_tiles_kernel(const uint2* pairs, int n, const float* head, const float* tail, const int* spans,
                  T* dw, int d, float scale) {
    __shared__ float part[kJoinParts][32][kE];
    grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, chunks = (d + 32 * kE - 1) / (32 * kE);
    const long long items = (long long)spans[0] * chunks;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int tile_id = spans[1 + item / chunks], c = ((int)(item % chunks) * 32 + lane) * kE;
        const unsigned id = pairs[(size_t)tile_id * kTile + kTile - 1].x;
        int tiles = 1;                                       // that begin with the id
        for (bool on = true; on;) {
            const long long p = ((long long)tile_id + tiles + threadIdx.x) * kTile;
            const int more = __syncthreads_count(p < n && pairs[p].x == id);
            tiles += more;
            on = more == 32 * kJoinParts;
        }
        const int share = (tiles + kJoinParts - 1) / kJoinParts, q0 = y * share, q1 = min(tiles, q0 + share);
        float sum[kE] = {};
        if (c < d) {
#pragma unroll 8
            for (int q = q0; q < q1; q++) {
                float f[kE];
                load<float, kE>((q ? head : tail) + (size_t)(tile_id + q) * d + c, f);
#pragma unroll
                for (int e = 0; e < kE; e++) sum[e] += f[e];
            }
        }
#pragma unroll
        for (int e = 0; e < kE; e++) part[y][lane][e] = sum[e];
        __syncthreads();
        if (y == 0 && c < d) {
            for (int i = 1; i < kJoinParts; i++)
#pragma unroll
                for (int e = 0; e < kE; e++) sum[e] += part[i][lane][e];
#pragma unroll
            for (int e = 0; e < kE; e++) sum[e] *= scale;
            store<T, kE>(dw + (size_t)id * d + c, sum);
        }
        __syncthreads();
    }
}

// ---- few tokens ------------------------------------------------------------------------------------------
// Up to kFewTokens everything in one launch, without a sort: a block per token looks all ids over; the first token of an id adds up the id's
// rows, a warp 32 vectors of columns, or, of more rows than warps, eight contiguous parts of them beside each other and then those in order.  The
// blocks behind clear the rows of dW that no token has.  (523 tokens, 32000 x 768, forward and backward: 18.6 us with the sort, 14.5 so; 1024 tokens 18.9 and 18.6.)
constexpr int kFewTokens = 1024, kClearBytes = 32768;
template <typename T, int kE>
__global__ void __launch_bounds__(32 * kJoinParts)
few_tokens_kernel(const int64_t* ids, int n, int vocab, int64_t skip, const T* grad, T* dw, int d, float scale,
                  int rows_each) {
    __shared__ int key[kFewTokens];
    __shared__ union {
        unsigned marked[kClearBytes / 32 + 1];
        struct {
            int found[kFewTokens / 32];
            unsigned short at[kFewTokens];
            float part[kJoinParts][32][kE];
        } sum;
    } sm;
    const int tid = threadIdx.x, lane = tid & 31, y = tid >> 5;
    grid_launch_dependents();
    grid_dependency_wait();
    for (int i = tid; i < n; i += 32 * kJoinParts) {
        const int64_t id = ids[i];
        key[i] = id >= 0 && id < vocab && id != skip ? (int)id : -1;
    }
    if ((int)blockIdx.x >= n) {
        const int64_t row0 = (int64_t)(blockIdx.x - n) * rows_each;
        const int rows = (int)min((int64_t)rows_each, vocab - row0);
        for (int i = tid; i <= rows / 32; i += 32 * kJoinParts) sm.marked[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += 32 * kJoinParts) {
            const int64_t r = key[i] - row0;
            if (key[i] >= 0 && r >= 0 && r < rows) atomicOr(&sm.marked[r >> 5], 1u << (r & 31));
        }
        __syncthreads();
        const int vecs = d / kE;
        const float zeros[kE] = {};
        for (int i = tid; i < rows * vecs; i += 32 * kJoinParts) {
            const int r = i / vecs;
            if (!(sm.marked[r >> 5] >> (r & 31) & 1)) store<T, kE>(dw + (row0 + r) * d + (i - r * vecs) * kE, zeros);
        }
        return;
    }
    const int t = blockIdx.x;
    __syncthreads();
    const int id = key[t];
    if (id < 0) return;
    // the id's tokens in their order: a warp looks through every eighth 32 of them
    bool before = false;
    for (int w = y; w < (n + 31) / 32; w += kJoinParts) {
        const int p = w * 32 + lane;
        const bool same = p < n && key[p] == id;
        before |= same && p < t;
        const unsigned ballot = __ballot_sync(~0u, same);
        if (lane == 0) sm.sum.found[w] = (int)ballot;
    }
    if (__syncthreads_or(before)) return;
    int count = 0;
    for (int w = 0; w < (n + 31) / 32; w++) {
        const unsigned ballot = (unsigned)sm.sum.found[w];
        if (w % kJoinParts == y && ballot >> lane & 1) sm.sum.at[count + __popc(ballot & ((1u << lane) - 1))] = (unsigned short)(w * 32 + lane);
        count += __popc(ballot);
    }
    __syncthreads();
    const bool parts = count > kJoinParts;
    const int share = parts ? (count + kJoinParts - 1) / kJoinParts : count, q0 = parts ? y * share : 0, q1 = min(count, q0 + share);
    for (int c0 = parts ? 0 : y * 32 * kE; c0 < d; c0 += (parts ? 1 : kJoinParts) * 32 * kE) {
        const int c = c0 + lane * kE;
        float sum[kE] = {};
        if (c < d) {
            constexpr int kAhead = 4;
            for (int q = q0; q < q1; q += kAhead) {
                float f[kAhead][kE];
#pragma unroll
                for (int k = 0; k < kAhead; k++)
                    if (q + k < q1) load<T, kE>(grad + (size_t)sm.sum.at[q + k] * d + c, f[k]);
#pragma unroll
                for (int k = 0; k < kAhead; k++)
                    if (q + k < q1)
#pragma unroll
                        for (int e = 0; e < kE; e++) sum[e] += f[k][e];
            }
        }
        if (parts) {
            __syncthreads();   // (the part before has been read)
#pragma unroll
            for (int e = 0; e < kE; e++) sm.sum.part[y][lane][e] = sum[e];
            __syncthreads();
            if (y != 0) continue;
            for (int i = 1; i < kJoinParts; i++)
#pragma unroll
                for (int e = 0; e < kE; e++) sum[e] += sm.sum.part[i][lane][e];
        }
        if (c >= d) continue;
#pragma unroll
        for (int e = 0; e < kE; e++) sum[e] *= scale;
        store<T, kE>(dw + (size_t)id * d + c, sum);
    }
}

// ---- host ----------------------------------------------------------------------------------------------
inline size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }
// Pairs of a tile: few where there are few of them (523 tokens by 32: 10 us for 17 blocks of four rounds of loads).
constexpr int kFewPairs = 8192, kTileFew = 8, kTileMany = 32;

struct Layout {
    size_t buf0, buf1, head, tail, spans, bytes;
    int tiles;
};
Layout layout(int64_t n, int d) {
    Layout l;
    const int tile = n <= kFewPairs ? kTileFew : kTileMany;
    l.tiles = (int)((n + tile - 1) / tile);
    size_t o = 0;
    auto take = [&](size_t b) { const size_t at = o; o += up(b, 256); return at; };
    l.buf0 = take(8 * (size_t)n); l.buf1 = take(8 * (size_t)n);
    l.head = take(4 * (size_t)l.tiles * d); l.tail = take(4 * (size_t)l.tiles * d);
    l.spans = take(4 * ((size_t)l.tiles + 1));
    l.bytes = o;
    return l;
}
int check_sizes(int64_t n, int vocab, int d, int dtype) {
    if (n < 1 || vocab < 1 || d < 1 || (dtype != CDSSM_BF16 && dtype != CDSSM_F32)) return CDSSM_ERR_BAD_ARG;
    if (n > (1 << 28) || d > (1 << 16) || vocab > (1 << 26)) return CDSSM_ERR_UNSUPPORTED;
    return CDSSM_OK;
}

template <typename T, int kE>
int forward(const int64_t* ids, const void* w, int64_t w_stride, void* out, int64_t n, int vocab, int d, float scale, cudaStream_t st) {
    return launch_overlapped(embed_kernel<T, kE>, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, ids, static_cast<const T*>(w), w_stride,
                             static_cast<T*>(out), n, vocab, d, scale);
}

template <typename T, int kE>
int few(const int64_t* ids, int n, int vocab, int64_t skip, const void* grad, void* dw, int d, float scale, cudaStream_t st) {
    const int rows_each = (int)std::max<size_t>(1, kClearBytes / ((size_t)d * sizeof(T)));
    const int64_t blocks = (int64_t)n + (vocab + rows_each - 1) / rows_each;
    return launch_overlapped(few_tokens_kernel<T, kE>, dim3((unsigned)blocks), dim3(32 * kJoinParts), 0, st, ids, n, vocab, skip,
                             static_cast<const T*>(grad), static_cast<T*>(dw), d, scale, rows_each);
}

template <typename T, int kE, int kTile>
int sums_by(const uint2* pairs, int n, int vocab, const void* grad, void* dw, char* ws, const Layout& l, int d, float scale, int sms, cudaStream_t st) {
    const int vecs = d / kE, threads = std::min(256, (vecs + 31) / 32 * 32);
    float *const head = reinterpret_cast<float*>(ws + l.head), *const tail = reinterpret_cast<float*>(ws + l.tail);
    int* const spans = reinterpret_cast<int*>(ws + l.spans);
    if (int rc = launch_overlapped(sum_tiles_kernel<T, kE, kTile>, dim3(l.tiles, (vecs + threads - 1) / threads), dim3(threads), 0, st, pairs, n, vocab,
                                   static_cast<const T*>(grad), static_cast<T*>(dw), head, tail, spans, d, scale))
        return rc;
    constexpr int kJoinE = kE == 1 ? 1 : 4;
    return launch_overlapped(join_tiles_kernel<T, kJoinE, kTile>, dim3(std::min(l.tiles * ((d + 127) / 128), 4 * sms)), dim3(32 * kJoinParts), 0, st,
                             pairs, n, head, tail, spans, static_cast<T*>(dw), d, scale);
}
template <typename T, int kE>
int sums(const uint2* pairs, int n, int vocab, const void* grad, void* dw, char* ws, const Layout& l, int d, float scale, int sms, cudaStream_t st) {
    return n <= kFewPairs ? sums_by<T, kE, kTileFew>(pairs, n, vocab, grad, dw, ws, l, d, scale, sms, st)
                          : sums_by<T, kE, kTileMany>(pairs, n, vocab, grad, dw, ws, l, d, scale, sms, st);
}

}  // namespace emb
}  // namespace cdssm

using namespace cdssm;

extern "C" int cdssm_b200_embedding_fwd(const int64_t* ids, const void* w, int64_t w_row_stride, void* out, int64_t n, int vocab, int d, float scale,
                                        int dtype, void* stream) {
    if (!ids || !w || !out || w_row_stride < 0) return CDSSM_ERR_BAD_ARG;
    if (int rc = emb::check_sizes(n, vocab, d, dtype)) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    const int e = dtype == CDSSM_BF16 ? 8 : 4;
    const bool vec = d % e == 0 && w_row_stride % e == 0 && (((uintptr_t)w | (uintptr_t)out) & 15) == 0;
    if (dtype == CDSSM_BF16)
        return vec ? emb::forward<__nv_bfloat16, 8>(ids, w, w_row_stride, out, n, vocab, d, scale, st)
                   : emb::forward<__nv_bfloat16, 1>(ids, w, w_row_stride, out, n, vocab, d, scale, st);
    return vec ? emb::forward<float, 4>(ids, w, w_row_stride, out, n, vocab, d, scale, st)
               : emb::forward<float, 1>(ids, w, w_row_stride, out, n, vocab, d, scale, st);
}

extern "C" size_t cdssm_b200_embedding_bwd_workspace_bytes(int64_t n, int vocab, int d, int dtype) {
    return emb::check_sizes(n, vocab, d, dtype) == CDSSM_OK ? emb::layout(n, d).bytes : 0;
}

extern "C" int cdssm_b200_embedding_bwd(const int64_t* ids, const void* grad, void* grad_w, void* workspace, size_t workspace_bytes, int64_t n,
                                        int vocab, int d, int64_t padding_idx, float scale, int dtype, void* stream) {
    if (!ids || !grad || !grad_w || !workspace) return CDSSM_ERR_BAD_ARG;
    if (int rc = emb::check_sizes(n, vocab, d, dtype)) return rc;
    if (((uintptr_t)grad | (uintptr_t)grad_w) & 15) return CDSSM_ERR_BAD_ARG;
    const emb::Layout l = emb::layout(n, d);
    if (workspace_bytes < l.bytes || ((uintptr_t)workspace & 255)) return CDSSM_ERR_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    if (n <= emb::kFewTokens) {
        if (dtype == CDSSM_BF16)
            return d % 8 == 0 ? emb::few<__nv_bfloat16, 8>(ids, (int)n, vocab, padding_idx, grad, grad_w, d, scale, st)
                              : emb::few<__nv_bfloat16, 1>(ids, (int)n, vocab, padding_idx, grad, grad_w, d, scale, st);
        return d % 4 == 0 ? emb::few<float, 4>(ids, (int)n, vocab, padding_idx, grad, grad_w, d, scale, st)
                          : emb::few<float, 1>(ids, (int)n, vocab, padding_idx, grad, grad_w, d, scale, st);
    }
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    char* const ws = static_cast<char*>(workspace);
    uint2 *const b0 = reinterpret_cast<uint2*>(ws + l.buf0), *const b1 = reinterpret_cast<uint2*>(ws + l.buf1);
    int bits = 1;
    while ((int64_t)1 << bits <= vocab) bits++;   // keys 0 .. vocab
    const int passes = (bits + emb::kMostBits - 1) / emb::kMostBits, per_pass = (bits + passes - 1) / passes;
    // what one block sorts in four rounds needs no cluster; eight blocks are the most that every launch may ask for
    const int cluster = n > emb::kSortThreads * 4 ? 8 : 1;
    if (int rc = allow_smem<emb::SortSmem>((const void*)emb::sort_kernel, sizeof(emb::SortSmem))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(emb::kSortThreads);
    cfg.dynamicSmemBytes = sizeof(emb::SortSmem);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (int rc = counted(check_cuda(cudaLaunchKernelEx(&cfg, emb::sort_kernel, ids, (int)n, vocab, padding_idx, per_pass, passes, b0, b1,
                                                       reinterpret_cast<int*>(ws + l.spans)))))
        return rc;
    const size_t bytes = (size_t)vocab * d * (dtype == CDSSM_BF16 ? 2 : 4), vecs = bytes / 16;
    const size_t blocks = std::max<size_t>(1, (vecs + emb::kSortThreads - 1) / emb::kSortThreads);
    if (blocks > 0x7fffffff) return CDSSM_ERR_UNSUPPORTED;
    if (int rc = launch_overlapped(emb::clear_kernel, dim3((unsigned)blocks), dim3(emb::kSortThreads), 0, st, static_cast<uint4*>(grad_w), vecs,
                                   static_cast<unsigned char*>(grad_w) + vecs * 16, (int)(bytes % 16)))
        return rc;
    const uint2* const sorted = passes & 1 ? b0 : b1;
    if (dtype == CDSSM_BF16)
        return d % 8 == 0 ? emb::sums<__nv_bfloat16, 8>(sorted, (int)n, vocab, grad, grad_w, ws, l, d, scale, sms, st)
                          : emb::sums<__nv_bfloat16, 1>(sorted, (int)n, vocab, grad, grad_w, ws, l, d, scale, sms, st);
    return d % 4 == 0 ? emb::sums<float, 4>(sorted, (int)n, vocab, grad, grad_w, ws, l, d, scale, sms, st)
                      : emb::sums<float, 1>(sorted, (int)n, vocab, grad, grad_w, ws, l, d, scale, sms, st);
}
