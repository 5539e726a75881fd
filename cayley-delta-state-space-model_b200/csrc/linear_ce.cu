// Softmax cross entropy of hidden rows against a large vocabulary, and its gradients, without the logits in memory.
//
// With z = x W^T (x: rows x d, W: vocab x d), m_t = max_v z_tv and s_t = sum_v exp(z_tv - m_t):
//     loss_t = (m_t - z_t,y(t)) + log s_t
//     dz_tv  = g_t (exp(z_tv - m_t) / s_t - [v = y(t)])        g_t: the upstream gradient of row t
//     dx = dz W,   dW = dz^T x
// Forward: one product whose epilogue keeps the running maximum and sum of a row over a run of vocabulary tiles; the runs of a row are
// joined by a small kernel.  Backward, a piece of the vocabulary at a time: z of the piece anew, dz of it rounded to the products'
// type into scratch, then both products that read it in one launch.  Rows without a target are left out before the first product.
//
// Where all rows have one upstream gradient (mean, sum) it is a factor of dx and dW, not of dz: dz holds p - [v = y] then, and a factor's
// own rounding to bf16 does not shift all of a gradient the same way.  Where every row has its own, it is a factor of dx's rows and, in two bf16
// parts, of the x in dW: dz's one large entry of a row, near -1, is hardly rounded at all so (gradients off by 2.0e-3 of themselves instead of 2.5e-3,
// their own rounding 1.7e-3; a quarter more products).  float32, and bf16 of few rows, whose dz keeps more bits, have it in dz.
//
// All products are tcgen05 ones of TMA tiles by pairs of blocks: 256 x 256 outputs, each block loads half of both operands and keeps 128
// rows of the result, fp32 accumulators, two of them in tensor memory so that the epilogue of a tile runs beside the products of the next.
// float32 operands enter as three bf16 parts (exact to 24 bits) and six of the nine part products, the small ones first.  The tensor
// cores' float32 sums are cut off, not rounded, so that the error of a long sum grows with its length: sums that must be good to float32,
// and long ones of any kind, are folded into registers every so many steps (kFoldLogits, kFold3, kFoldLong).
//
// What bounds it: with many rows the power cap.  8 x 2048 rows of width 768: losses of 32000 words 567 to 582 us by GPU, 1.38 to 1.42 PFLOP/s (the
// library's products keep up 1.39), a training step of 50257 words with an eighth of the rows ignored 3.14 to 3.81 ms, 1.16 to 1.41 PFLOP/s of its four
// products; tensor pipe busy 83 / 83 / 81 % in losses / dz / dx and dW.  With few rows the dependent launches and W's way: 61 rows, 50257 words: 25 us, W
// alone 12.  float32, 1531 rows of 50257 words: losses 497 us, with gradients 2.22 to 2.32 ms: z anew is six part products there, 0.5 ms, where keeping it
// would be 0.1 ms of memory.
#include "cdssm_common.cuh"
#include "sm100_ptx.cuh"
#include "tile_map.cuh"
#include <cuda_bf16.h>
#include <algorithm>
#include <type_traits>

namespace cdssm {

unsigned long long wait_limit_ns();

namespace ce {

using namespace sm100;

constexpr int kM = 256, kN = 256, kK = 64;              // rows and columns of a pair's tile, depth of a stage
constexpr int kHalf = 128;                              // of either, a block's
constexpr int kStages = 7, kSoloStages = 4;             // of 32 KB, of 48
constexpr int kEpilogueWarps = 8, kThreads = 128 + 32 * kEpilogueWarps;
constexpr int kTmemCols = 2 * kN;

enum Mode { kStats, kGradLogits, kGradProducts };

// Depth blocks after which a sum is folded.  Losses of width 768 in one piece are off by 7e-7 of themselves (float32 sums in registers 3e-7), in
// pieces of 4 blocks by 3e-7, but those take an eighth longer (8 x 2048 rows: 571 -> 645 us; 61 rows: 25.8 -> 28.8).  Sums of bf16 gradients, which are
// rounded to 2^-8 in the end, run on up to so many rows (of dW) and words (of dx).  Unfolded, sums of one sign lose 2e-5 of 16 384 rows, 1.4e-4 of
// 65 536 and 7e-4 of 262 144, folded nothing to speak of, in the same time where there are many rows (30 000 rows, 8191 words: 1745 us both;
// 262 144 x 4096, 1024 words: 3.19 ms both); 500 rows of 50 257 words, cut in shares anyway, 188 and 193.
constexpr int kFoldLogits = 12, kFold3 = 4;
constexpr int kLongRows = 16384, kLongWords = 65536, kFoldLong = 16;

// Part products in the order in which they are added up: the small ones first, so that they are not lost beside the large one's rounding.
// float32 operands: (2,1), (1,2), (2,2) are below 2^-24 of the whole.  dz of a few rows of bf16 (kFewRows): its two parts.
constexpr int kTerms3 = 6;

struct Args {
    // what the forward leaves for the backward; Tp: rows padded to kM
    const int* count;            // rows that have a target; behind it, the forward's status
    const int* rows;             // (Tp) compact row -> row of the caller, -1 behind the last
    const int* target;           // (Tp) its word, -2: outside of the vocabulary
    float *row_max, *row_inv;    // (Tp) m and 1 / s
    float* hit;                  // (Tp) z of the target
    float2* part;                // (2 x runs, Tp) maximum and sum of a run of tiles, of either half of its columns
    const float* grad;           // upstream gradient: one value, or one a row of the caller
    int grad_rows, mean, row_factor;   // one a row; a mean's; one a row that is no factor of dz
    int planes, dz_planes;
    int terms, terms_dx;         // part products, of dx
    int group, folds;            // depth blocks that go through all of them together; whether a group's sum is folded
    int few, x_rows, stacked;    // see kFewRows: whether there are few rows; the rows that are loaded; dx of both parts of dz in one product
    int Tp, d, V;
    int n_tiles;                 // forward: vocabulary tiles
    const __nv_bfloat16* ahead;  // W, where rows of it may be asked for early
    int64_t ahead_stride;
    int v0, vn, vn_tiles;        // backward: first word and words of the piece
    __nv_bfloat16* dz;           // (dz_planes, Tp, dz_pitch)
    int dz_pitch;
    void *dx, *dw;
    float* acc;                  // (Tp, acc_pitch) dx of the pieces before, summed
    int acc_pitch, d_tiles, f32, first, last, whole_sectors;
    const int64_t* caller_target;   // of all rows
    int64_t n_rows, ignore;
    float4* slots;               // partial tiles of the split ones: two a block
    // where a block notes a wait that ran out.  Forward: one word, 0 before.  Backward: a word a block, which the first kernel sets, by the
    // forward's word as well, so that nothing of one backward pass is left for the next pass over the same saved rows
    int* status;
    int status_words;            // backward: of the first kernel's blocks, the most of any
    unsigned long long wait_ns;
    int withhold;
};

// kSolo: a block by itself (few rows, z alone): 128 rows and all 256 columns of a tile.  The second block of a pair would multiply rows that are not
// there, so two blocks take two tiles in the time of a pair's one (16 rows, 32000 words of width 2048: 39.9 us as pairs, 35.8 so; 61 rows,
// 50257 words of width 768: 25.9 and 25.2).
template <bool kSolo> struct __align__(1024) Smem {
    static constexpr int kStages = kSolo ? kSoloStages : ce::kStages;
    uint8_t a[kStages][kHalf * kK * 2];
    uint8_t b[kStages][(kSolo ? kN : kHalf) * kK * 2];
    // full and acc_empty: of both blocks, the first one's; empty and acc_full: arrived at in both by the first one's products
    uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};

__device__ __forceinline__ void term_planes(const Args& a, bool of_dz, bool of_dw, int term, int& pa, int& pb) {
    constexpr uint32_t ta = 2u | 0u << 2 | 1u << 4 | 1u << 6 | 0u << 8 | 0u << 10, tb = 0u | 2u << 2 | 1u << 4 | 0u << 6 | 1u << 8 | 0u << 10;
    pa = a.planes == 3 ? (ta >> (2 * term)) & 3 : of_dz && !a.row_factor ? a.dz_planes - 1 - term : 0;
    pb = a.planes == 3 ? (tb >> (2 * term)) & 3 : of_dw && a.row_factor ? 1 - term : 0;
}

// The hardware's 2^x, good to 2^-22: beside bf16's 2^-8 nothing, and of float32's gradients (4e-7) the smaller part.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// ---- the blocks' shares of the work ---------------------------------------------------------
// A segment: depth blocks [k0, k1) of one tile.
struct Segment {
    int dw;          // kGradProducts: 0 a tile of dx, 1 of dW
    int m, n;        // row and column tile
    int k0, k1, kt;  // of kt in all
    bool last;       // kStats: of its run
    int run;
};

// Rows that are read as part of a sum: whole depth blocks.  Rows behind them are never looked at in dz.
__device__ __forceinline__ int summed_rows(int count) { return max(1, (count + kK - 1) / kK) * kK; }
__device__ __forceinline__ int row_tiles(int count) { return max(1, (count + kM - 1) / kM); }

__device__ __forceinline__ int pair_id() { return blockIdx.x >> 1; }
__device__ __forceinline__ int pairs() { return gridDim.x >> 1; }

// Vocabulary tiles of a run: the fewest rounds of tiles, and few runs, whose sums have to be joined (8 x 2048 rows, 32000 words: runs of one tile
// 109 rounds and 586 us, of eight 112 rounds and 583; 4096 rows of width 2048: of two 28 rounds, of three 30, a tenth more; the price of a run was
// weighed at these two).
constexpr int kMostRun = 8;
__device__ __forceinline__ int best_run(int row_tiles, int n_tiles, int pairs) {
    int best = 1;
    float least = INFINITY;
    for (int run = 1; run <= kMostRun; run++) {
        const int units = row_tiles * ((n_tiles + run - 1) / run);
        const float cost = (float)((units + pairs - 1) / pairs * min(run, n_tiles)) + (float)units * 1e-3f;
        if (cost < least) {
            least = cost;
            best = run;
        }
    }
    return best;
}

// Forward and dz: a run of vocabulary tiles of one row tile is a pair's unit.  Row tiles change fastest, so the pairs that
// run beside each other read the same rows of W and every row of W leaves DRAM about once.
template <bool kSolo> __device__ __forceinline__ int worker_id() { return kSolo ? (int)blockIdx.x : pair_id(); }
template <bool kSolo> __device__ __forceinline__ int workers() { return kSolo ? (int)gridDim.x : pairs(); }
template <bool kSolo> struct RunWalk {
    int unit, units, mt, run_len, n_tiles, kt, n, n_end, m, run;
    __device__ RunWalk(const Args& a, int count, int n_tiles_) : n_tiles(n_tiles_) {
        mt = row_tiles(count);
        run_len = best_run(mt, n_tiles, workers<kSolo>());
        units = mt * ((n_tiles + run_len - 1) / run_len);
        kt = (a.d + kK - 1) / kK * a.terms;
        unit = worker_id<kSolo>() - workers<kSolo>();
        n = n_end = 0;
    }
    __device__ bool next(Segment& s) {
        if (n >= n_end) {
            unit += workers<kSolo>();
            if (unit >= units) return false;
            run = unit / mt;
            m = unit - run * mt;
            n = run * run_len;
            n_end = min(n + run_len, n_tiles);
        }
        s = {0, m, n, 0, kt, kt, n + 1 == n_end, run};
        n++;
        return true;
    }
};

// dx and dW.  Pairs form groups as wide as a row of column tiles (group_width()), a column a pair: a group reads its rows of dz at one time and
// dz leaves DRAM once for either product.  (Column tiles as work of their own, cut where it suits the grid: 1.28 GB read instead of 0.83 for dz of
// 262 MB.)  Of the tile rows as many whole ones as fill the groups evenly; the depth blocks of the rows that are left, dx before dW, are cut into as
// many equal shares as there are groups.  Rows of a small depth are whole ones all: what they take is their way out (28 of 2 blocks as two
// shares: 61 us, whole 40), and groups that have one of dW more than others get so much less of dx (both weighed at this size, 6 rows of 32000 words of
// width 512).
constexpr int kSplitDepth = 16, kWayOut = 10;   // depth blocks; what the way out takes in terms of them
// The widest part of a row of column tiles that leaves at most a tenth of the pairs without a group.
__host__ __device__ inline int group_width(int d_tiles, int pairs) {
    for (int w = d_tiles < 16 ? d_tiles : 16; w > 1; w--)
        if (d_tiles % w == 0 && w <= pairs && pairs / w * w * 10 >= pairs * 9) return w;
    return 1;
}
struct SplitTiles {
    int wide, parts;         // pairs of a group; groups' widths of a row of tiles
    int nx, nw, fx, fw, kx, kw, G;
    int rest, busy, low, share, more;   // depth blocks of the rest; groups with a row more and their share; the others', one more for the first ones
    __device__ SplitTiles(int mt, int vt, int d_tiles, int kx_, int kw_, int pairs, bool even) : kx(kx_), kw(kw_) {
        wide = group_width(d_tiles, pairs);
        parts = d_tiles / wide;
        G = pairs / wide;
        nx = mt * parts;
        nw = vt * parts;
        fx = kx < kSplitDepth ? nx : nx / G * G;
        fw = kw < kSplitDepth ? nw : nw / G * G;
        rest = (nx - fx) * kx + (nw - fw) * kw;
        busy = even ? 0 : fw % G;
        low = max(0, (rest + busy * kWayOut) / G - kWayOut);
        share = (rest - busy * low) / (G - busy);
        more = rest - busy * low - share * (G - busy);
    }
    __device__ int begin(int group) const {
        const int x = group - busy;
        return x <= 0 ? group * low : busy * low + x * share + min(x, more);
    }
    // the row that depth block i of the rest belongs to, and where it begins
    __device__ void at(int i, int& dw, int& row, int& start) const {
        const int x = (nx - fx) * kx;
        dw = i >= x;
        const int j = dw ? (i - x) / kw : i / kx;
        row = (dw ? fw : fx) + j;
        start = dw ? x + j * kw : j * kx;
    }
    __device__ int tile_m(int row) const { return row / parts; }
    __device__ int tile_n(int row, int member) const { return row % parts * wide + member; }
};
__device__ __forceinline__ SplitTiles split_tiles(const Args& a, int count, int pairs) {
    const int mt = row_tiles(count);
    return SplitTiles(a.dx ? mt : 0, a.dw ? (a.vn + kM - 1) / kM : 0, a.d_tiles, (a.vn + kK - 1) / kK * a.terms_dx,
                      summed_rows(count) / kK * a.terms, pairs, a.stacked);
}
struct SplitWalk {
    SplitTiles t;
    int phase = 0, i, member, group;
    int at, end;
    __device__ SplitWalk(const Args& a, int count) : t(split_tiles(a, count, pairs())) {
        group = pair_id() / t.wide;
        member = pair_id() % t.wide;
        i = group;
        at = end = 0;
        if (group < t.G) {
            at = t.begin(group);
            end = t.begin(group + 1);
        }
    }
    __device__ bool next(Segment& s) {
        if (group >= t.G) return false;
        while (phase < 2) {
            if (i < (phase ? t.fw : t.fx)) {
                const int k = phase ? t.kw : t.kx;
                s = {phase, t.tile_m(i), t.tile_n(i, member), 0, k, k, true, 0};
                i += t.G;
                return true;
            }
            phase++;
            i = group;
        }
        if (at >= end) return false;
        int dw, row, start;
        t.at(at, dw, row, start);
        const int k = dw ? t.kw : t.kx, stop = min(start + k, end);
        s = {dw, t.tile_m(row), t.tile_n(row, member), at - start, stop - start, k, true, 0};
        at = stop;
        return true;
    }
};
template <int kMode, bool kSolo> struct WalkOf { using type = RunWalk<kSolo>; };
template <> struct WalkOf<kGradProducts, false> { using type = SplitWalk; };
template <int kMode, bool kSolo>
__device__ __forceinline__ typename WalkOf<kMode, kSolo>::type make_walk(const Args& a, int count) {
    if constexpr (kMode == kGradProducts) return SplitWalk(a, count);
    else return RunWalk<kSolo>(a, count, kMode == kStats ? a.n_tiles : a.vn_tiles);
}

// ---- pairs of blocks ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t block_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The first block's copy of a barrier, as both blocks address it.
__device__ __forceinline__ uint32_t in_first(const void* bar) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
    return r;
}
// (Of this block's scope: what it orders is the reading of tensor memory, behind tcgen05's own fence.  At the cluster's it waits for the warp's
// stores to DRAM.  Nothing that is written to memory may be handed to the other block by it.)
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* dst) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(kTmemCols) : "memory");
}
// D (+)= A B over both blocks' shared memory (the same offsets in both) and tensor memory.
__device__ __forceinline__ void pair_umma_elect(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 ad, bd;\n\t"
        "mov.b64 ad, {%1, %5};\n\t"
        "mov.b64 bd, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %3, p;\n\t}" ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc),
        "r"(kDescHiSw128)
        : "memory");
}
// Both blocks' copies of the barrier are arrived at when the products issued so far are done.
__device__ __forceinline__ void pair_commit_elect(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
        "h"((unsigned short)3)
        : "memory");
}

// A tile into this block's shared memory; its bytes are counted at its own barrier.
__device__ __forceinline__ void solo_load_3d(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// A tile into this block's shared memory; its bytes are counted at the first block's barrier.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// 32 bytes of one row: a whole sector of DRAM.  dz goes out of registers straight: shared memory is what the products' operands fill (its
// way in and out there cost a tenth of the kernel).
__device__ __forceinline__ void store_sector(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// The depth blocks of a segment one by one: place in the depth, part product, and whether a fold ends with the block.  (With divisions in
// every step of producer and products, float32 ran at half of its speed.)
struct Steps {
    int depth, terms, group;
    int base, n, i, term;   // of the present group: where it begins, its blocks, the block, the part product
    __device__ Steps(const Args& a, const Segment& s) : terms(s.dw ? a.terms : a.terms_dx), group(a.group) {
        const int k0 = s.k0, kt = s.kt;
        depth = terms == 1 ? kt : kt / terms;
        const int g = k0 / (group * terms), r = k0 - g * group * terms;
        base = g * group;
        n = min(group, depth - base);
        term = terms == 1 ? 0 : r / n;
        i = r - term * n;
    }
    __device__ int kc() const { return base + i; }
    __device__ bool next() {   // true: the block before was the last of its group
        if (++i < n) return false;
        i = 0;
        if (++term < terms) return false;
        term = 0;
        base += group;
        n = min(group, depth - base);
        return true;
    }
};
// groups that blocks [k0, k1) touch
__device__ __forceinline__ int groups_of(const Args& a, const Segment& s) {
    const int per = a.group * (s.dw ? a.terms : a.terms_dx);
    return (s.k1 - 1) / per - s.k0 / per + 1;
}

struct Maps {   // kStats, kGradLogits: a x, b W; kGradProducts: (a dz, b W) for dx, (a2 dz, b2 x) for dW
    CUtensorMap a, b, a2, b2;
};

// ---- producer: one thread of either block ------------------------------------------------------
template <int kMode, bool kSolo>
__device__ __forceinline__ bool produce(Smem<kSolo>& sm, const Maps& maps, const Args& a, int count) {
    constexpr int kStages = Smem<kSolo>::kStages;
    volatile int* ab = &sm.abort_flag;
    auto walk = make_walk<kMode, kSolo>(a, count);
    Segment s;
    uint32_t it = 0;
    const int rank = kSolo ? 0 : block_rank(), am = rank * kHalf, bn = rank * kHalf;
    const uint32_t full0 = kSolo ? 0 : in_first(&sm.full[0]);
    while (walk.next(s)) {
        Steps steps(a, s);
#pragma unroll 1
        for (int k = s.k0; k < s.k1; k++, it++) {
            const int st = it % kStages;
            if (!mbar_wait_suspend(&sm.empty[st], (it / kStages & 1) ^ 1, ab, a.wait_ns)) return false;
            if constexpr (kSolo) {
                mbar_arrive_expect_tx(&sm.full[st], (a.x_rows + kN) * kK * 2);
                int pa, pb;
                term_planes(a, false, false, steps.term, pa, pb);
                const int kc = steps.kc() * kK;
                steps.next();
                solo_load_3d(sm.a[st], &maps.a, &sm.full[st], kc, 0, pa);
#pragma unroll
                for (int j = 0; j < kN / kHalf; j++)
                    solo_load_3d(sm.b[st] + j * kHalf * kK * 2, &maps.b, &sm.full[st], kc, a.v0 + s.n * kN + j * kHalf, pb);
                continue;
            }
            // (dx of few rows: the second block has none, or takes the second part of dz)
            const bool few = kMode == kGradProducts && a.few && !s.dw, part_each = few && a.stacked, rows_here = !few || part_each || rank == 0;
            if (rank == 0) {
                const uint32_t rows = few ? (part_each ? 2 : 1) * a.x_rows : 2 * kHalf;
                mbar_arrive_expect_tx(&sm.full[st], (rows + 2 * kHalf) * kK * 2);
            }
            const uint32_t full = full0 + st * 8;
            int pa = 0, pb = 0;
            if (steps.terms > 1) term_planes(a, kMode == kGradProducts, kMode == kGradProducts && s.dw, steps.term, pa, pb);
            const int kc = steps.kc() * kK;
            steps.next();
            if (kMode != kGradProducts) {
                tma_load_3d(sm.a[st], &maps.a, full, kc, s.m * kM + am, pa);
                tma_load_3d(sm.b[st], &maps.b, full, kc, a.v0 + s.n * kN + bn, pb);
            } else if (!s.dw) {
                if (rows_here) tma_load_3d(sm.a[st], &maps.a, full, kc, part_each ? 0 : s.m * kM + am, part_each ? rank : pa);
#pragma unroll
                for (int j = 0; j < kHalf / 64; j++)
                    tma_load_3d(sm.b[st] + j * 64 * kK * 2, &maps.b, full, s.n * kN + bn + j * 64, a.v0 + kc, pb);
            } else {
#pragma unroll
                for (int j = 0; j < kHalf / 64; j++) {
                    tma_load_3d(sm.a[st] + j * 64 * kK * 2, &maps.a2, full, s.m * kM + am + j * 64, kc, pa);
                    tma_load_3d(sm.b[st] + j * 64 * kK * 2, &maps.b2, full, s.n * kN + bn + j * 64, kc, pb);
                }
            }
        }
    }
    // the last products have let go of every stage: nothing arrives here once the block is gone
    for (uint32_t i = it > kStages ? it - kStages : 0; i < it; i++)
        if (!mbar_wait_suspend(&sm.empty[i % kStages], i / kStages & 1, ab, a.wait_ns)) return false;
    return true;
}

// ---- products: one warp of the first block -------------------------------------------------------
template <int kMode, bool kSolo>
__device__ __forceinline__ bool multiply(Smem<kSolo>& sm, const Args& a, int count) {
    constexpr int kStages = Smem<kSolo>::kStages;
    volatile int* ab = &sm.abort_flag;
    auto walk = make_walk<kMode, kSolo>(a, count);
    Segment s;
    uint32_t it = 0, tile = 0;
    const uint32_t tm = sm.tmem_base;
    while (walk.next(s)) {
        // (a K-major row of a tile is 128 bytes: 16 columns are 32 bytes on; an MN-major one holds 64 rows of the operand: 16 of the
        // depth are 16 rows of 128 bytes on, the next 64 rows of the operand 8192 bytes)
        const bool a_mn = kMode == kGradProducts && s.dw, b_mn = kMode == kGradProducts;
        const uint32_t idesc = umma_idesc_bf16(kSolo ? kHalf : kM, kN, false, false) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
        const uint32_t a_step = a_mn ? 2048 >> 4 : 32 >> 4, b_step = b_mn ? 2048 >> 4 : 32 >> 4;
        const uint32_t a_lbo = a_mn ? 8192 : 16, b_lbo = b_mn ? 8192 : 16;
        Steps steps(a, s);
        bool begins = true;
#pragma unroll 1
        for (int k = s.k0; k < s.k1; k++, it++) {
            const int st = it % kStages, acc = tile & 1;
            if (begins && !mbar_wait_suspend(&sm.acc_empty[acc], (tile >> 1 & 1) ^ 1, ab, a.wait_ns)) return false;
            if (!mbar_wait_suspend(&sm.full[st], it / kStages & 1, ab, a.wait_ns)) return false;
            tc_fence_after();
            const uint32_t da = desc_lo_sw128(smem_u32(sm.a[st]), a_lbo), db = desc_lo_sw128(smem_u32(sm.b[st]), b_lbo);
#pragma unroll
            for (int j = 0; j < kK / 16; j++) {
                if constexpr (kSolo) umma_bf16_elect(tm + acc * kN, da + j * a_step, db + j * b_step, idesc, !begins || j > 0);
                else pair_umma_elect(tm + acc * kN, da + j * a_step, db + j * b_step, idesc, !begins || j > 0);
            }
            auto commit = [](uint64_t* bar) {
                if constexpr (kSolo) umma_commit_elect(bar);
                else pair_commit_elect(bar);
            };
            commit(&sm.empty[st]);
            begins = (steps.next() && a.folds) || k + 1 == s.k1;
            if (begins) {
                commit(&sm.acc_full[acc]);
                tile++;
            }
        }
    }
    return true;
}

// ---- epilogues: eight warps of either block, a row a thread, 128 columns --------------------------
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(p);
}

// Columns of an output row from registers, a sector at a time where rows begin at whole ones (aligned), else singly
template <typename T, int kCols>
__device__ __forceinline__ void store_row(T* row, int col, int cols, const float (&v)[kCols], bool aligned) {
    constexpr int kE = 32 / sizeof(T);
    if (aligned && kCols % kE == 0) {
#pragma unroll
        for (int j = 0; j + kE <= kCols; j += kE) {
            if (col + j < cols) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if constexpr (sizeof(T) == 2) w[e] = pack2(v[j + 2 * e], v[j + 2 * e + 1]);
                    else w[e] = __float_as_uint(v[j + e]);
                }
                store_sector(row + col + j, w);
            }
        }
    } else if (aligned) {   // four columns
        if (col < cols) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(row + col) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
            else *reinterpret_cast<float4*>(row + col) = make_float4(v[0], v[1], v[2], v[3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kCols; j++)
            if (col + j < cols) {
                if constexpr (sizeof(T) == 2) row[col + j] = __float2bfloat16_rn(v[j]);
                else row[col + j] = v[j];
            }
    }
}

// What all of dz has been left without.
__device__ __forceinline__ float gradient_factor(const Args& a, int count) {
    return a.grad_rows ? 1.f : a.mean ? a.grad[0] / (float)max(count, 1) : a.grad[0];
}

// Columns of a row of a finished tile of dx or dW.  dx of several pieces is summed in float32 and rounded once, by the last.
template <int kCols>
__device__ __forceinline__ void emit(const Args& a, int count, float factor, int dw, int row, int col, float (&v)[kCols]) {
    if (col >= a.d) return;
    if (dw) {
        if (row >= a.vn) return;
#pragma unroll
        for (int j = 0; j < kCols; j++) v[j] *= factor;
        const size_t at = (size_t)(a.v0 + row) * a.d;
        if (a.f32) store_row(static_cast<float*>(a.dw) + at, col, a.d, v, a.whole_sectors);
        else store_row(static_cast<__nv_bfloat16*>(a.dw) + at, col, a.d, v, a.whole_sectors);
        return;
    }
    if (row >= count) return;
    float* acc = a.acc + (size_t)row * a.acc_pitch + col;
    if (!a.first) {
#pragma unroll
        for (int j = 0; j < kCols; j += 4) {
            const float4 p = *reinterpret_cast<const float4*>(acc + j);
            v[j] += p.x; v[j + 1] += p.y; v[j + 2] += p.z; v[j + 3] += p.w;
        }
    }
    if (!a.last) {
#pragma unroll
        for (int j = 0; j < kCols; j += 4) *reinterpret_cast<float4*>(acc + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        return;
    }
    const int to = a.rows[row];
    if (a.row_factor) factor = a.grad[to];
#pragma unroll
    for (int j = 0; j < kCols; j++) v[j] *= factor;
    const size_t at = (size_t)to * a.d;
    if (a.f32) store_row(static_cast<float*>(a.dx) + at, col, a.d, v, a.whole_sectors);
    else store_row(static_cast<__nv_bfloat16*>(a.dx) + at, col, a.d, v, a.whole_sectors);
}

constexpr int kSlotFloat4 = kM * kN / 4;
// where lane `lane` of warp `warp` (of the pair's sixteen) keeps four columns of a partial tile: a warp's store is 512 bytes in a row
__device__ __forceinline__ size_t slot_at(int slot, int warp, int chunk, int j4, int lane) {
    return (size_t)slot * kSlotFloat4 + ((warp * 4 + chunk) * 8 + j4) * 32 + lane;
}

// kFold: the tile's sums come in folds and are added up here, in 128 registers a thread; else they are read from tensor memory as used.
template <int kMode, bool kFold, bool kSolo>
__device__ __forceinline__ bool finish(Smem<kSolo>& sm, const Args& a, int count) {
    volatile int* ab = &sm.abort_flag;
    auto walk = make_walk<kMode, kSolo>(a, count);
    Segment s;
    const int warp = (threadIdx.x >> 5) - 4, lane = threadIdx.x & 31, quarter = warp & 3, half = warp >> 2;
    const int rank = kSolo ? 0 : block_rank(), lrow = rank * kHalf + quarter * 32 + lane;   // row of the tile
    const uint32_t acc_empty = kSolo ? smem_u32(&sm.acc_empty[0]) : in_first(&sm.acc_empty[0]);
    auto release = [&](int acc) {                        // of the accumulator: a lane of every warp
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(acc_empty + acc * 8);
    };
    const uint32_t tm = sm.tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 128;
    float top = -INFINITY, sum = 0.f;
    int run_rows = -1, target = -1;                      // of the present row tile
    float mx = 0.f, inv = 0.f, g = 0.f;
    const float factor = kMode == kGradProducts ? gradient_factor(a, count) : 0.f;
    uint32_t tile = 0;
    while (walk.next(s)) {
        const int row = s.m * kM + lrow;
        if (kMode != kGradProducts && run_rows != s.m) {
            run_rows = s.m;
            target = a.target[row];
            if (kMode == kGradLogits) {
                mx = a.row_max[row];
                inv = a.row_inv[row];
                g = 0.f;
                if (row < count) g = target == -2 ? NAN : a.grad_rows && !a.row_factor ? a.grad[a.rows[row]] : 1.f;   // (-2: no word)
            }
        }
        const bool part_each = kMode == kGradProducts && a.stacked && !s.dw;
        // whether nobody reads the warp's rows
        const bool idle = s.m * kM + (part_each ? 0 : rank * kHalf) + quarter * 32 >= (kMode == kStats ? count : summed_rows(count));
        float folded[kFold ? 128 : 1] = {};
        int acc = tile & 1;
        if constexpr (kFold) {
#pragma unroll 1
            for (int k = groups_of(a, s); k > 0; k--) {
                acc = tile & 1;
                if (!mbar_wait_suspend(&sm.acc_full[acc], tile >> 1 & 1, ab, a.wait_ns)) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    if (idle && (kMode != kGradProducts || !s.dw)) break;
                    float z[64];
                    tmem_ld32x2(tm + acc * kN + c * 64, z, tm + acc * kN + c * 64 + 32, z + 32);
                    if (c == 1) release(acc);
#pragma unroll
                    for (int j = 0; j < 64; j++) folded[c * 64 + j] += z[j];
                }
                if (idle && (kMode != kGradProducts || !s.dw)) release(acc);
                tile++;
            }
        } else {
            if (!mbar_wait_suspend(&sm.acc_full[acc], tile >> 1 & 1, ab, a.wait_ns)) return false;
            tc_fence_after();
        }
        auto columns = [&](int c, float* z) {            // 32 of them
            if constexpr (kFold) {
#pragma unroll
                for (int j = 0; j < 32; j++) z[j] = folded[c * 32 + j];
            } else {
                tmem_ld32(tm + acc * kN + c * 32, z);
            }
        };
        bool held = !kFold;                              // the accumulator: let go when its last columns are in registers
        auto let_go = [&] {
            if (held) release(acc);
            held = false;
        };
        constexpr int kUnroll = kFold ? 4 : 1;
        if (kMode == kStats) {
#pragma unroll kUnroll
            for (int c = 0; c < 4; c++) {
                if (idle) break;
                const int v0 = s.n * kN + half * 128 + c * 32;
                if (v0 >= a.V) break;
                float z[32];
                columns(c, z);
                if (c == 3) let_go();
                if (v0 + 32 > a.V) {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (v0 + j >= a.V) z[j] = -INFINITY;
                }
                const unsigned rel = (unsigned)(target - v0);
                if (__any_sync(~0u, rel < 32u)) {
                    float hit = 0.f;
#pragma unroll
                    for (int j = 0; j < 32; j++) hit = rel == (unsigned)j ? z[j] : hit;
                    if (rel < 32u) a.hit[row] = hit;
                }
                float best = z[0];
#pragma unroll
                for (int j = 1; j < 32; j++) best = fmaxf(best, z[j]);
                best = fmaxf(best, top);
                const float ref = best == -INFINITY ? 0.f : best;
                float add = 0.f;
#pragma unroll
                for (int j = 0; j < 32; j++) add += ex2((z[j] - ref) * kLog2e);
                sum = sum * ex2((top - ref) * kLog2e) + add;
                top = best;
            }
        } else if (kMode == kGradLogits) {
            const float scale = g * inv;
#pragma unroll kUnroll
            for (int c = 0; c < 2; c++) {
                if (idle) break;
                const int col = s.n * kN + half * 128 + c * 64, v0 = a.v0 + col;
                float z[64];
                if constexpr (kFold) {
                    columns(2 * c, z);
                    columns(2 * c + 1, z + 32);
                } else {
                    tmem_ld32x2(tm + acc * kN + c * 64, z, tm + acc * kN + c * 64 + 32, z + 32);
                }
                if (c == 1) let_go();
#pragma unroll
                for (int j = 0; j < 64; j++) z[j] = ex2((z[j] - mx) * kLog2e) * scale;
                // (1 is taken from the target's p in float32: nothing is lost where p is near one)
                const unsigned rel = (unsigned)(target - v0);
                if (__any_sync(~0u, rel < 64u)) {
#pragma unroll
                    for (int j = 0; j < 64; j++) z[j] = rel == (unsigned)j ? z[j] - g : z[j];
                }
                if (v0 + 64 > a.V) {
#pragma unroll
                    for (int j = 0; j < 64; j++)
                        if (v0 + j >= a.V) z[j] = 0.f;
                }
                const bool live = row < count;
#pragma unroll 1
                for (int p = 0; p < a.dz_planes; p++) {
                    __nv_bfloat16* const to = a.dz + ((size_t)p * a.Tp + row) * a.dz_pitch + col;
#pragma unroll
                    for (int j = 0; j < 64; j += 16) {
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) w[e] = live ? pack2(z[j + 2 * e], z[j + 2 * e + 1]) : 0u;
                        store_sector(to + j, w);
                        if (p + 1 < a.dz_planes) {       // what the rounding has left
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                z[j + 2 * e] -= __uint_as_float(w[e] << 16);
                                z[j + 2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
                            }
                        }
                    }
                }
            }
        } else {
            const bool whole = s.k0 == 0 && s.k1 == s.kt;
            const int slot = 2 * pair_id() + (s.k0 == 0 ? 1 : 0);
#pragma unroll kUnroll
            for (int c = 0; c < 4; c++) {
                if (!s.dw && idle) break;
                float v[32];
                columns(c, v);
                if (c == 3) let_go();
                if (whole) {
                    emit(a, count, factor, s.dw, row, s.n * kN + half * 128 + c * 32, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        a.slots[slot_at(slot, rank * 8 + warp, c, j, lane)] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                }
            }
        }
        let_go();
        if constexpr (!kFold) tile++;
        if (kMode == kStats && s.last) {
            a.part[(size_t)(2 * s.run + half) * a.Tp + row] = make_float2(top, sum);
            top = -INFINITY;
            sum = 0.f;
        }
    }
    return true;
}

// The rows of W that the block's first tile reads, into L2 while the kernels before this one are under way (all that was there before the
// call is done: index_rows_kernel).  With one row tile the first unit of a pair goes by its number alone.
template <bool kSolo>
__device__ __forceinline__ void request_first_tile(const Args& a) {
    constexpr int kEach = kSolo ? kN / 32 : kHalf / 32;   // rows a lane
    const int run = best_run(1, a.n_tiles, workers<kSolo>());
    const int row = worker_id<kSolo>() * run * kN + (kSolo ? 0 : (int)block_rank() * kHalf) + (int)(threadIdx.x & 31) * kEach;
    const int bytes = (a.d * 2) & ~15;
    for (int r = row; bytes && r < min(row + kEach, a.V); r++)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(a.ahead + (size_t)r * a.ahead_stride), "r"(bytes) : "memory");
}

template <int kMode, bool kFold, bool kSolo>
__device__ __forceinline__ void product_block(const Maps& maps, const Args& a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    using Sm = Smem<kSolo>;
    Sm& sm = *reinterpret_cast<Sm*>(smem_raw);
    constexpr int kStages = Sm::kStages;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.b);
        if (kMode == kGradProducts) { prefetch_tmap(&maps.a2); prefetch_tmap(&maps.b2); }
    }
    if ((smem_u32(smem_raw) & 1023u) != 0) {   // the swizzled tiles need 1024-byte alignment
        grid_dependency_wait();
        if (threadIdx.x == 0) {
            if (kMode == kStats) atomicCAS(a.status, 0, 499);
            else a.status[blockIdx.x] = 499;
        }
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; i++) { mbar_init(&sm.full[i], 1); mbar_init(&sm.empty[i], 1); }
        for (int i = 0; i < 2; i++) { mbar_init(&sm.acc_full[i], 1); mbar_init(&sm.acc_empty[i], (kSolo ? 1 : 2) * kEpilogueWarps); }
        sm.abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        if constexpr (kSolo) tmem_alloc(&sm.tmem_base, kTmemCols);
        else pair_tmem_alloc(&sm.tmem_base);
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    if constexpr (!kSolo) cluster_sync();
    tc_fence_after();
    if (kMode == kStats && a.ahead && warp == 2) request_first_tile<kSolo>(a);
    grid_launch_dependents();
    grid_dependency_wait();
    const int count = a.count[0], before = kMode == kGradLogits && a.first ? a.count[1] : 0;
    bool ok = true;
    // (a warpgroup's registers: 128 x 40 + 256 x 232 are the 384 x 168 of the launch)
    if (warp < 4) {
        if constexpr (kFold) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            asm volatile("fence.proxy.async.global;" ::: "memory");   // packed rows and dz were plain stores; TMA reads them
            if ((threadIdx.x & 31) == 0 && !a.withhold) ok = produce<kMode, kSolo>(sm, maps, a, count);
        } else if (warp == 1 && (kSolo || block_rank() == 0)) {
            ok = multiply<kMode, kSolo>(sm, a, count);
        }
    } else {
        if constexpr (kFold) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        ok = finish<kMode, kFold, kSolo>(sm, a, count);
    }
    if (kMode == kStats && !ok) atomicCAS(a.status, 0, 400 + warp);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (kMode != kStats && threadIdx.x == 0) {   // (whoever gives up sets the flag)
        if (sm.abort_flag) a.status[blockIdx.x] = 400;
        else if (kMode == kGradLogits && a.first) a.status[blockIdx.x] = before;
    }
    if (sm.abort_flag) {   // copies and products that are under way end within microseconds: none outlives the pair's memory
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2'000'000ull) __nanosleep(1000);
    }
    __syncthreads();
    if constexpr (!kSolo) cluster_sync();
    if (warp == 1) {
        if constexpr (kSolo) tmem_dealloc(sm.tmem_base, kTmemCols);
        else pair_tmem_dealloc(sm.tmem_base);
    }
}

template <int kMode, bool kFold>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const Args a) {
    product_block<kMode, kFold, false>(maps, a);
}
template <int kMode, bool kFold>
__global__ void __launch_bounds__(kThreads, 1)
solo_kernel(const __grid_constant__ Maps maps, const Args a) {
    product_block<kMode, kFold, true>(maps, a);
}

// dx of the rows without a target is zero.  After a wait that ran out both gradients are NaN.
__device__ __forceinline__ void blank(const Args& a, bool failed) {
    const int64_t step = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (failed) {
        auto fill = [&](void* to, int64_t n) {   // NaN, as it is in either type
            unsigned short* const p = static_cast<unsigned short*>(to);
            if (p) for (int64_t i = at; i < n * (a.f32 ? 2 : 1); i += step) p[i] = 0x7fff;
        };
        fill(a.dx, a.n_rows * a.d);
        fill(a.dw, (int64_t)a.V * a.d);
        return;
    }
    if (!a.dx) return;
    for (int64_t r = at >> 5; r < a.n_rows; r += step >> 5) {
        if (a.caller_target[r] != a.ignore) continue;
        for (int i = threadIdx.x & 31; i < a.d; i += 32) {
            if (a.f32) static_cast<float*>(a.dx)[r * a.d + i] = 0.f;
            else static_cast<__nv_bfloat16*>(a.dx)[r * a.d + i] = __nv_bfloat16(0.f);
        }
    }
}

// Sums the shares of the tiles that were split, in the order of their depth, and hands them out: a warp for 32 rows x 4 columns, shares
// eight at a time.  A block finds the split rows first, the first boundary in each (up to 127 of them: a thread per boundary); then their tiles'
// parts go round the warps.  pairs: of the launch before.
// (A column of blocks per boundary: 17 us where two tiles have 74 shares, nearly all of it blocks without work; 32 x 32 a warp 34.)
constexpr int kMostPairs = 128;
__global__ void __launch_bounds__(256) join_split_kernel(const Args a, int pairs) {
    __shared__ int firsts[kMostPairs];
    __shared__ unsigned found[kMostPairs / 32];
    grid_launch_dependents();
    grid_dependency_wait();
    bool gave_up = false;
    for (int i = threadIdx.x; i < a.status_words; i += 256) gave_up |= __ldcg(a.status + i) != 0;
    if (__syncthreads_or(gave_up)) {   // (nothing is joined over the NaN)
        if (a.last) blank(a, true);
        return;
    }
    const int count = *a.count, lane = threadIdx.x & 31;
    const SplitTiles t = split_tiles(a, count, pairs);
    // (every block has them in the same order)
    const int p0 = threadIdx.x;
    bool mine = false;
    if (p0 > 0 && p0 < t.G && t.begin(p0) < t.rest) {
        int dw, row, start;
        t.at(t.begin(p0), dw, row, start);
        mine = t.begin(p0) != start && t.begin(p0 - 1) <= start;
    }
    const unsigned ballot = __ballot_sync(~0u, mine);
    if (lane == 0 && p0 < kMostPairs) found[p0 >> 5] = ballot;
    __syncthreads();
    int n_split = 0, before = __popc(ballot & ((1u << lane) - 1));
    for (int w = 0; w < kMostPairs / 32; w++) {
        if (w < p0 >> 5) before += __popc(found[w]);
        n_split += __popc(found[w]);
    }
    if (mine) firsts[before] = p0;
    __syncthreads();
    const float factor = gradient_factor(a, count);
    const int items = n_split * t.wide * 512, warps = gridDim.x * 8;
    for (int item = blockIdx.x * 8 + (threadIdx.x >> 5); item < items; item += warps) {
        const int tile = item >> 9, p = firsts[tile / t.wide], member = tile % t.wide, warp = item >> 5 & 15, chunk = item >> 3 & 3, j4 = item & 7;
        int dw, row, start;
        t.at(t.begin(p), dw, row, start);
        const int stop = start + (dw ? t.kw : t.kx), row0 = t.tile_m(row) * kM + (warp >> 3) * kHalf + (warp & 3) * 32;
        if (!dw && row0 >= count) continue;
        const bool part_each = a.stacked && !dw;   // (every row of dx is split then; the other part's sums are the second block's)
        // p - 1 has the row's first blocks; the last share is the one that reaches its end (groups without a share are passed over)
        float v[4] = {};
        constexpr int kAhead = 8;
        for (int q0 = p - 1; q0 < t.G && (q0 < p || t.begin(q0) < stop); q0 += kAhead) {
            float4 x[kAhead];
            bool on[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) {
                const int q = q0 + k;
                on[k] = q < t.G && (q < p || t.begin(q) < stop) && t.begin(q) < t.begin(q + 1);
                if (on[k]) {
                    const int slot = 2 * (q * t.wide + member) + (q < p ? 1 : 0);
                    x[k] = __ldcg(a.slots + slot_at(slot, warp, chunk, j4, lane));
                    if (part_each) {
                        const float4 y = __ldcg(a.slots + slot_at(slot, warp + 8, chunk, j4, lane));
                        x[k] = make_float4(x[k].x + y.x, x[k].y + y.y, x[k].z + y.z, x[k].w + y.w);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; k++)
                if (on[k]) { v[0] += x[k].x; v[1] += x[k].y; v[2] += x[k].z; v[3] += x[k].w; }
        }
        emit(a, count, factor, dw, row0 + lane, t.tile_n(row, member) * kN + (warp >> 2 & 1) * 128 + chunk * 32 + j4 * 4, v);
    }
    if (a.last) blank(a, false);
}

// ---- rows in, losses out -------------------------------------------------------------------------
constexpr int kIndexThreads = 1024;

// Compact numbers of the rows that have a target, in their order: a block per 1024 rows counts the ones before its own anew (all
// of the targets come from L2 and a second launch costs more, up to some 10^5 rows; of a million rows that is 4 GB read, by L2's rate some 0.5 ms beside
// 50 ms of products).  Rows without one lose 0.
// The first kernel of a call: it lets the next ones start when all before it is done, so that they may read the caller's operands ahead.
struct Index {
    const int64_t* target;
    int64_t ignore, n_rows;
    int Tp, vocab;
    int *header, *rows, *words;
    float* loss_rows;
};
__device__ __forceinline__ void note_row(const Index& x, int at, int64_t t, int64_t y) {
    x.rows[at] = (int)t;
    x.words[at] = y >= 0 && y < x.vocab ? (int)y : -2;
}
__device__ __forceinline__ void note_end(const Index& x, int total, int tid, int threads) {
    if (tid == 0) {
        x.header[0] = total;   // rows that have a target
        x.header[1] = 0;       // status
        x.header[2] = 0;       // blocks of join_runs_kernel that are done
    }
    for (int i = total + tid; i < x.Tp; i += threads) {
        x.rows[i] = -1;
        x.words[i] = -1;
    }
}
__global__ void __launch_bounds__(kIndexThreads) index_rows_kernel(const Index x) {
    __shared__ int warp_sum[32], before_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t base = (int64_t)blockIdx.x * kIndexThreads;
    int n = 0;
    grid_dependency_wait();
    grid_launch_dependents();
#pragma unroll 4
    for (int64_t i = tid; i < base; i += kIndexThreads) n += x.target[i] != x.ignore;
    n = __reduce_add_sync(~0u, n);
    const int64_t t = base + tid;
    const int64_t y = t < x.n_rows ? x.target[t] : x.ignore;
    const bool on = t < x.n_rows && y != x.ignore;
    const unsigned ballot = __ballot_sync(~0u, on);
    if (lane == 0) {
        before_sum[warp] = n;
        warp_sum[warp] = __popc(ballot);
    }
    __syncthreads();
    int before = __reduce_add_sync(~0u, before_sum[lane]);
    const int mine = warp_sum[lane];
    const int total = before + __reduce_add_sync(~0u, mine);
    before += __reduce_add_sync(~0u, lane < warp ? mine : 0) + __popc(ballot & ((1u << lane) - 1));
    if (on) note_row(x, before, t, y);
    else if (t < x.n_rows && x.loss_rows) x.loss_rows[t] = 0.f;
    if (blockIdx.x + 1 == gridDim.x) note_end(x, total, tid, kIndexThreads);
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// The parts of a float32 value: what each rounding has left.  Infinities and NaN are their first part alone.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
    p[0] = __float2bfloat16_rn(x);
    float r = x - __bfloat162float(p[0]);
    if (!isfinite(r)) r = 0.f;
    p[1] = __float2bfloat16_rn(r);
    p[2] = __float2bfloat16_rn(r - __bfloat162float(p[1]));
}

// A row of a matrix as the products read it: `pitch` bf16 values, zeros behind the d-th, a plane a part; src NULL: zeros.
template <typename T, int kPlanes>
__device__ __forceinline__ void pack_row(const T* src, __nv_bfloat16* dst, int64_t plane, int d, int pitch, bool vec) {
    const int lane = threadIdx.x & 31;
    if (kPlanes == 1 && vec) {   // (bf16, 16-byte aligned rows: pitch is d)
        const uint4* s = reinterpret_cast<const uint4*>(src);
        constexpr int kAhead = 4;
        for (int i0 = lane; i0 < pitch / 8; i0 += 32 * kAhead) {
            uint4 u[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) u[k] = src && i0 + 32 * k < pitch / 8 ? s[i0 + 32 * k] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < kAhead; k++)
                if (i0 + 32 * k < pitch / 8) reinterpret_cast<uint4*>(dst)[i0 + 32 * k] = u[k];
        }
        return;
    }
    for (int i = 2 * lane; i < pitch; i += 64) {
        __nv_bfloat16 p[2][3];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float v = src && i + e < d ? as_float(src[i + e]) : 0.f;
            if (kPlanes == 3) split3(v, p[e]);
            else p[e][0] = __float2bfloat16_rn(v);
        }
#pragma unroll
        for (int q = 0; q < kPlanes; q++) {
            const __nv_bfloat162 both = {p[0][q], p[1][q]};
            *reinterpret_cast<__nv_bfloat162*>(dst + q * plane + i) = both;
        }
    }
}

// All rows, a warp each.  rows: the caller's row of each (NULL: the same; -1: none); the summed ones of *count if count is given.
template <typename T, int kPlanes>
__global__ void __launch_bounds__(256)
pack_rows_kernel(const T* x, int64_t stride, const int* rows, const int* count, int64_t n_rows, int d,
                 int pitch, __nv_bfloat16* out, int vec) {
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    grid_launch_dependents();
    grid_dependency_wait();
    if (r >= n_rows || (count && r >= summed_rows(*count))) return;
    const int64_t from = rows ? rows[r] : r;
    pack_row<T, kPlanes>(from < 0 ? nullptr : x + from * stride, out + r * pitch, n_rows * (int64_t)pitch, d, pitch, vec);
}

// index_rows_kernel and pack_rows_kernel in one, for up to kIndexThreads rows: a block looks all targets over for the eight rows that it
// packs, the first one writes the numbers down as well.  (61 rows: two launches 6 us, one 4.)
template <typename T, int kPlanes>
__global__ void __launch_bounds__(256)
index_and_pack_kernel(const Index x, const T* src, int64_t stride, int64_t n_rows, int d, int pitch, __nv_bfloat16* out, int vec) {
    constexpr int kEach = kIndexThreads / 256;
    __shared__ int warp_sum[8 * kEach], mine[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, first = blockIdx.x * 8;
    grid_dependency_wait();
    grid_launch_dependents();
    if (tid < 8) mine[tid] = -1;
    int64_t y[kEach];
    unsigned ballot[kEach];
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int t = (warp * kEach + k) * 32 + lane;
        y[k] = t < x.n_rows ? x.target[t] : x.ignore;
        ballot[k] = __ballot_sync(~0u, y[k] != x.ignore);
        if (lane == 0) warp_sum[warp * kEach + k] = __popc(ballot[k]);
    }
    __syncthreads();
    const int sums = warp_sum[lane], total = __reduce_add_sync(~0u, sums);
#pragma unroll
    for (int k = 0; k < kEach; k++) {
        const int t = (warp * kEach + k) * 32 + lane;
        const int at = __reduce_add_sync(~0u, lane < warp * kEach + k ? sums : 0) + __popc(ballot[k] & ((1u << lane) - 1));
        const bool on = y[k] != x.ignore;
        if (on && at >= first && at < first + 8) mine[at - first] = t;
        if (blockIdx.x == 0) {
            if (on) note_row(x, at, t, y[k]);
            else if (t < x.n_rows && x.loss_rows) x.loss_rows[t] = 0.f;
        }
    }
    if (blockIdx.x == 0) note_end(x, total, tid, 256);
    __syncthreads();
    const int64_t r = first + warp;
    if (r >= n_rows || r >= summed_rows(total)) return;
    pack_row<T, kPlanes>(mine[warp] < 0 ? nullptr : src + mine[warp] * stride, out + r * pitch, n_rows * (int64_t)pitch, d, pitch, vec);
}

// Packed bf16 rows times their upstream gradients, in two parts, a warp each.
__global__ void __launch_bounds__(256)
scale_rows_kernel(const __nv_bfloat16* x, const int* rows, const int* count, const float* grad, int Tp, int pitch, __nv_bfloat16* out) {
    const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    grid_launch_dependents();
    grid_dependency_wait();
    if (r >= summed_rows(*count)) return;
    const int from = rows[r];
    const float g = from < 0 ? 0.f : grad[from];
    const uint4* const src = reinterpret_cast<const uint4*>(x + r * pitch);
    uint4* const dst = reinterpret_cast<uint4*>(out + r * pitch);
    uint4* const rest = reinterpret_cast<uint4*>(out + (Tp + r) * pitch);
    for (int i = threadIdx.x & 31; i < pitch / 8; i += 32) {
        const uint4 u = src[i];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = from < 0 ? 0.f : __uint_as_float(w[e] << 16) * g, b = from < 0 ? 0.f : __uint_as_float(w[e] & 0xffff0000u) * g;
            hi[e] = pack2(a, b);
            lo[e] = pack2(a - __uint_as_float(hi[e] << 16), b - __uint_as_float(hi[e] & 0xffff0000u));
        }
        dst[i] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        rest[i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// Joins the runs of a row: m, 1 / s and the loss, and (mean, sum) the losses' sum: every block leaves its own, the last one to come adds
// them up in their order.  Eight rows a block, 32 threads a row: a call of few rows has few of them and hundreds of runs each (400 runs of
// 61 rows with a thread per row and eighth of the runs: 28 us).
constexpr int kJoinRows = 8;
__global__ void __launch_bounds__(256)
join_runs_kernel(const float2* part, int n_tiles, int workers, int Tp, int* header, const int* rows, const int* words,
                 float* row_max, float* row_inv, const float* hit, float* loss, int reduction,
                 double* sums) {
    __shared__ float2 join[8][kJoinRows];
    __shared__ double warp_sum[8];
    __shared__ bool is_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x * kJoinRows + (tid & 7);
    grid_launch_dependents();
    grid_dependency_wait();
    const int count = header[0], run = best_run(row_tiles(count), n_tiles, workers), n_parts = 2 * ((n_tiles + run - 1) / run);
    const bool failed = header[1] != 0;
    float top = -INFINITY, sum = 0.f;
    auto add = [&](float2 p) {
        const float best = fmaxf(top, p.x), ref = best == -INFINITY ? 0.f : best;
        sum = sum * ex2((top - ref) * kLog2e) + p.y * ex2((p.x - ref) * kLog2e);
        top = best;
    };
    if (r < count) {
        constexpr int kAhead = 4;
        for (int i = tid >> 3; i < n_parts; i += 32 * kAhead) {
            float2 p[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; k++) p[k] = i + 32 * k < n_parts ? __ldcg(part + (size_t)(i + 32 * k) * Tp + r) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int k = 0; k < kAhead; k++) add(p[k]);
        }
    }
#pragma unroll
    for (int o = 8; o < 32; o <<= 1) {
        const float2 p = {__shfl_down_sync(~0u, top, o), __shfl_down_sync(~0u, sum, o)};
        add(p);
    }
    if (lane < kJoinRows) join[warp][lane] = make_float2(top, sum);
    __syncthreads();
    double mine = 0.0;
    if (warp == 0) {
        if (lane < kJoinRows && r < count) {
            top = -INFINITY;
            sum = 0.f;
            for (int i = 0; i < 8; i++) add(join[i][lane]);
            row_max[r] = top;
            row_inv[r] = 1.f / sum;
            // (a row without any logit that is a number: NaN, as exp(-inf - -inf))
            const float l = words[r] == -2 || failed || top == -INFINITY ? NAN : (top - hit[r]) + logf(sum);
            if (reduction == CDSSM_CE_NONE) loss[rows[r]] = l;
            mine = (double)l;
        }
        for (int o = 4; o; o >>= 1) mine += __shfl_down_sync(~0u, mine, o);
    }
    if (reduction == CDSSM_CE_NONE) return;
    if (tid == 0) {
        sums[blockIdx.x] = mine;
        __threadfence();
        is_last = atomicAdd(&header[2], 1) + 1 == (int)gridDim.x;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    double total = 0.0;
    for (int i = tid; i < (int)gridDim.x; i += 256) total += __ldcg(&sums[i]);
    for (int o = 16; o; o >>= 1) total += __shfl_down_sync(~0u, total, o);
    if (lane == 0) warp_sum[warp] = total;
    __syncthreads();
    if (tid == 0) {
        total = 0.0;
        for (int i = 0; i < 8; i++) total += warp_sum[i];
        *loss = (float)(reduction == CDSSM_CE_MEAN ? total / (double)count : total);   // (mean of no rows: NaN)
    }
}

// ---- host ------------------------------------------------------------------------------------------
inline size_t up(size_t n, size_t to) { return (n + to - 1) / to * to; }

struct Sizes {
    int64_t rows;
    int d, V, planes, dz_planes, Tp, pitch, n_tiles, pieces, vn, d_tiles;
    bool f32;
    // saved, without and with W's parts (a W that is not read in place: the backward needs them as well, which mostly follows at once)
    size_t o_rows, o_words, o_max, o_inv, o_hit, o_x, o_w, saved, saved_w;
    // scratch of the forward and of the backward
    size_t o_part, o_sums, fwd, o_status, o_dz, o_acc, o_slots, o_scaled, bwd;
};
// Up to this many rows the second block of a pair would have none of its own: z is made by blocks by themselves (Smem), and bf16's dz keeps 16 bits, in
// two parts.  (Where a row has one large entry, its target's, that entry's rounding to 8 bits is all of the row's error; beyond, the rows' roundings
// average out and the products' time shows.  50257 words of width 768, a training step of 128 and of 129 rows: 120 and 115 us; with an upstream gradient a
// row 118 and 125.)  dx takes a part a block, W once, if its rows of tiles are few and deep enough that every one is split.
constexpr int kFewRows = kHalf;
constexpr size_t kPieceBytes = 512ull << 20;   // of dz, beyond which the vocabulary is cut

bool sizes_of(int64_t rows, int d, int vocab, int dtype, int sms, Sizes& s) {
    if (rows < 1 || d < 1 || vocab < 1 || (dtype != CDSSM_BF16 && dtype != CDSSM_F32)) return false;
    s.rows = rows; s.d = d; s.V = vocab;
    s.f32 = dtype == CDSSM_F32;
    s.planes = s.f32 ? 3 : 1;
    s.dz_planes = s.f32 ? 3 : rows <= kFewRows ? 2 : 1;
    s.Tp = (int)up(rows, kM);
    s.pitch = (int)up(d, 8);
    s.n_tiles = (vocab + kN - 1) / kN;
    const size_t column = (size_t)s.Tp * 2 * s.dz_planes;
    const size_t most = std::max<size_t>(kN, kPieceBytes / column / kN * kN);
    s.pieces = (int)((up(vocab, kN) + most - 1) / most);
    s.vn = (int)up((vocab + s.pieces - 1) / s.pieces, kN);
    s.pieces = (vocab + s.vn - 1) / s.vn;
    s.d_tiles = (d + kN - 1) / kN;
    size_t o = 256;
    auto take = [&](size_t bytes) { const size_t at = o; o += up(bytes, 256); return at; };
    s.o_rows = take(4ull * s.Tp); s.o_words = take(4ull * s.Tp); s.o_max = take(4ull * s.Tp); s.o_inv = take(4ull * s.Tp);
    s.o_hit = take(4ull * s.Tp); s.o_x = take(2ull * s.planes * s.Tp * s.pitch);
    s.saved = o;
    s.o_w = take(2ull * s.planes * (size_t)vocab * s.pitch);
    s.saved_w = o;
    o = 0;
    s.o_part = take(8ull * 2 * s.n_tiles * s.Tp); s.o_sums = take(8ull * (s.Tp / kJoinRows));
    s.fwd = o;
    o = 0;
    s.o_status = take(4ull * sms);
    s.o_dz = take(column * s.vn); s.o_acc = take(s.pieces > 1 ? 4ull * s.Tp * s.d_tiles * kN : 0);
    s.o_slots = take(2ull * (sms / 2) * kM * kN * 4);
    s.o_scaled = take(s.dz_planes == 1 ? 2ull * 2 * s.Tp * s.pitch : 0);
    s.bwd = o;
    return true;
}

int checked_sizes(int64_t rows, int d, int vocab, int dtype, Sizes& s) {
    if (rows < 1 || d < 1 || vocab < 1) return CDSSM_ERR_BAD_ARG;
    if (rows > (1 << 24) || d > (1 << 16) || vocab > (1 << 24)) return CDSSM_ERR_UNSUPPORTED;   // (tile numbers and row numbers in 32 bits)
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    if (sms / 2 > kMostPairs) return CDSSM_ERR_UNSUPPORTED;
    return sizes_of(rows, d, vocab, dtype, sms, s) ? CDSSM_OK : CDSSM_ERR_BAD_ARG;
}

// Tensor maps are made by the driver, which wants a context in this thread: a backward pass runs in one of its own, where no runtime call may
// have brought it about yet (allocations come from the framework's cache).
int bind_context() {
    int dev = 0;
    if (int rc = check_cuda(cudaGetDevice(&dev))) return rc;
    return check_cuda(cudaSetDevice(dev));
}

// (planes, rows, cols) bf16, boxes of box_r rows x box_c columns
bool make_map(CUtensorMap* m, const void* base, int64_t cols, int64_t rows, int planes, int64_t pitch, int box_c, int box_r) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * rows * 2};
    const cuuint32_t box[3] = {(cuuint32_t)box_c, (cuuint32_t)box_r, 1}, step[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int kMode, bool kFold, bool kSolo> struct Tag {};
template <int kMode, bool kFold, bool kSolo>
int launch_as(const Maps& maps, const Args& a, int grid, cudaStream_t st) {
    void (*kernel)(Maps, Args);
    if constexpr (kSolo) kernel = solo_kernel<kMode, kFold>;
    else kernel = product_kernel<kMode, kFold>;
    if (int rc = allow_smem<Tag<kMode, kFold, kSolo>>((const void*)kernel, sizeof(Smem<kSolo>))) return rc;
    return launch_overlapped(kernel, dim3(grid), dim3(kThreads), sizeof(Smem<kSolo>), st, maps, a);
}
void set_terms(Args& a, bool grad_products) {
    a.terms = a.planes == 3 ? kTerms3 : !grad_products ? 1 : a.row_factor ? 2 : a.dz_planes;
    a.terms_dx = a.planes != 3 && (a.row_factor || a.stacked) ? 1 : a.terms;
}
// workers: pairs, or blocks by themselves (few rows, not kGradProducts)
template <int kMode>
int launch_products(const Maps& maps, Args a, int workers, cudaStream_t st) {
    set_terms(a, kMode == kGradProducts);
    // (two parts of dz: block by block, so that the other operand's comes from L2 the second time)
    const bool long_sums = kMode == kGradProducts && (a.Tp > kLongRows || a.dz_pitch > kLongWords);
    a.group = a.planes == 3 ? kFold3 : long_sums ? kFoldLong : kMode == kGradProducts ? 1 : kFoldLogits;
    a.folds = a.planes == 3 || long_sums || (kMode != kGradProducts && a.group * kK < a.d);
    if constexpr (kMode != kGradProducts)
        if (a.few) return a.folds ? launch_as<kMode, true, true>(maps, a, workers, st) : launch_as<kMode, false, true>(maps, a, workers, st);
    return a.folds ? launch_as<kMode, true, false>(maps, a, 2 * workers, st) : launch_as<kMode, false, false>(maps, a, 2 * workers, st);
}

bool in_place(const void* w, int64_t stride, int dtype) {   // a matrix that TMA reads as it lies
    return dtype == CDSSM_BF16 && stride % 8 == 0 && ((uintptr_t)w & 15) == 0;
}

template <typename T, int kPlanes>
int pack(const void* x, int64_t stride, const int* rows, const int* count, int64_t n, const Sizes& s, void* out, bool vec, cudaStream_t st) {
    return launch_overlapped(pack_rows_kernel<T, kPlanes>, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, static_cast<const T*>(x), stride, rows,
                             count, n, s.d, s.pitch, static_cast<__nv_bfloat16*>(out), vec);
}
int pack_any(const void* x, int64_t stride, const int* rows, const int* count, int64_t n, const Sizes& s, void* out, cudaStream_t st) {
    if (s.f32) return pack<float, 3>(x, stride, rows, count, n, s, out, false, st);
    return pack<__nv_bfloat16, 1>(x, stride, rows, count, n, s, out, s.d % 8 == 0 && in_place(x, stride, CDSSM_BF16), st);
}

int index_and_pack(const Index& index, const void* x, int64_t stride, const Sizes& s, void* out, cudaStream_t st) {
    const dim3 grid(s.Tp / 8), block(256);
    __nv_bfloat16* const to = static_cast<__nv_bfloat16*>(out);
    const int vec = s.d % 8 == 0 && in_place(x, stride, CDSSM_BF16);
    return s.f32 ? launch_overlapped(index_and_pack_kernel<float, 3>, grid, block, 0, st, index, static_cast<const float*>(x), stride, s.Tp, s.d, s.pitch, to, 0)
                 : launch_overlapped(index_and_pack_kernel<__nv_bfloat16, 1>, grid, block, 0, st, index, static_cast<const __nv_bfloat16*>(x), stride, s.Tp,
                                     s.d, s.pitch, to, vec);
}

void fill_saved(Args& a, const Sizes& s, char* saved) {
    a = Args{};
    int* header = reinterpret_cast<int*>(saved);
    a.count = header;
    a.status = header + 1;
    a.rows = reinterpret_cast<int*>(saved + s.o_rows);
    a.target = reinterpret_cast<int*>(saved + s.o_words);
    a.row_max = reinterpret_cast<float*>(saved + s.o_max);
    a.row_inv = reinterpret_cast<float*>(saved + s.o_inv);
    a.hit = reinterpret_cast<float*>(saved + s.o_hit);
    a.few = s.rows <= kFewRows;
    a.x_rows = a.few ? (int)up(s.rows, 32) : kHalf;
    a.planes = s.planes; a.dz_planes = s.dz_planes; a.Tp = s.Tp; a.d = s.d; a.V = s.V;
    a.n_tiles = s.n_tiles; a.d_tiles = s.d_tiles;
    a.f32 = s.f32;
    a.wait_ns = wait_limit_ns();
}

}  // namespace ce
}  // namespace cdssm

using namespace cdssm;

extern "C" size_t cdssm_b200_linear_ce_saved_bytes(int64_t rows, int d, int vocab, const void* w, int64_t w_row_stride, int dtype) {
    ce::Sizes s;
    if (ce::checked_sizes(rows, d, vocab, dtype, s) != CDSSM_OK) return 0;
    return ce::in_place(w, w_row_stride, dtype) ? s.saved : s.saved_w;
}
extern "C" size_t cdssm_b200_linear_ce_workspace_bytes(int64_t rows, int d, int vocab, int dtype, int backward) {
    ce::Sizes s;
    return ce::checked_sizes(rows, d, vocab, dtype, s) == CDSSM_OK ? (backward ? s.bwd : s.fwd) : 0;
}

extern "C" int cdssm_b200_linear_ce_fwd(const void* x, int64_t x_row_stride, const void* w, int64_t w_row_stride, const int64_t* target,
                                        float* loss, void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes, int64_t rows,
                                        int d, int vocab, int64_t ignore_index, int reduction, int dtype, int flags, void* stream) {
    if (!x || !w || !target || !loss || !saved || !workspace || reduction < CDSSM_CE_NONE || reduction > CDSSM_CE_SUM) return CDSSM_ERR_BAD_ARG;
    if (x_row_stride < 0 || w_row_stride < d) return CDSSM_ERR_BAD_ARG;
    ce::Sizes s;
    if (int rc = ce::checked_sizes(rows, d, vocab, dtype, s)) return rc;
    const bool direct = ce::in_place(w, w_row_stride, dtype);
    if (saved_bytes < (direct ? s.saved : s.saved_w) || workspace_bytes < s.fwd || ((uintptr_t)saved & 255) || ((uintptr_t)workspace & 255)) return CDSSM_ERR_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    char *const sv = static_cast<char*>(saved), *const ws = static_cast<char*>(workspace);
    ce::Args a;
    ce::fill_saved(a, s, sv);
    int* header = reinterpret_cast<int*>(sv);
    const ce::Index index = {target, ignore_index, rows, s.Tp, vocab, header, const_cast<int*>(a.rows), const_cast<int*>(a.target),
                             reduction == CDSSM_CE_NONE ? loss : nullptr};
    if (rows <= ce::kIndexThreads) {
        if (int rc = ce::index_and_pack(index, x, x_row_stride, s, sv + s.o_x, st)) return rc;
    } else {
        if (int rc = launch_overlapped(ce::index_rows_kernel, dim3((unsigned)((rows + ce::kIndexThreads - 1) / ce::kIndexThreads)),
                                       dim3(ce::kIndexThreads), 0, st, index))
            return rc;
        if (int rc = ce::pack_any(x, x_row_stride, a.rows, a.count, s.Tp, s, sv + s.o_x, st)) return rc;
    }
    if (!direct)
        if (int rc = ce::pack_any(w, w_row_stride, nullptr, nullptr, vocab, s, sv + s.o_w, st)) return rc;
    if (int rc = ce::bind_context()) return rc;
    ce::Maps maps{};
    if (!ce::make_map(&maps.a, sv + s.o_x, s.pitch, s.Tp, s.planes, s.pitch, ce::kK, a.x_rows) ||
        !ce::make_map(&maps.b, direct ? w : sv + s.o_w, direct ? d : s.pitch, vocab, s.planes, direct ? w_row_stride : s.pitch, ce::kK, ce::kHalf))
        return CDSSM_ERR_CUDA;
    a.part = reinterpret_cast<float2*>(ws + s.o_part);
    a.withhold = (flags & CDSSM_SCAN_TEST_WITHHOLD) != 0;
    if (direct && s.Tp == ce::kM) {
        a.ahead = static_cast<const __nv_bfloat16*>(w);
        a.ahead_stride = w_row_stride;
    }
    const int workers = (int)std::min<int64_t>((int64_t)(s.Tp / ce::kM) * s.n_tiles, a.few ? sms : sms / 2);
    if (int rc = ce::launch_products<ce::kStats>(maps, a, workers, st)) return rc;
    return launch_overlapped(ce::join_runs_kernel, dim3(s.Tp / ce::kJoinRows), dim3(256), 0, st, a.part, s.n_tiles, workers, s.Tp, header, a.rows, a.target,
                             a.row_max, a.row_inv, a.hit, loss, reduction, reinterpret_cast<double*>(ws + s.o_sums));
}

extern "C" int cdssm_b200_linear_ce_bwd(const float* grad_loss, const void* w, int64_t w_row_stride, const int64_t* target, const void* saved,
                                        size_t saved_bytes, void* grad_x, void* grad_w, void* workspace, size_t workspace_bytes, int64_t rows,
                                        int d, int vocab, int64_t ignore_index, int reduction, int dtype, int flags, void* stream) {
    if (!grad_loss || !w || !target || !saved || !workspace || (!grad_x && !grad_w) || reduction < CDSSM_CE_NONE || reduction > CDSSM_CE_SUM)
        return CDSSM_ERR_BAD_ARG;
    if (w_row_stride < d || ((uintptr_t)grad_x & 15) || ((uintptr_t)grad_w & 15)) return CDSSM_ERR_BAD_ARG;
    ce::Sizes s;
    if (int rc = ce::checked_sizes(rows, d, vocab, dtype, s)) return rc;
    const bool direct = ce::in_place(w, w_row_stride, dtype);
    if (saved_bytes < (direct ? s.saved : s.saved_w) || workspace_bytes < s.bwd || ((uintptr_t)saved & 255) || ((uintptr_t)workspace & 255)) return CDSSM_ERR_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    char *const sv = static_cast<char*>(const_cast<void*>(saved)), *const ws = static_cast<char*>(workspace);   // (saved is read alone)
    const void* const wb = direct ? w : sv + s.o_w;
    const int64_t w_cols = direct ? d : s.pitch, w_pitch = direct ? w_row_stride : s.pitch;
    ce::Args a;
    ce::fill_saved(a, s, sv);
    a.status = reinterpret_cast<int*>(ws + s.o_status);
    a.status_words = a.few ? sms : sms / 2 * 2;
    a.row_factor = reduction == CDSSM_CE_NONE && s.dz_planes == 1;
    if (int rc = ce::bind_context()) return rc;
    ce::Maps logits{}, grads{};
    if (!ce::make_map(&logits.a, sv + s.o_x, s.pitch, s.Tp, s.planes, s.pitch, ce::kK, a.x_rows) ||
        !ce::make_map(&logits.b, wb, w_cols, vocab, s.planes, w_pitch, ce::kK, ce::kHalf) ||
        !ce::make_map(&grads.a, ws + s.o_dz, s.vn, s.Tp, s.dz_planes, s.vn, ce::kK, a.x_rows) ||
        !ce::make_map(&grads.b, wb, w_cols, vocab, s.planes, w_pitch, 64, ce::kK) ||
        !ce::make_map(&grads.a2, ws + s.o_dz, s.vn, s.Tp, s.dz_planes, s.vn, 64, ce::kK) ||
        !ce::make_map(&grads.b2, a.row_factor ? ws + s.o_scaled : sv + s.o_x, s.pitch, s.Tp, a.row_factor ? 2 : s.planes, s.pitch, 64, ce::kK))
        return CDSSM_ERR_CUDA;
    a.grad = grad_loss;
    a.grad_rows = reduction == CDSSM_CE_NONE;
    a.mean = reduction == CDSSM_CE_MEAN;
    a.dx = grad_x; a.dw = grad_w;
    a.whole_sectors = s.d % (s.f32 ? 8 : 16) == 0 && (((uintptr_t)grad_x | (uintptr_t)grad_w) & 31) == 0;
    a.dz = reinterpret_cast<__nv_bfloat16*>(ws + s.o_dz);
    a.dz_pitch = s.vn;
    a.caller_target = target;
    a.n_rows = rows;
    a.ignore = ignore_index;
    a.acc = reinterpret_cast<float*>(ws + s.o_acc);
    a.acc_pitch = s.d_tiles * ce::kN;
    a.slots = reinterpret_cast<float4*>(ws + s.o_slots);
    a.withhold = (flags & CDSSM_SCAN_TEST_WITHHOLD) != 0;
    if (a.row_factor && grad_w)
        if (int rc = launch_overlapped(ce::scale_rows_kernel, dim3(s.Tp / 8), dim3(256), 0, st, reinterpret_cast<const __nv_bfloat16*>(sv + s.o_x), a.rows,
                                       a.count, grad_loss, s.Tp, s.pitch, reinterpret_cast<__nv_bfloat16*>(ws + s.o_scaled)))
            return rc;
    for (int p = 0; p < s.pieces; p++) {
        a.v0 = p * s.vn;
        a.vn = std::min(s.vn, vocab - a.v0);
        a.vn_tiles = (a.vn + ce::kN - 1) / ce::kN;
        const int wide = ce::group_width(s.d_tiles, sms / 2);
        a.stacked = s.dz_planes == 2 && (a.vn + ce::kK - 1) / ce::kK >= ce::kSplitDepth && 2 * (s.d_tiles / wide) + 2 <= sms / 2 / wide;
        a.first = p == 0;
        a.last = p + 1 == s.pieces;
        if (int rc = ce::launch_products<ce::kGradLogits>(logits, a, a.few ? sms : sms / 2, st)) return rc;
        if (int rc = ce::launch_products<ce::kGradProducts>(grads, a, sms / 2, st)) return rc;
        ce::set_terms(a, true);
        if (int rc = launch_overlapped(ce::join_split_kernel, dim3(4 * sms), dim3(256), 0, st, a, sms / 2)) return rc;
    }
    return CDSSM_OK;
}
