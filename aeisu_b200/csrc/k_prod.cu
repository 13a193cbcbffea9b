// Matrix products on tcgen05, D[p][q] = sum_k A[p][k] B[q][k]: block-scaled FP8 or 16-bit operands,
// dense, with the rows of one side grouped by expert, or with the contraction grouped by expert.
//
// One persistent, warp-specialised kernel.  A tile is 128 x BN of the output, taken by one CTA, or
// 256 x 256, taken by a pair of CTAs (cta_group::2): each holds 128 rows of A and of the accumulator and
// half of B's rows, so that a pair reads and stages B once.  Per step of 128 bytes of the contraction,
// warp 0 copies the operands' tiles by TMA into a ring of 128-byte swizzled stages, warp 1 (of the
// pair's first CTA) issues four MMAs into FP32 accumulators in TMEM, warps 4..11 write the finished tile
// out (TMEM lane = row of A).  Warps 2 and 3 serve the form of the product:
//   * FP8: kind::mxf8f6f4.block_scale applies a power-of-two scale per row and 32 values inside the
//     tensor core; a block of 128 is four such steps with the same scale.  The scales of 128 rows and
//     four blocks form the 512-byte atom that tcgen05.cp spreads over the TMEM lanes (row r, block j at
//     (r % 32) * 16 + (r / 32) * 4 + j); warps 2 and 3 gather it from global memory once per four
//     steps, in turn and ahead of time, and the MMA names the byte j.  The accumulator never leaves TMEM
//     before the tile is done.
//   * contraction grouped by expert: a group's last step may reach into the next group's rows; warp 2
//     zeroes those rows of both operands in shared memory before the MMA sees the stage.
// The writers take a whole tile into registers and hand TMEM back before they store, because 256 columns
// leave no room for a second accumulator beside the scales.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "blockscale_dev.cuh"
#include "blockscale_host.h"
#include "tc.cuh"

namespace aeisu {
namespace {

using namespace tc;

constexpr int kBM = 128;              // rows of A per tile: the TMEM lanes
constexpr int kStepBytes = 128;       // contraction bytes per step: one swizzle row
constexpr int kWriters = 8;           // warps that write tiles out
constexpr int kThreads = 128 + 32 * kWriters;
constexpr int kRing = 201 * 1024 + 512;   // shared memory of the operand ring
constexpr int kTurn = 2048;           // shared memory of a writer: 32 rows of 64 bytes
// FP8 contractions up to here fill half of a step's rows: boxes of 64 bytes, two MMAs (170,496 x 64 -> 128: 18.5 us;
// in rows of 128 bytes, half of them out of range, 23.1).
constexpr int kNarrow = kStepBytes / 2;
constexpr int kErrWait = 1;           // error code: a wait ran out
constexpr int kAtom = 512;            // scales of 128 rows and four block columns
constexpr int kScaleSlots = 4;        // atoms that are staged at a time (even: two warps fill them)

// What is grouped by the offsets.
enum Grouping { kDense = 0, kRowsA = 1, kRowsB = 2, kContraction = 3 };

__device__ int g_product_error;

// Division of 0 <= t < 2^31 by a constant of the launch: floor(t / d) = hi(t * mul) >> shift with
// mul = ceil(2^(32 + shift) / d), 2^shift < d <= 2^(shift + 1).
struct Divider {
    uint32_t mul, shift, d;
    __device__ __forceinline__ int quotient(int t) const {
        return d == 1 ? t : int(__umulhi(uint32_t(t), mul) >> shift);
    }
};

struct ProdJob {
    Divider by_tiles, by_band, by_tp, by_rest;   // tiles of one part or group, of 16 row tiles; row tiles, of the last band
    Divider by_lanes;            // CTAs, or pairs of them
    int tp, tq;                  // row tiles of A and B
    int P, Q, K;                 // rows of A, rows of B, contraction (whole sides; per batch entry)
    int grouping, groups;
    const int* off;
    int narrow;                  // FP8, contraction of at most 64: a step stages 64 bytes of each row
    int a_mn, b_mn;              // operand stored with its rows contiguous (contraction strided)
    uint32_t idesc;              // instruction descriptor without the columns
    ScaleRef sa, sb;
    int a_rows, b_rows;          // rows that carry scales, for clamping
    void* out;
    int out_type;
    long long out_ld, out_batch;
    int swapped;                 // 1: out[q][p], else out[p][q]
    int cols;                    // columns of out
    const void* bias;
    int bias_type;
    int split, steps_per_split;  // the contraction in `split` parts:
    int cluster;                 //   of the CTAs of a cluster, joined in its shared memory (split > 1), or (1)
    long long split_stride;      //   each to its own partial output
    int balance;                 // tiles of unequal groups of a contraction are dealt to the least loaded CTAs
    int out_vec;                 // rows of out start on 32-byte boundaries
    int zero_outside, zero_rows;
    const void* values;          // 16-bit rows of B that the kernel quantises itself, or null
    int values_type;
    long long values_ld;
    int early_a;                 // A is older than the kernel before (see after_quantize)
    int after_quantize;          // starts while the quantiser of its float operand still runs; the other
                                 // operand and the offsets are older
};

// OWN: the kernel quantises B's rows itself.
template <bool FP8, int BN, int CTAS, bool OWN>
struct Shape {
    static constexpr int kGroup = OWN ? 1 : 4;               // steps that share an atom of scales
    static constexpr int kBRows = BN / CTAS;                 // rows of B that a CTA stages
    static constexpr int kATile = kBM * kStepBytes, kBTile = kBRows * kStepBytes;
    static constexpr int kAtomsB = (BN + 127) / 128;         // every CTA needs the scales of all BN
    static constexpr int kScaleBytes = FP8 ? kAtom * (1 + kAtomsB) : 0;
    static constexpr int kStage = kATile + kBTile;
    static constexpr int kStages = (kRing - kScaleSlots * kScaleBytes) / kStage;
    // Each slot has its own scale columns too: they are written again only after the MMAs that read them
    // have been committed with the slot.
    static constexpr int kScaleCols = FP8 ? 4 * (1 + kAtomsB) : 0;
    // Accumulators of two tiles where TMEM's 512 columns hold them beside the scales.
    static constexpr int kAccs = 2 * BN + kScaleSlots * kScaleCols <= 512 ? 2 : 1;
    static constexpr int kColsUsed = kAccs * BN + kScaleSlots * kScaleCols;
    static constexpr int kCols = kColsUsed <= 32 ? 32 : kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128
                                 : kColsUsed <= 256 ? 256 : 512;
    // Writers: one warp per 32 lanes, two where each then has at least 32 columns.
    static constexpr int kHalves = BN >= 64 ? 2 : 1, kWide = BN / kHalves;
    static constexpr int kBars = 4 * kStages + 4 * kScaleSlots + 2 * kAccs + 1;
    static constexpr int kBarBytes = (kBars * 8 + 15) / 16 * 16;   // what lies behind is read in 16-byte words
    static constexpr size_t kSmem = 1024 + size_t(kStages) * kStage + kScaleSlots * kScaleBytes + kWriters * kTurn + kBarBytes;
    // Behind it the bias of each writer's columns (dense) or the groups' bounds and tiles.
    static constexpr size_t kBias = kWriters * kWide * sizeof(float);
};

// ---- PTX ---------------------------------------------------------------------------------------

// K-major operand tile, rows of 128 swizzled bytes: eight rows per 1024-byte atom.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// The same with rows of 64 swizzled bytes: eight rows per 512-byte atom.
__device__ __forceinline__ uint64_t desc_narrow(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(512 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(4) << 61);
}
// Row-contiguous operand tile: chunks of 64 rows of the operand (128 swizzled bytes) by 64
// contraction values, 8192 bytes from chunk to chunk, 1024 from eight contraction values to the next.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(8192 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

template <int CTAS>
__device__ __forceinline__ void mma_block_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                                 uint32_t sfb, uint32_t acc) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma_half(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (CTAS == 1)
        mma_f16(d, a, b, idesc, acc);
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
            :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// A 512-byte scale atom to four TMEM columns, repeated in the lanes of all four warps; with a pair, in
// each CTA from its own shared memory.
template <int CTAS>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t saddr) {
    if constexpr (CTAS == 1)
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(taddr), "l"(sdesc(saddr, 128, 128))
                     : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(taddr), "l"(sdesc(saddr, 128, 128))
                     : "memory");
}
// Arrive on `bar`, at the same place in every CTA of the tile, when the MMAs issued so far are done.
template <int CTAS>
__device__ __forceinline__ void commit_all(uint64_t* bar) {
    if constexpr (CTAS == 1)
        commit(bar);
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
            :: "r"(smem_addr(bar)), "h"(uint16_t(3)) : "memory");
}
// TMEM columns by one full warp (of each CTA of the tile).
template <int CTAS>
__device__ __forceinline__ void columns_alloc(uint32_t* slot, uint32_t n) {
    if constexpr (CTAS == 1) {
        tmem_alloc(slot, n);
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(smem_addr(slot)), "r"(n) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void columns_free(uint32_t base, uint32_t n) {
    if constexpr (CTAS == 1) tmem_free(base, n);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(base), "r"(n) : "memory");
}
// Tile load into this CTA's shared memory; `bar` is a cluster address with CTAS == 2.
template <int CTAS>
__device__ __forceinline__ void tma_3d(uint32_t smem, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    if constexpr (CTAS == 1)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
            :: "r"(smem), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2"
            " [%0], [%1, {%2, %3, %4}], [%5];"
            :: "r"(smem), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

// Thread block clusters: rank, barrier and another CTA's shared memory.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t address_in(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    return a;
}
// Arrive on a barrier of the tile's first CTA, from the CTA of rank `rank`.  Without `data` nothing in
// memory is handed over (TMEM columns that have been read), and the arrival need not wait for this
// thread's stores.
template <int CTAS>
__device__ __forceinline__ void arrive_first(uint64_t* bar, int rank, bool data) {
    if (CTAS == 1 || rank == 0)
        mbar_arrive(bar);
    else if (data)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];"
                     :: "r"(address_in(smem_addr(bar), 0)) : "memory");
    else
        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];"
                     :: "r"(address_in(smem_addr(bar), 0)) : "memory");
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
    return e != 0;
}

// The clock is read only once a first try has failed: the MMA warp's waits are part of every step.
// A wait that lasts as long as many steps of a contraction takes kStepCycles more for each of them (they take about 540).
constexpr long long kWaitCycles = 4000000000LL, kStepCycles = 20000;
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, long long more = 0) {
    return mbar_try_wait(bar, parity) || mbar_wait_bounded(bar, parity, &g_product_error, kErrWait, kWaitCycles + more);
}
// As wait, for a phase that threads of the other CTA complete as well.  (An acquire on the barrier: a
// fence of cluster scope here doubled the time of every step.)
template <int CTAS>
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity) {
    if constexpr (CTAS == 1) return wait(bar, parity);
    auto done = [&] {
        uint32_t d;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(d) : "r"(smem_addr(bar)), "r"(parity) : "memory");
        return d != 0;
    };
    if (done()) return true;
    const long long t0 = clock64();
    while (!done()) {
        if (clock64() - t0 > kWaitCycles) {
            atomicCAS(&g_product_error, 0, kErrWait);
            return false;
        }
    }
    return true;
}

// ---- tiles -------------------------------------------------------------------------------------

struct Tile {
    int e;               // batch entry of the grouped operand or output
    int p0, q0;          // first rows of A and B (absolute); p0 < 0: no tile
    int p1, q1;          // ends of the rows that are stored
    int k0, k1;          // contraction range (absolute)
    int part;            // part of a split contraction
};

// Cumulative row tiles of the groups, in shared memory; offsets are clamped to [0, rows] and to be
// no smaller than the one before, so that no value of theirs leads out of the tensors.
struct Groups {
    const int* bound;    // [groups + 1]
    const int* cum;      // [groups + 1] row tiles before each group; of a contraction the groups by falling size
    const int* dealt;    // [groups] tile of each group (in that order) dealt to this CTA beside full rounds, or -1
    int lane;            // this CTA or pair among all
    bool deal;           // tiles go by `dealt`
};

constexpr int kDealGroups = 64;   // groups that are sorted and dealt at most
constexpr int kBand = 16;   // row tiles of a band

__device__ __forceinline__ int tile_count(const ProdJob& j, const Groups& g) {
    if (j.grouping == kDense) return j.tp * j.tq * j.split;
    if (j.grouping == kContraction)
        return g.deal ? (j.by_lanes.quotient(int(j.by_tiles.d)) + 1) * j.groups : j.tp * j.tq * j.groups;
    return g.cum[j.groups] * (j.grouping == kRowsA ? j.tq : j.tp);
}

template <int BM, int BN>
__device__ __forceinline__ Tile tile_at(const ProdJob& j, const Groups& g, int t, int step) {
    Tile x{0, 0, 0, j.P, j.Q, 0, j.K, 0};
    if (j.grouping == kDense) {
        // Bands of 16 row tiles, walked column by column: CTAs that run at the same time share both
        // operands' tiles in L2.
        x.part = j.by_tiles.quotient(t);
        t -= x.part * int(j.by_tiles.d);
        const int band = j.by_band.quotient(t), first = band * kBand;
        t -= band * int(j.by_band.d);
        const bool last = j.tp - first < kBand;
        const int col = last ? j.by_rest.quotient(t) : t / kBand;
        x.p0 = (first + t - col * (last ? int(j.by_rest.d) : kBand)) * BM;
        x.q0 = col * BN;
        x.k0 = x.part * j.steps_per_split * step;
        x.k1 = x.k0 + min(j.K - x.k0, j.steps_per_split * step);   // (the last part's whole length may end beyond 2^31)
    } else if (j.grouping == kContraction) {
        // Groups from the longest to the shortest: the time of a tile goes by the rows of its group.
        int i;
        if (g.deal) {
            // Entry t of this CTA (or pair): full rounds of a group's tiles, then the one dealt to it, if any.
            const int per = j.by_lanes.quotient(int(j.by_tiles.d)) + 1;
            i = t / per;
            const int round = t - i * per;
            t = round < per - 1 ? round * int(j.by_lanes.d) + g.lane : g.dealt[i];
            if (t < 0) {
                x.p0 = -1;
                return x;
            }
        } else {
            i = j.by_tiles.quotient(t);
            t -= i * int(j.by_tiles.d);
        }
        x.e = g.cum[i];
        const int col = j.by_tp.quotient(t);
        x.p0 = (t - col * j.tp) * BM;
        x.q0 = col * BN;
        x.k0 = g.bound[x.e];
        x.k1 = g.bound[x.e + 1];
    } else {
        const int other = j.grouping == kRowsA ? j.tq : j.tp;
        int lo = 0, hi = j.groups - 1;       // last group whose tiles start at or before t
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (g.cum[mid] * other <= t) lo = mid;
            else hi = mid - 1;
        }
        x.e = lo;
        const int own = g.cum[lo + 1] - g.cum[lo], in = t - g.cum[lo] * other;
        const int col = own == 1 ? in : in / own, row = in - col * own;
        if (j.grouping == kRowsA) {
            x.p0 = g.bound[lo] + row * BM;
            x.p1 = g.bound[lo + 1];
            x.q0 = col * BN;
        } else {
            x.q0 = g.bound[lo] + row * BN;
            x.q1 = g.bound[lo + 1];
            x.p0 = col * BM;
        }
    }
    return x;
}

// Columns that the MMAs of a tile compute: those that are stored, in whole steps of the instruction; a pair's
// CTAs take half of these rows of B each.  (Rows stored with their contraction strided come in chunks of 64.)
template <int BN, int CTAS>
__device__ __forceinline__ int tile_columns(const ProdJob& j, const Tile& x) {
    constexpr int kGrain = 16 * CTAS;
    return j.b_mn ? BN : min(BN, (x.q1 - x.q0 + kGrain - 1) / kGrain * kGrain);
}

// ---- scales ------------------------------------------------------------------------------------

// How the scales of an operand are read.
enum ScaleWay { kPerBlock, kPerRow, kPerRowWords };

// What this lane reads for the atom of rows row0 .. row0 + 127 and block columns kb .. kb + 3, all loads
// at once and nothing made of them yet, so that they are in flight while the previous atom is waited for.
// Rows past the end repeat earlier ones, block columns past the end the last one; neither is used.
struct RawScales {
    uint32_t v[16];
};
// Scales may be the work of a quantiser that ran beside this kernel's start, so they are read by ordinary loads that
// stay behind grid_dep_wait, not through the read-only path, which asks for data that no one writes meanwhile.
__device__ __forceinline__ uint32_t load_scale(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_scale_word(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void load_scales(RawScales& r, const ScaleRef& s, ScaleWay way, int e, int row0, int rows,
                                            int kb, int blocks) {
    const int lane = threadIdx.x & 31;
    const uint8_t* col[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) col[b] = s.ptr + e * s.batch_stride + (long long)min(kb + b, blocks - 1) * s.ld;
    if (way == kPerBlock) {
        // A tile of such an operand starts on a block of 128 rows or in its middle and does not leave it.
        const int at = min(row0, rows - 1) >> s.shift;
#pragma unroll
        for (int b = 0; b < 4; ++b) r.v[b] = load_scale(col[b] + at);
    } else if (way == kPerRowWords) {
        const int at = min(row0 + 4 * lane, rows - 4);
#pragma unroll
        for (int b = 0; b < 4; ++b) r.v[b] = load_scale_word(col[b] + at);
    } else {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                r.v[4 * b + i] = load_scale(col[b] + (min(row0 + 32 * i + lane, rows - 1) >> s.shift));
    }
}
// The atom into shared memory: row r, block j at (r % 32) * 16 + (r / 32) * 4 + j.
__device__ __forceinline__ void store_scales(const RawScales& r, ScaleWay way, uint8_t* atom) {
    const int lane = threadIdx.x & 31;
    if (way == kPerBlock) {
        const uint32_t w = r.v[0] | r.v[1] << 8 | r.v[2] << 16 | r.v[3] << 24;
        reinterpret_cast<uint4*>(atom)[lane] = make_uint4(w, w, w, w);
    } else if (way == kPerRowWords) {
        // four rows of four blocks: a 4 x 4 byte transpose
        const uint32_t a = __byte_perm(r.v[0], r.v[1], 0x5140), b = __byte_perm(r.v[2], r.v[3], 0x5140);
        const uint32_t c = __byte_perm(r.v[0], r.v[1], 0x7362), d = __byte_perm(r.v[2], r.v[3], 0x7362);
        const uint32_t w[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x5410),
                               __byte_perm(c, d, 0x7632)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 4 * lane + i;
            *reinterpret_cast<uint32_t*>(atom + (row & 31) * 16 + (row >> 5) * 4) = w[i];
        }
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = r.v[i] | r.v[4 + i] << 8 | r.v[8 + i] << 16 | r.v[12 + i] << 24;
        reinterpret_cast<uint4*>(atom)[lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// Words of four rows where every tile starts at a multiple of four rows and the columns are as aligned; tiles
// of ragged groups start anywhere.
__device__ __forceinline__ ScaleWay scale_way(const ScaleRef& s, int rows, bool ragged) {
    if (s.shift) return ragged ? kPerRow : kPerBlock;
    return !ragged && rows >= 4 && s.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(s.ptr) & 3) == 0 &&
                   s.batch_stride % 4 == 0 ? kPerRowWords : kPerRow;
}

// ---- epilogue ----------------------------------------------------------------------------------

__device__ __forceinline__ float load_elem(const void* p, int type, long long i) {
    if (type == kF32) return static_cast<const float*>(p)[i];
    if (type == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int type, long long i, float v) {
    if (type == kF32) static_cast<float*>(p)[i] = v;
    else if (type == kF16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
template <typename T> __device__ __forceinline__ T rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Columns of this thread's lane into registers, without the wait.
template <int W>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t* r) {
    if constexpr (W == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
            "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
    } else {
#pragma unroll
        for (int c = 0; c < W; c += 32) tmem_ld_x32(taddr + c, *reinterpret_cast<uint32_t(*)[32]>(r + c));
    }
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The warp's 32 rows by W columns to out[p][q].  Each lane stores its row, 32 bytes at a time: whole
// sectors, no exchange between lanes.  (Turned through shared memory, so that four lanes store a run of 64
// bytes, each run of 32 columns took a chain of 800 cycles.)  Where rows do not start on 32-byte
// boundaries, or columns end, runs of 64 bytes do turn through shared memory, and elements are stored one
// by one, neighbouring lanes at neighbouring addresses.
template <typename T, int W>
__device__ __forceinline__ void write_rows(const ProdJob& j, uint32_t* v, const float* bias, uint8_t* turn,
                                           long long base, int p0, int p1, int q0, int q1) {
    constexpr int kRun = 64 / sizeof(T) < W ? 64 / sizeof(T) : W, kWords = kRun * sizeof(T) / 4;
    const int lane = threadIdx.x & 31;
    if (j.bias) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const float4 b = *reinterpret_cast<const float4*>(bias + i);
            v[i] = __float_as_uint(__uint_as_float(v[i]) + b.x);
            v[i + 1] = __float_as_uint(__uint_as_float(v[i + 1]) + b.y);
            v[i + 2] = __float_as_uint(__uint_as_float(v[i + 2]) + b.z);
            v[i + 3] = __float_as_uint(__uint_as_float(v[i + 3]) + b.w);
        }
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) v[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
    }
    T* out = static_cast<T*>(j.out) + base;
    if (j.out_vec && q0 + W <= q1) {
        if (p0 + lane < p1) {
            T* dst = out + (p0 + lane) * j.out_ld + q0;
#pragma unroll
            for (int i = 0; i < W * int(sizeof(T)) / 4; i += 8)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                             :: "l"(reinterpret_cast<uint32_t*>(dst) + i), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]),
                                "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
                             : "memory");
        }
        return;
    }
    uint8_t* put = turn + lane * 64;
    const int turned = (lane >> 1) & 3;     // 16-byte pieces exclusive-or'ed with the row pair: no bank conflicts
#pragma unroll
    for (int c = 0; c < W / kRun; ++c) {
        if (q0 + c * kRun < q1) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i)
                *reinterpret_cast<uint4*>(put + ((i ^ turned) << 4)) =
                    make_uint4(v[c * kWords + 4 * i], v[c * kWords + 4 * i + 1], v[c * kWords + 4 * i + 2],
                               v[c * kWords + 4 * i + 3]);
            __syncwarp();
#pragma unroll 4
            for (int at = lane; at < 32 * kRun; at += 32) {
                const int r = at / kRun, k = at % kRun, b = k * int(sizeof(T));
                if (p0 + r < p1 && q0 + c * kRun + k < q1)
                    out[(p0 + r) * j.out_ld + q0 + c * kRun + k] =
                        *reinterpret_cast<const T*>(turn + r * 64 + (((b >> 4) ^ ((r >> 1) & 3)) << 4) + (b & 15));
            }
            __syncwarp();
        }
    }
}

// The same to out[q][p]: a column's 32 values lie together.
template <typename T, int W>
__device__ __forceinline__ void write_columns(const ProdJob& j, const uint32_t* v, long long base, int p, int p1, int q0,
                                              int q1) {
    T* out = static_cast<T*>(j.out) + base;
    if (p >= p1) return;
    const float b = j.bias ? load_elem(j.bias, j.bias_type, p) : 0.f;
#pragma unroll
    for (int c = 0; c < W; ++c)
        if (q0 + c < q1) out[(q0 + c) * j.out_ld + p] = rounded<T>(__uint_as_float(v[c]) + b);
}

// A tile's part goes to the ring in the order of the output: [column][128 rows] where out[q][p], else [row][BN + 4
// columns], whose four columns more keep the rows' 16-byte pieces in different banks.
template <int BN, int W>
__device__ __forceinline__ void put_part(const ProdJob& j, const uint32_t* v, uint8_t* ring, int row, int col) {
    uint32_t* tile = reinterpret_cast<uint32_t*>(ring);
    if (j.swapped) {
#pragma unroll
        for (int i = 0; i < W; ++i) tile[(col + i) * kBM + row] = v[i];
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4)
            *reinterpret_cast<uint4*>(tile + row * (BN + 4) + col + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
}
// The parts of a tile, one in the shared memory of each of the cluster's CTAs, added in their order; each CTA
// takes its share of the lines (rows or columns) of the output, a thread four neighbouring values, with the
// loads of all parts and of two lines under way at once.
template <int BN, int PARTS>
__device__ __forceinline__ void join_cluster(const ProdJob& j, const Tile& x, int rank, uint32_t tile) {
    const int lines = j.swapped ? BN : kBM, wide = j.swapped ? kBM : BN, pitch = j.swapped ? kBM : BN + 4;
    const int line0 = j.swapped ? x.q0 : x.p0, line1 = j.swapped ? x.q1 : x.p1;      // of the output, and its values
    const int at0 = j.swapped ? x.p0 : x.q0, at1 = j.swapped ? x.p1 : x.q1;
    const int share = lines / PARTS, quads = wide / 4, t = threadIdx.x - 128;
    uint32_t part[PARTS];
#pragma unroll
    for (int i = 0; i < PARTS; ++i) part[i] = address_in(tile, i);
#pragma unroll 2
    for (int u = t; u < share * quads; u += 32 * kWriters) {
        const int line = rank * share + u / quads, c = u % quads * 4, l = line0 + line, at = at0 + c;
        if (l >= line1 || at >= at1) continue;
        float4 v[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[i].x), "=f"(v[i].y), "=f"(v[i].z), "=f"(v[i].w)
                         : "r"(part[i] + uint32_t(line * pitch + c) * 4) : "memory");
        float4 s = v[0];
#pragma unroll
        for (int i = 1; i < PARTS; ++i) s.x += v[i].x, s.y += v[i].y, s.z += v[i].z, s.w += v[i].w;
        const float o[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < at1)
                store_elem(j.out, j.out_type, l * j.out_ld + at + i,
                           o[i] + (j.bias ? load_elem(j.bias, j.bias_type, at + i) : 0.f));
    }
}

// Few rows quantised on the spot (OWN): a warp's half, eight rows, of the rows q0 .. q0 + 15 of the 16-bit B by
// 128 columns from k on, four lanes to a row.  Loaded a step ahead, turned into codes of the stage's swizzled
// tile and scales of the atom's first block; the same arithmetic as the quantiser's, which these calls do
// without.
struct OwnRows {
    blockq::Vals<__half> v[2];   // 32 values; the type only matters where they are read
};
__device__ __forceinline__ void load_own(OwnRows& o, const ProdJob& j, const Tile& x, int half, int k) {
    const int lane = threadIdx.x & 31, q = x.q0 + half * 8 + (lane >> 2), c = k + (lane & 3) * 32;
    const __half* row = static_cast<const __half*>(j.values) + q * j.values_ld;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (q < x.q1 && c + i * 8 < j.K) w = __ldg(reinterpret_cast<const uint4*>(row + c + i * 8));
        reinterpret_cast<uint4*>(o.v[i >> 1].w)[i & 1] = w;
    }
}
template <typename T>
__device__ __forceinline__ void store_own(OwnRows& o, int half, uint8_t* tile, uint8_t* atom) {
    const int lane = threadIdx.x & 31, row = half * 8 + (lane >> 2);
    auto& v = reinterpret_cast<blockq::Vals<T>(&)[2]>(o.v);
    float amax = fmaxf(blockq::finite_max(v[0]), blockq::finite_max(v[1]));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
    const uint32_t s = blockq::scale_of<false>(amax);
    const float inv = blockq::inverse_scale(s);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint4 q;
        uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            w[c] = blockq::codes4<false>(v[i].get(4 * c) * inv, v[i].get(4 * c + 1) * inv, v[i].get(4 * c + 2) * inv,
                                         v[i].get(4 * c + 3) * inv);
        *reinterpret_cast<uint4*>(tile + row * 128 + ((((lane & 3) * 2 + i) ^ (row & 7)) << 4)) = q;
    }
    if ((lane & 3) == 0) *reinterpret_cast<uint32_t*>(atom + row * 16) = s;   // rows from 16 on: no output reads them
}

template <bool FP8, int BN, int CTAS, bool OWN = false>
__global__ void __launch_bounds__(kThreads, 1)
k_product(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
          const __grid_constant__ ProdJob j) {
    using S = Shape<FP8, BN, CTAS, OWN>;
    static_assert(!OWN || (FP8 && BN == 16 && CTAS == 1 && S::kHalves == 1), "rows are quantised 16 at a time");
    constexpr int kStep = FP8 ? kStepBytes : kStepBytes / 2;   // contraction values per step
    constexpr int BM = kBM * CTAS;
    extern __shared__ uint8_t raw[];
    __shared__ uint32_t tmem_slot;
    // (Aligned by an offset, not by a cast of the address, which would turn every access generic.)
    uint8_t* ring = raw + (-smem_addr(raw) & 1023u);
    uint8_t* scales = ring + S::kStages * S::kStage;
    uint8_t* turns = scales + kScaleSlots * S::kScaleBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(turns + kWriters * kTurn);
    uint64_t* empty = full + S::kStages;
    uint64_t* fixed = empty + S::kStages;
    uint64_t* landed = fixed + S::kStages;
    uint64_t* scales_full = landed + S::kStages;
    uint64_t* scales_empty = scales_full + kScaleSlots;
    uint64_t* scales_here = scales_empty + kScaleSlots;
    uint64_t* scales_there = scales_here + kScaleSlots;
    uint64_t* acc_full = scales_there + kScaleSlots;
    uint64_t* acc_empty = acc_full + S::kAccs;
    uint64_t* drain = acc_empty + S::kAccs;
    int* bound = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(full) + S::kBarBytes);
    int* cum = bound + j.groups + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // A pair takes a tile; otherwise a cluster takes one tile, each of its CTAs a part of the contraction.
    const int rank = CTAS == 2 || j.cluster > 1 ? int(cluster_rank()) : 0;

    if (warp == 3) columns_alloc<CTAS>(&tmem_slot, S::kCols);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(full + i, OWN ? 3 : 1);
            mbar_init(empty + i, 1);
            mbar_init(fixed + i, CTAS);
            mbar_init(landed + i, 1);
        }
        for (int i = 0; i < kScaleSlots; ++i) {
            mbar_init(scales_full + i, OWN ? 2 : 1);
            mbar_init(scales_there + i, 1);
            mbar_init(scales_empty + i, 1);
            mbar_init(scales_here + i, 1);
        }
        for (int i = 0; i < S::kAccs; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, 4 * S::kHalves * CTAS);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    int* dealt = cum + j.groups + 1;
    Groups g{bound, cum, dealt, int(blockIdx.x) / CTAS, false};
    if (j.grouping != kDense) {
        const int rows = j.grouping == kContraction ? j.K : j.grouping == kRowsA ? j.P : j.Q;
        const int high = j.grouping == kRowsB ? BN : BM;
        if (warp == 0) {
            // Bounds made rising and tiles added up, 32 groups at a time.
            int low = 0, tiles = 0;
            for (int i = 0; i <= j.groups; i += 32) {
                int b = i + lane <= j.groups ? min(max(j.off[i + lane], 0), rows) : 0;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(~0u, b, d);
                    if (lane >= d) b = max(b, o);
                }
                b = max(b, low);
                const int before = __shfl_up_sync(~0u, b, 1);
                // tiles of the group that ends at this bound
                int n = i + lane == 0 ? 0 : (b - (lane ? before : low) + high - 1) / high;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(~0u, n, d);
                    if (lane >= d) n += o;
                }
                if (i + lane <= j.groups) {
                    bound[i + lane] = b;
                    cum[i + lane] = tiles + n;
                }
                low = __shfl_sync(~0u, b, 31);
                tiles += __shfl_sync(~0u, n, 31);
            }
        }
        if (j.grouping == kContraction) {
            __syncthreads();
            for (int i = threadIdx.x; i < j.groups; i += kThreads) {
                int at = i;
                if (j.groups <= kDealGroups) {
                    const int size = bound[i + 1] - bound[i];
                    at = 0;
                    for (int o = 0; o < j.groups; ++o) {
                        const int other = bound[o + 1] - bound[o];
                        at += other > size || (other == size && o < i);
                    }
                }
                cum[at] = i;
            }
            __syncthreads();
            // The tiles of a group that do not make a full round go to the CTAs with the least to do so far,
            // longest groups first.  That takes about 1,300 cycles per group, and pays where the longest
            // group is far above the mean: 16 groups of 0 to 5,000 of 16,384 rows, 1,024 x 2,048, 85 -> 78 us; 16
            // equal groups, 55 -> 64 us.
            const int longest = bound[cum[0] + 1] - bound[cum[0]];
            g.deal = j.balance && 2LL * longest * j.groups > 3LL * (bound[j.groups] - bound[0]);
            if (g.deal) {
                // A CTA's load and number make one key, so that a rank is a count of smaller keys.
                const int lanes = int(j.by_lanes.d), left = int(j.by_tiles.d) % lanes, padded = (lanes + 3) / 4;
                const int share = lanes <= kThreads / 4 ? 4 : 2;        // threads that count for one key
                const int own = int(threadIdx.x) / share, sub = int(threadIdx.x) % share;
                int* load = dealt + j.groups + (-smem_addr(dealt + j.groups) & 15u) / 4;
                for (int i = threadIdx.x; i < 8 * padded; i += kThreads)
                    load[i] = i % (4 * padded) < lanes ? i % (4 * padded) : 0x7fffffff;
                for (int i = 0; i < j.groups; ++i) {
                    __syncthreads();
                    const int* now = load + (i & 1) * 4 * padded;
                    int* then = load + (~i & 1) * 4 * padded;
                    // a tile costs its steps, and starting and ending it about as much as four
                    const int cost = ((bound[cum[i] + 1] - bound[cum[i]]) / kStep + 4) << 9;
                    const int mine = own < lanes ? now[own] : 0;
                    int at = 0;
#pragma unroll 5
                    for (int o = sub; o < padded; o += share) {
                        const int4 k = reinterpret_cast<const int4*>(now)[o];
                        at += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
                    }
                    at += __shfl_xor_sync(~0u, at, 1);
                    if (share == 4) at += __shfl_xor_sync(~0u, at, 2);
                    if (own < lanes && sub == 0) {
                        then[own] = mine + (at < left ? cost : 0);
                        if (own == g.lane) dealt[i] = at < left ? int(j.by_tiles.d) - left + at : -1;
                    }
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    const int tiles = tile_count(j, g);
    const int first_tile = g.deal          ? 0
                           : CTAS == 2     ? int(blockIdx.x) / 2
                           : j.cluster > 1 ? rank * (tiles / j.split) + int(blockIdx.x) / j.cluster
                                           : int(blockIdx.x);
    const int stride = g.deal ? 1 : CTAS == 2 ? int(gridDim.x) / 2 : j.cluster > 1 ? tiles : int(gridDim.x);
    const int a_off = CTAS == 2 ? rank * kBM : 0;

    // Warps 0 and 1 run their loops as whole warps and elect a lane for the copies and MMAs only: addresses
    // and descriptors then stay in uniform registers.  With one lane running the loop an MMA step took
    // 700 cycles to issue, against the 512 that it takes to execute.
    if (warp == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        long long issued = 0;
        uint32_t on_landed = 0, landed_phase = 0;   // by stage: its last copies count on `landed`, whose next phase is this
        const int staged = FP8 && !OWN && j.narrow ? S::kStage / 2 : S::kStage;   // bytes per step
        // Weights are on their way before the quantiser has ended: A's copies of the first stages.
        int early = 0;
        if (CTAS == 1 && j.early_a && first_tile < tiles) {
            const Tile x = tile_at<BM, BN>(j, g, first_tile, kStep);
            if (elected())
                for (int k = x.k0; k < x.k1 && early < S::kStages; k += kStep, ++early) {
                    mbar_arrive_expect_tx(full + early, staged);
                    tma_3d<1>(smem_addr(ring) + early * S::kStage, &ma, k, x.p0, j.grouping == kRowsB ? x.e : 0,
                              smem_addr(full + early));
                }
            early = __reduce_max_sync(~0u, early);
        }
        if (j.after_quantize) grid_dep_wait();
        for (int t = first_tile; ok && t < tiles; t += stride) {
            const Tile x = tile_at<BM, BN>(j, g, t, kStep);
            if (x.p0 < 0) continue;
            const int ea = j.grouping == kRowsB ? x.e : 0, eb = j.grouping == kRowsA ? x.e : 0;
            const int b_off = CTAS == 2 ? rank * (tile_columns<BN, CTAS>(j, x) / 2) : 0;
            for (int k = x.k0; k < x.k1; k += kStep) {
                if (!(ok = __all_sync(~0u, wait(empty + stage, phase ^ 1)))) break;
                // A pair's copies all count on its first CTA's barrier.  Where rows have to be zeroed first, each
                // CTA's count on a barrier of its own, and the stage's barrier passes at once.
                const bool tail = j.grouping == kContraction && k + kStep > x.k1;
                if (elected()) {
                    const uint32_t a = smem_addr(ring) + stage * S::kStage, b = a + S::kATile;
                    uint64_t* counted = (tail ? landed : full) + stage;
                    const uint32_t bar = CTAS == 1 ? smem_addr(counted) : address_in(smem_addr(counted), tail ? rank : 0);
                    const bool begun = CTAS == 1 && issued < early;
                    if (tail) {
                        mbar_arrive_expect_tx(landed + stage, S::kStage);
                        if (CTAS == 1 || rank == 0) mbar_arrive(full + stage);
                    } else if (!begun && (CTAS == 1 || rank == 0)) {
                        mbar_arrive_expect_tx(full + stage, OWN ? S::kATile : staged * CTAS);
                    }
                    if (begun) {
                    } else if (j.a_mn) {
                        for (int c = 0; c < kBM / 64; ++c) tma_3d<CTAS>(a + c * 8192, &ma, x.p0 + a_off + c * 64, k, ea, bar);
                    } else {
                        tma_3d<CTAS>(a, &ma, k, x.p0 + a_off, ea, bar);
                    }
                    if (OWN) {
                    } else if (j.b_mn) {
                        for (int c = 0; c < S::kBRows / 64; ++c)
                            tma_3d<CTAS>(b + c * 8192, &mb, x.q0 + b_off + c * 64, k, eb, bar);
                    } else {
                        tma_3d<CTAS>(b, &mb, k, x.q0 + b_off, eb, bar);
                    }
                }
                __syncwarp();
                on_landed = (on_landed & ~(1u << stage)) | uint32_t(tail) << stage;
                landed_phase ^= uint32_t(tail) << stage;
                ++issued;
                if (++stage == S::kStages) stage = 0, phase ^= 1;
            }
        }
        // Every copy has landed before the CTA may end: those that no MMA waited for are waited for here (a pair's by its
        // first CTA, since the other one cannot end before it; those on `landed` by the CTA that they go to).
        for (int i = 0; !ok && i < S::kStages && issued - i > 0; ++i) {
            const long long n = issued - 1 - i;
            const int at = int(n % S::kStages);
            if (on_landed >> at & 1) wait(landed + at, (landed_phase >> at & 1) ^ 1);
            else if (CTAS == 1 || rank == 0) wait(full + at, uint32_t(n / S::kStages) & 1);
        }
    } else if (warp == 1) {
        if (CTAS == 1 || rank == 0) {
            int stage = 0, acc = 0, slot = 0;
            uint32_t phase = 0, acc_phase = 0, fixed_phase = 0, slot_phase = 0;
            bool ok = true;
            const uint32_t a_k = (j.a_mn ? 2048 : 32) >> 4, b_k = (j.b_mn ? 2048 : 32) >> 4;
            const uint32_t first_a = smem_addr(ring), first_b = first_a + S::kATile;
            const bool narrow = FP8 && !OWN && j.narrow;
            const uint64_t desc_a = narrow ? desc_narrow(first_a) : j.a_mn ? desc_mnmajor(first_a) : desc_kmajor(first_a);
            const uint64_t desc_b = narrow ? desc_narrow(first_b) : j.b_mn ? desc_mnmajor(first_b) : desc_kmajor(first_b);
            for (int t = first_tile; ok && t < tiles; t += stride) {
                const Tile x = tile_at<BM, BN>(j, g, t, kStep);
                if (x.p0 < 0) continue;
                if (!(ok = __all_sync(~0u, wait(acc_empty + acc, acc_phase ^ 1)))) break;
                const uint32_t d = tmem + acc * BN, idesc = j.idesc | uint32_t(tile_columns<BN, CTAS>(j, x) >> 3) << 17;
                uint32_t byte = 0;
                for (int k = x.k0; k < x.k1; k += kStep) {
                    if (j.grouping == kContraction && k + kStep > x.k1) {
                        ok = wait_all<CTAS>(fixed + stage, (fixed_phase >> stage) & 1);
                        fixed_phase ^= 1u << stage;
                    } else {
                        ok = wait(full + stage, phase);
                    }
                    if (FP8 && byte == 0) ok = ok && wait(scales_full + slot, slot_phase);
                    if (!(ok = __all_sync(~0u, ok))) break;
                    fence_after_sync();
                    const bool group_ends = FP8 && (byte == S::kGroup - 1 || k + kStep >= x.k1);
                    if (elected()) {
                        const uint64_t da = desc_a + uint32_t(stage * (S::kStage >> 4));
                        const uint64_t db = desc_b + uint32_t(stage * (S::kStage >> 4));
                        const uint32_t more = k > x.k0;
                        if constexpr (FP8) {
                            const uint32_t sf = tmem + S::kAccs * BN + slot * S::kScaleCols;
                            if (byte == 0) {
                                const uint32_t src = smem_addr(scales) + slot * S::kScaleBytes;
#pragma unroll
                                for (int i = 0; i <= S::kAtomsB; ++i) scales_to_tmem<CTAS>(sf + 4 * i, src + i * kAtom);
                            }
                            const uint32_t id = idesc | (byte << 4) | (byte << 29);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (i < 2 || !narrow)
                                    mma_block_scaled<CTAS>(d, da + i * 2, db + i * 2, id, sf, sf + 4, i ? 1 : more);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) mma_half<CTAS>(d, da + i * a_k, db + i * b_k, idesc, i ? 1 : more);
                        }
                        commit_all<CTAS>(empty + stage);
                        if (group_ends) commit_all<CTAS>(scales_empty + slot);
                    }
                    __syncwarp();
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                    if (FP8) {
                        byte = group_ends ? 0 : byte + 1;
                        if (group_ends && ++slot == kScaleSlots) slot = 0, slot_phase ^= 1;
                    }
                }
                if (elected()) commit_all<CTAS>(acc_full + acc);
                __syncwarp();
                if (++acc == S::kAccs) acc = 0, acc_phase ^= 1;
            }
            if (!ok) {   // let the MMAs in flight land before TMEM goes
                if (elected()) commit_all<CTAS>(drain);
                __syncwarp();
                wait(drain, 0);
            }
        }
        if constexpr (FP8 && CTAS == 2) {
            // The second CTA tells the first that its scales are in place.  Its release of cluster scope takes
            // about as long as a step, and here it holds up no load.
            if (lane == 0 && rank == 1) {
                int slot = 0;
                uint32_t phase = 0;
                bool ok = true;
                for (int t = first_tile; ok && t < tiles; t += stride) {
                    const Tile x = tile_at<BM, BN>(j, g, t, kStep);
                    for (int k = x.k0; k < x.k1; k += S::kGroup * kStep) {
                        if (!(ok = wait(scales_here + slot, phase))) break;
                        arrive_first<CTAS>(scales_there + slot, rank, true);
                        if (++slot == kScaleSlots) slot = 0, phase ^= 1;
                    }
                }
            }
        }
    } else if (warp == 2 || (FP8 && warp == 3) || (OWN && (warp == 8 || warp == 9))) {
        [[maybe_unused]] const int turn = warp & 1, half = warp >> 3;   // which atoms; OWN: which rows
        [[maybe_unused]] int stage = OWN ? turn : 0;
        [[maybe_unused]] uint32_t stage_phase = 0;
        uint32_t phase = 0;
        [[maybe_unused]] bool ok = true;
        if constexpr (FP8) {
            if (j.after_quantize) grid_dep_wait();
            const int blocks = (j.K + kBlock - 1) / kBlock;
            const ScaleWay way_a = scale_way(j.sa, j.a_rows, j.grouping == kRowsA);
            const ScaleWay way_b = scale_way(j.sb, j.b_rows, j.grouping == kRowsB);
            RawScales raw_a, raw_b[S::kAtomsB];
            OwnRows own;
            auto load = [&](const Tile& x, int k) {
                const int ea = j.grouping == kRowsB ? x.e : 0, eb = j.grouping == kRowsA ? x.e : 0;
                load_scales(raw_a, j.sa, way_a, ea, x.p0 + a_off, j.a_rows, k / kBlock, blocks);
                if constexpr (OWN) {
                    load_own(own, j, x, half, k);
                } else {
#pragma unroll
                    for (int i = 0; i < S::kAtomsB; ++i)
                        load_scales(raw_b[i], j.sb, way_b, eb, x.q0 + 128 * i, j.b_rows, k / kBlock, blocks);
                }
            };
            // The two warps (of OWN: two pairs) take every other group each.
            int t = first_tile, k = 0;
            Tile x{};
            // To the first step of a tile that has one, and from group to group.
            auto settle = [&] {
                while (t < tiles) {
                    x = tile_at<BM, BN>(j, g, t, kStep);
                    k = x.k0;
                    if (x.k0 < x.k1) break;
                    t += stride;
                }
            };
            auto advance = [&] {
                k += S::kGroup * kStep;
                if (k >= x.k1) {
                    t += stride;
                    settle();
                }
            };
            settle();
            if (turn == 1 && t < tiles) advance();
            if (t < tiles) load(x, k);
            int slot = turn;
            for (bool more = t < tiles; more;) {
                if (!__all_sync(~0u, wait(scales_empty + slot, phase ^ 1))) break;
                uint8_t* dst = scales + slot * S::kScaleBytes;
                if (!OWN || half == 0) store_scales(raw_a, way_a, dst);
                if constexpr (OWN) {
                    if (!__all_sync(~0u, wait(empty + stage, stage_phase ^ 1))) break;
                    uint8_t* tile = ring + stage * S::kStage + S::kATile;
                    if (j.values_type == kF16) store_own<__half>(own, half, tile, dst + kAtom);
                    else store_own<__nv_bfloat16>(own, half, tile, dst + kAtom);
                } else {
#pragma unroll
                    for (int i = 0; i < S::kAtomsB; ++i) store_scales(raw_b[i], way_b, dst + (1 + i) * kAtom);
                }
                fence_async_smem();
                __syncwarp();
                if constexpr (OWN) {
                    if (lane == 0) mbar_arrive(full + stage);
                    if ((stage += 2) >= S::kStages) stage -= S::kStages, stage_phase ^= 1;
                }
                // The first CTA's warp also takes in the other one's word, an acquire of cluster scope that would
                // cost the MMA warp 480 cycles per group.
                if (CTAS == 2 && rank == 0 && !__all_sync(~0u, wait_all<CTAS>(scales_there + slot, phase))) break;
                if (lane == 0) mbar_arrive((rank == 0 || CTAS == 1 ? scales_full : scales_here) + slot);
                if ((slot += 2) >= kScaleSlots) slot -= kScaleSlots, phase ^= 1;
                advance();
                if (t < tiles) advance();
                more = t < tiles;
                if (more) load(x, k);
            }
        } else if (j.grouping == kContraction) {
            // (This warp waits on barriers that only these steps use: it is no part of the ring's flow, so a
            // barrier that every step passes could run two phases ahead of it.)
            uint32_t landed_phase = 0;
            long long passed = 0;   // steps since the last wait: it goes on while they do
            for (int t = first_tile; ok && t < tiles; t += stride) {
                const Tile x = tile_at<BM, BN>(j, g, t, kStep);
                if (x.p0 < 0) continue;
                for (int k = x.k0; k < x.k1; k += kStep, ++passed) {
                    const int rows = x.k1 - k;
                    if (rows < kStep) {
                        if (!(ok = __all_sync(~0u, wait(landed + stage, (landed_phase >> stage) & 1, passed * kStepCycles)))) break;
                        landed_phase ^= 1u << stage;
                        passed = 0;
                        // eight lanes to a row of 128 bytes
                        uint8_t* at = ring + stage * S::kStage + (lane & 7) * 16;
#pragma unroll
                        for (int c = 0; c < S::kStage / 8192; ++c)
                            for (int r = rows + (lane >> 3); r < kStep; r += 4)
                                *reinterpret_cast<uint4*>(at + c * 8192 + r * 128) = make_uint4(0, 0, 0, 0);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) arrive_first<CTAS>(fixed + stage, rank, true);
                    }
                    if (++stage == S::kStages) stage = 0;
                }
            }
        }
    } else if (warp >= 4 && warp < 4 + 4 * S::kHalves) {
        const int quad = warp & 3, half = (warp - 4) >> 2, col = half * S::kWide;
        uint8_t* turn = turns + (warp - 4) * kTurn;
        float* bias = reinterpret_cast<float*>(bound) + (warp - 4) * S::kWide;
        int acc = 0, bias_q = -1;
        uint32_t acc_phase = 0;
        for (int t = first_tile; t < tiles; t += stride) {
            const Tile x = tile_at<BM, BN>(j, g, t, kStep);
            if (x.p0 < 0) continue;
            if (j.bias && !j.swapped && bias_q != x.q0) {
                for (int i = lane; i < S::kWide; i += 32)
                    bias[i] = x.q0 + col + i < j.Q ? load_elem(j.bias, j.bias_type, x.q0 + col + i) : 0.f;
                __syncwarp();
                bias_q = x.q0;
            }
            if (!__all_sync(~0u, wait(acc_full + acc, acc_phase, (x.k1 - x.k0) / kStep * kStepCycles))) break;
            fence_after_sync();
            uint32_t v[S::kWide];
            if (x.k0 < x.k1) {
                tmem_load<S::kWide>(tmem + (uint32_t(quad * 32) << 16) + acc * BN + col, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < S::kWide; ++i) asm volatile("" : "+r"(v[i]));
            } else {
#pragma unroll
                for (int i = 0; i < S::kWide; ++i) v[i] = 0;
            }
            fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_first<CTAS>(acc_empty + acc, rank, false);
            if (++acc == S::kAccs) acc = 0, acc_phase ^= 1;

            const int p0 = x.p0 + a_off + quad * 32, q0 = x.q0 + col;
            const long long base = x.part * j.split_stride + (j.grouping == kContraction ? x.e * j.out_batch : 0);
            if (CTAS == 1 && j.cluster > 1) {
                // every MMA of this CTA is done with the ring
                put_part<BN, S::kWide>(j, v, ring, quad * 32 + lane, col);
            } else if (j.swapped) {
                if (j.out_type == kF32) write_columns<float, S::kWide>(j, v, base, p0 + lane, x.p1, q0, x.q1);
                else if (j.out_type == kF16) write_columns<__half, S::kWide>(j, v, base, p0 + lane, x.p1, q0, x.q1);
                else write_columns<__nv_bfloat16, S::kWide>(j, v, base, p0 + lane, x.p1, q0, x.q1);
            } else {
                if (j.out_type == kF32) write_rows<float, S::kWide>(j, v, bias, turn, base, p0, x.p1, q0, x.q1);
                else if (j.out_type == kF16) write_rows<__half, S::kWide>(j, v, bias, turn, base, p0, x.p1, q0, x.q1);
                else write_rows<__nv_bfloat16, S::kWide>(j, v, bias, turn, base, p0, x.p1, q0, x.q1);
            }
            __syncwarp();
        }
        if (j.zero_outside) {
            // A warp takes a row at a time: the rows before the first group, then those behind the last.  (Bytes of a
            // row, and the row after the last one, may pass 2^31.)
            const int before = bound[0], skip = bound[j.groups] - before, size = j.out_type == kF32 ? 4 : 2;
            constexpr int kWarps = 4 * S::kHalves;
            for (long long i = int(blockIdx.x) * kWarps + warp - 4; i < j.zero_rows - skip; i += int(gridDim.x) * kWarps) {
                uint8_t* row = static_cast<uint8_t*>(j.out) + (i < before ? i : i + skip) * j.out_ld * size;
                const long long bytes = (long long)j.cols * size, whole = j.out_vec ? bytes / 16 * 16 : 0;
                for (long long c = lane * 16; c < whole; c += 32 * 16) *reinterpret_cast<uint4*>(row + c) = make_uint4(0, 0, 0, 0);
                for (long long c = whole + lane * 2; c < bytes; c += 32 * 2) *reinterpret_cast<uint16_t*>(row + c) = 0;
            }
        }
    }
    if (CTAS == 1 && j.cluster > 1) {
        __syncwarp();
        cluster_sync();
        if (warp >= 4 && first_tile < tiles) {
            const Tile x = tile_at<BM, BN>(j, g, first_tile, kStep);
            if (j.cluster == 2) join_cluster<BN, 2>(j, x, rank, smem_addr(ring));
            else if (j.cluster == 4) join_cluster<BN, 4>(j, x, rank, smem_addr(ring));
            else join_cluster<BN, 8>(j, x, rank, smem_addr(ring));
        }
    }
    fence_before_sync();
    __syncthreads();
    // No CTA ends while another one may still read its shared memory or signal its barriers.
    if (CTAS == 2 || j.cluster > 1) cluster_sync();
    fence_after_sync();
    if (warp == 3) columns_free<CTAS>(tmem, S::kCols);
}

// out = sum of the parts in order, plus the bias of the column.  G threads share an output: each adds a run of
// parts, then the runs are added in order.  One where outputs are many; eight where parts are (144 parts of
// 64 x 128: 7.2 us with one, whose loads follow one another, 3.7 with eight).
template <int G>
__global__ void __launch_bounds__(256) k_join_parts(const float* part, int parts, long long stride, int rows, int cols,
                                                    void* out, int out_type, long long out_ld, const void* bias,
                                                    int bias_type) {
    constexpr int kOutputs = 256 / G;
    __shared__ float sh[G][kOutputs];
    const long long n = (long long)rows * cols;
    const int o = int(threadIdx.x) % kOutputs, run = int(threadIdx.x) / kOutputs, per = (parts + G - 1) / G;
    const int first = run * per, last = min(parts, first + per);
    for (long long i0 = (long long)blockIdx.x * kOutputs; i0 < n; i0 += (long long)gridDim.x * kOutputs) {
        const long long i = i0 + o;
        float s = 0.f;
        if (i < n) {
#pragma unroll 16
            for (int k = first; k < last; ++k) s += part[k * stride + i];
        }
        if constexpr (G > 1) {
            sh[run][o] = s;
            __syncthreads();
            s = sh[0][o];
#pragma unroll
            for (int r = 1; r < G; ++r) s += sh[r][o];
            __syncthreads();
        }
        if (i < n && run == 0) {
            const int r = int(i / cols), c = int(i % cols);
            if (bias) s += load_elem(bias, bias_type, c);
            store_elem(out, out_type, r * out_ld + c, s);
        }
    }
}

// ---- host --------------------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    if (!fn) fail(AEISU_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    return fn;
}

// Operand map: innermost the contiguous direction in boxes of 128 bytes (narrow: 64), `high` of the other.
CUtensorMap operand_map(const MatrixRef& m, int high, bool narrow = false) {
    const int eb = elem_bytes(m.type);
    const int inner = m.trans ? m.rows : m.cols, outer = m.trans ? m.cols : m.rows;
    CUtensorMap map{};
    const cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(outer), cuuint64_t(m.batch)};
    const long long batch = m.batch > 1 ? m.batch_stride : ((m.ld * outer * eb + 15) / 16 * 16) / eb;
    const cuuint64_t strides[2] = {cuuint64_t(m.ld) * eb, cuuint64_t(batch) * eb};
    const cuuint32_t box[3] = {cuuint32_t((narrow ? kStepBytes / 2 : kStepBytes) / eb), cuuint32_t(high), 1};
    const cuuint32_t one[3] = {1, 1, 1};
    const CUtensorMapDataType type = m.type == kF16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : m.type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUresult r = encoder()(&map, type, 3, const_cast<void*>(m.ptr), dims, strides, box, one,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) fail(AEISU_ERR_CUDA, "cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
    return map;
}

void check_operand(const MatrixRef& m, const ScaleRef* s) {
    require(m.ptr, "tensor pointer is null");
    const int eb = elem_bytes(m.type);
    require(m.rows >= 1 && m.cols >= 1 && m.batch >= 1, "matrix sizes are out of range");
    require(m.ld >= (m.trans ? m.rows : m.cols), "matrix rows overlap");
    require(aligned(m.ptr, 16) && m.ld * eb % 16 == 0 && (m.batch == 1 || m.batch_stride * eb % 16 == 0),
            "operand rows must start on 16-byte boundaries");
    require(is_code(m.type) == (s != nullptr), "FP8 operands, and only they, come with scales");
    require(is_code(m.type) || m.type == kF16 || m.type == kBF16, "operands must be FP8, float16 or bfloat16");
    if (s) {
        require(s->ptr && (s->shift == 0 || s->shift == 7), "blocks have 1 or 128 rows");
        require(!m.trans, "FP8 operands are stored row by row");
    }
}

int sm_count(int device) {
    static std::mutex mu;
    static int known[64] = {};
    require(device >= 0 && device < 64, "device index is out of range");
    std::lock_guard<std::mutex> lock(mu);
    if (!known[device]) AEISU_CUDA(cudaDeviceGetAttribute(&known[device], cudaDevAttrMultiProcessorCount, device));
    return known[device];
}

template <bool FP8, int BN, int CTAS, bool OWN = false>
void launch(const CUtensorMap& a, const CUtensorMap& b, const ProdJob& j, long long tiles, int device,
            cudaStream_t stream) {
    using S = Shape<FP8, BN, CTAS, OWN>;
    constexpr size_t most = S::kSmem + std::max(S::kBias, 2 * (kMaxGroups + 1) * sizeof(int));
    static_assert(most <= 227 * 1024, "shared memory of a CTA");
    const size_t lists = j.balance ? size_t(j.groups + 2 * j.by_lanes.d + 16) : 0;
    const size_t smem = S::kSmem + (j.grouping == kDense ? S::kBias : (2 * size_t(j.groups + 1) + lists) * sizeof(int));
    require(smem <= most, "too many groups");
    static std::mutex mu;
    static bool ready[64] = {};
    const int sms = sm_count(device);
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[device]) {
            AEISU_CUDA(cudaFuncSetAttribute(k_product<FP8, BN, CTAS, OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            int(most)));
            ready[device] = true;
        }
    }
    const int cluster = CTAS == 2 ? 2 : j.cluster;
    const long long ctas = CTAS == 2 ? 2 * std::min<long long>(tiles, sms / 2)
                                     : j.cluster > 1 ? tiles : std::min<long long>(tiles, sms);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(ctas), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = j.after_quantize;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    AEISU_CUDA(cudaLaunchKernelEx(&cfg, k_product<FP8, BN, CTAS, OWN>, a, b, j));
}

// Tile of a product: columns, and CTAs that share it.
struct TileShape {
    int bn, ctas;
    int rows() const { return kBM * ctas; }
    int b_rows() const { return bn / ctas; }
};

template <bool FP8>
void launch_shape(TileShape s, const CUtensorMap& a, const CUtensorMap& b, const ProdJob& j, long long tiles, int device,
                  cudaStream_t stream) {
    if constexpr (FP8)
        if (j.values) return launch<true, 16, 1, true>(a, b, j, tiles, device, stream);
    if (s.ctas == 2) return launch<FP8, 256, 2>(a, b, j, tiles, device, stream);
    switch (s.bn) {
        case 16: return launch<FP8, 16, 1>(a, b, j, tiles, device, stream);
        case 32: return launch<FP8, 32, 1>(a, b, j, tiles, device, stream);
        case 64: return launch<FP8, 64, 1>(a, b, j, tiles, device, stream);
        case 256: return launch<FP8, 256, 1>(a, b, j, tiles, device, stream);
        default: return launch<FP8, 128, 1>(a, b, j, tiles, device, stream);
    }
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// The tile for P x Q outputs, `count` of them: the one with the shortest time by waves of tiles over the
// SMs.  A step takes as long as the operand bytes that a CTA stages, A's 128 rows and its share of B's
// (256 rows: 512 cycles); starting and ending a tile, as long as 250 rows, 750 for a pair, whose CTAs
// signal each other.
TileShape choose_tile(long long row_tiles_of_128, int q, long long count, long long steps, bool pairs, int least,
                      int sms) {
    TileShape best{least, 1};
    double time = 0;
    for (const TileShape s : {TileShape{16, 1}, TileShape{32, 1}, TileShape{64, 1}, TileShape{128, 1}, TileShape{256, 1},
                              TileShape{256, 2}}) {
        if (s.bn < least || (s.ctas == 2 && !pairs)) continue;
        const long long tiles = ceil_div(row_tiles_of_128, s.ctas) * ceil_div(q, s.bn) * count;
        const double t = double(ceil_div(tiles, sms / s.ctas)) *
                         (double(steps) * (kBM + s.b_rows()) + (s.ctas == 2 ? 750 : 250));
        if (time == 0 || t < time) best = s, time = t;
    }
    return best;
}

uint32_t instruction(const MatrixRef& a, const MatrixRef& b, TileShape s) {
    const uint32_t size = uint32_t(s.rows() >> 4) << 24;
    if (is_code(a.type))
        return size | (uint32_t(a.type == kE5M2) << 7) | (uint32_t(b.type == kE5M2) << 10) | (1u << 23);
    const uint32_t f = a.type == kBF16 ? 1 : 0;
    return size | (1u << 4) | (f << 7) | (f << 10) | (uint32_t(a.trans) << 15) | (uint32_t(b.trans) << 16);
}

// How a dense product is cut: which side lies along the TMEM lanes, the tile and the parts of the
// contraction.
struct Plan {
    bool swap;
    TileShape tile;
    int split, steps;   // steps of the contraction per part
    int cluster;        // parts of a cluster (split), or 1: parts joined by a kernel
};

Plan plan_dense(int m, int n, int k, int sms) {
    Plan p{};
    const int steps = (k + kStepBytes - 1) / kStepBytes;
    // Few rows: the weights take the 128 lanes, so that no lane idles, and the rows the columns.
    p.swap = m <= 64 && n > m;
    const int P = p.swap ? n : m, Q = p.swap ? m : n;
    p.tile = choose_tile(ceil_div(P, kBM), Q, 1, steps, P > kBM, 16, sms);
    // Where one CTA per 128 rows and up to 128 columns leaves half of the SMs over, each takes as many columns
    // as there are, so that A is staged once, and the contraction is cut instead: into 2, 4 or 8 parts of at
    // least two steps, the CTAs of a cluster, which need no second kernel; where that fills less than half of
    // the SMs and the contraction is long, into as many parts as fill them, of at least eight steps, joined
    // by a kernel.
    TileShape widest{16, 1};
    while (widest.bn < std::min(Q, 128)) widest.bn *= 2;
    const long long t = ceil_div(P, kBM) * ceil_div(Q, widest.bn);
    if (t * 2 <= sms && steps >= 4) p.tile = widest;
    p.cluster = p.split = 1;
    p.steps = steps;
    if (t * 2 <= sms && steps >= 4) {
        while (p.cluster < 8 && t * p.cluster * 2 <= sms && steps >= 4 * p.cluster) p.cluster *= 2;
        const long long wide = std::min<long long>(sms / t, steps / 8);
        if (t < sms && wide >= 2 * p.cluster) {
            p.cluster = 1;
            p.split = int(wide);
        } else {
            p.split = p.cluster;
        }
        p.steps = (steps + p.split - 1) / p.split;
        if (p.cluster == 1) p.split = (steps + p.steps - 1) / p.steps;
    }
    return p;
}

Divider divider(long long d) {
    Divider v{0, 0, uint32_t(d)};
    while ((2ull << v.shift) < uint64_t(d)) ++v.shift;
    v.mul = uint32_t(((1ull << (32 + v.shift)) + uint64_t(d) - 1) / uint64_t(d));
    return v;
}
// Tiles of the job, and the divisions that number them.
void lay_tiles(ProdJob& j, TileShape s) {
    j.tp = int(ceil_div(j.P, s.rows()));
    j.tq = int(ceil_div(j.Q, s.bn));
    const long long all = (long long)j.tp * j.tq;
    require(all < (1LL << 28), "matrix is too large");
    j.by_tiles = divider(all);
    j.by_band = divider(kBand * (long long)j.tq);
    j.by_tp = divider(j.tp);
    j.by_rest = divider(std::max(1, j.tp % kBand));
}

bool whole_rows(const void* p, int type, long long ld, long long batch) {
    return aligned(p, 32) && ld * elem_bytes(type) % 32 == 0 && batch * elem_bytes(type) % 32 == 0;
}

}  // namespace

size_t product_workspace(int m, int n, int k, int device) {
    const Plan p = plan_dense(m, n, k, sm_count(device));
    return p.split > p.cluster ? size_t(p.split) * m * n * sizeof(float) : 0;
}

namespace {

constexpr int kOwnRows = 16;   // rows that a product quantises itself

// Whether the kernel quantises the rows of x itself: few of them, 16-bit and aligned.
bool takes_values(const MatrixRef& x, long long rows) {
    return (x.type == kF16 || x.type == kBF16) && aligned(x.ptr, 16) && x.ld % 8 == 0 && x.cols % 8 == 0 &&
           rows <= kOwnRows;
}
void give_values(ProdJob& j, const MatrixRef& x) {
    j.values = x.ptr;
    j.values_type = x.type;
    j.values_ld = x.ld;
}
// x as the operand that the kernel makes of it.
MatrixRef as_codes(const MatrixRef& x) {
    MatrixRef m = x;
    m.type = kE4M3;
    return m;
}

void dense(const MatrixRef& a, const ScaleRef& sa, const MatrixRef& b, const ScaleRef& sb, const ProductOut& out,
           void* workspace, size_t workspace_bytes, const MatrixRef* values, bool after_quantize, int device,
           cudaStream_t stream) {
    require(a.batch == 1 && b.batch == 1 && a.cols == b.cols, "contraction sizes differ");
    require(out.ptr && out.type >= kF32 && out.type <= kBF16 && out.ld >= b.rows, "output is out of range");
    OnDevice on(device);
    const Plan pl = plan_dense(a.rows, b.rows, a.cols, sm_count(device));
    const size_t need = pl.split > pl.cluster ? size_t(pl.split) * a.rows * b.rows * sizeof(float) : 0;
    require(need == 0 || (workspace && workspace_bytes >= need), "workspace is too small");
    const MatrixRef& A = pl.swap ? b : a;
    const MatrixRef& B = pl.swap ? a : b;
    ProdJob j{};
    j.P = A.rows;
    j.Q = B.rows;
    j.K = A.cols;
    j.idesc = instruction(A, B, pl.tile);
    j.sa = pl.swap ? sb : sa;
    j.sb = pl.swap ? sa : sb;
    j.a_rows = A.rows;
    j.b_rows = B.rows;
    j.swapped = pl.swap;
    j.cols = b.rows;
    lay_tiles(j, pl.tile);
    j.split = pl.split;
    j.steps_per_split = pl.steps;
    j.cluster = pl.cluster;
    j.after_quantize = after_quantize;
    j.early_a = after_quantize && pl.swap;
    if (values) {
        require(pl.swap && pl.tile.bn == kOwnRows, "rows are quantised 16 at a time");
        give_values(j, *values);
    }
    if (pl.split > pl.cluster) {
        j.out = workspace;
        j.out_type = kF32;
        j.out_ld = b.rows;
        j.split_stride = (long long)a.rows * b.rows;
    } else {
        j.out = out.ptr;
        j.out_type = out.type;
        j.out_ld = out.ld;
        j.bias = out.bias;
        j.bias_type = out.bias_type;
    }
    j.out_vec = whole_rows(j.out, j.out_type, j.out_ld, j.split_stride);
    const long long tiles = ceil_div(j.P, pl.tile.rows()) * ceil_div(j.Q, pl.tile.bn) * pl.split;
    require(tiles < (1LL << 30), "matrix is too large");
    j.narrow = !values && j.K <= kNarrow;
    const CUtensorMap ma = operand_map(A, kBM, j.narrow), mb = values ? ma : operand_map(B, pl.tile.b_rows(), j.narrow);
    launch_shape<true>(pl.tile, ma, mb, j, tiles, device, stream);
    if (pl.split > pl.cluster) {
        const long long n = (long long)a.rows * b.rows;
        const bool many = pl.split >= 32;
        const auto join = many ? k_join_parts<8> : k_join_parts<1>;
        const int per = many ? 32 : 256;
        join<<<unsigned(std::min<long long>((n + per - 1) / per, 148 * 8)), 256, 0, stream>>>(
            static_cast<const float*>(workspace), pl.split, j.split_stride, a.rows, b.rows, out.ptr, out.type, out.ld,
            out.bias, out.bias_type);
        AEISU_CUDA(cudaGetLastError());
    }
}

void grouped(const MatrixRef& x, const ScaleRef* sx, const MatrixRef& b, const ScaleRef* sb, const int* off,
             const ProductOut& out, bool zero_outside, const MatrixRef* values, bool after_quantize, int device,
             cudaStream_t stream) {
    require(x.batch == 1 && !x.trans && x.cols == b.cols, "contraction sizes differ");
    require((sx != nullptr) == (sb != nullptr) && (sx || x.type == b.type), "operand types do not go together");
    require(off && aligned(off, 4) && b.batch <= kMaxGroups, "a grouped product has offsets and at most 1024 groups");
    require(out.ptr && out.type >= kF32 && out.type <= kBF16 && out.ld >= b.rows && !out.bias, "output is out of range");
    OnDevice on(device);
    const bool fp8 = sx != nullptr;
    // Few rows per group on average: as for a dense product, the weights take the lanes.
    const int mean = (x.rows + b.batch - 1) / b.batch;
    const bool swap = mean <= 64 && b.rows >= kBM;
    ProdJob j{};
    const MatrixRef& A = swap ? b : x;
    const MatrixRef& B = swap ? x : b;
    // Rows per group are known on the GPU only: full row tiles are counted as if groups were even.  Pairs, whose
    // rows are twice as high, where groups have three of theirs on average (16-bit, 16 groups of 1,024 rows,
    // 1,024 x 2,048: 58 us in pairs, 66 us without; FP8, 8 groups of about 512, 2,048 x 2,048: 30 and 25 us).
    const int steps = int(ceil_div((long long)x.cols * elem_bytes(x.type), kStepBytes));
    const TileShape tile =
        swap ? choose_tile(ceil_div(b.rows, kBM) * b.batch, mean, 1, steps, false, 16, sm_count(device))
             : choose_tile(ceil_div(mean, kBM) * b.batch, b.rows, 1, steps, mean >= 6 * kBM, b.trans ? 64 : 16,
                           sm_count(device));
    j.P = A.rows;
    j.Q = B.rows;
    j.K = A.cols;
    j.grouping = swap ? kRowsB : kRowsA;
    j.groups = b.batch;
    j.off = off;
    j.a_mn = A.trans;
    j.b_mn = B.trans;
    j.idesc = instruction(A, B, tile);
    if (fp8) {
        j.sa = swap ? *sb : *sx;
        j.sb = swap ? *sx : *sb;
    }
    j.a_rows = A.rows;
    j.b_rows = B.rows;
    j.out = out.ptr;
    j.out_type = out.type;
    j.out_ld = out.ld;
    j.swapped = swap;
    j.cols = b.rows;
    lay_tiles(j, tile);
    j.split = j.cluster = 1;
    j.after_quantize = after_quantize;
    j.early_a = after_quantize && swap && fp8;
    if (values) {
        require(swap && tile.bn == kOwnRows, "rows are quantised 16 at a time");
        give_values(j, *values);
    }
    j.zero_outside = zero_outside;
    j.zero_rows = x.rows;
    j.out_vec = whole_rows(out.ptr, out.type, out.ld, 0);
    // Each group has at most one partly filled row tile.
    const int high = swap ? tile.bn : tile.rows(), wide = swap ? tile.rows() : tile.bn;
    const long long tiles = (ceil_div(x.rows, high) + std::min(b.batch, x.rows)) * ceil_div(b.rows, wide);
    require(tiles < (1LL << 30), "matrix is too large");
    j.narrow = fp8 && !values && j.K <= kNarrow;
    const CUtensorMap ma = operand_map(A, A.trans ? 64 : kBM, j.narrow);
    const CUtensorMap mb = values ? ma : operand_map(B, B.trans ? 64 : tile.b_rows(), j.narrow);
    if (fp8) launch_shape<true>(tile, ma, mb, j, tiles, device, stream);
    else launch_shape<false>(tile, ma, mb, j, tiles, device, stream);
}

}  // namespace

void product(const MatrixRef& a, const ScaleRef& sa, const MatrixRef& b, const ScaleRef& sb, const ProductOut& out,
             void* workspace, size_t workspace_bytes, bool after_quantize, int device, cudaStream_t stream) {
    check_operand(a, &sa);
    check_operand(b, &sb);
    dense(a, sa, b, sb, out, workspace, workspace_bytes, nullptr, after_quantize, device, stream);
}

bool product_of_values(const MatrixRef& x, const MatrixRef& b, const ScaleRef& sb, const ProductOut& out,
                       void* workspace, size_t workspace_bytes, int device, cudaStream_t stream) {
    if (!takes_values(x, x.rows) || b.rows <= x.rows) return false;
    check_operand(b, &sb);
    require(x.ptr && x.rows >= 1 && x.ld >= x.cols && !x.trans, "matrix sizes are out of range");
    dense(as_codes(x), ScaleRef{sb.ptr, 0, x.rows, 0}, b, sb, out, workspace, workspace_bytes, &x, false, device, stream);
    return true;
}

void grouped_product(const MatrixRef& x, const ScaleRef* sx, const MatrixRef& b, const ScaleRef* sb, const int* off,
                     const ProductOut& out, bool zero_outside, bool after_quantize, int device, cudaStream_t stream) {
    check_operand(x, sx);
    check_operand(b, sb);
    grouped(x, sx, b, sb, off, out, zero_outside, nullptr, after_quantize, device, stream);
}

bool grouped_product_of_values(const MatrixRef& x, const MatrixRef& b, const ScaleRef& sb, const int* off,
                               const ProductOut& out, bool zero_outside, int device, cudaStream_t stream) {
    if (!takes_values(x, ceil_div(x.rows, b.batch)) || b.rows < kBM) return false;
    check_operand(b, &sb);
    require(x.ptr && x.rows >= 1 && x.ld >= x.cols && !x.trans, "matrix sizes are out of range");
    const ScaleRef none{sb.ptr, 0, x.rows, 0};
    grouped(as_codes(x), &none, b, &sb, off, out, zero_outside, &x, false, device, stream);
    return true;
}

void grouped_weight_gradient(const MatrixRef& g, const MatrixRef& x, const int* off, int groups, void* out,
                             int out_type, int device, cudaStream_t stream) {
    check_operand(g, nullptr);
    check_operand(x, nullptr);
    require(g.batch == 1 && x.batch == 1 && g.trans && x.trans && g.cols == x.cols && g.type == x.type,
            "contraction sizes differ");
    require(off && aligned(off, 4) && groups >= 1 && groups <= kMaxGroups, "a grouped product has offsets and at most 1024 groups");
    require(out && out_type >= kF32 && out_type <= kBF16 && aligned(out, elem_bytes(out_type)), "output is out of range");
    OnDevice on(device);
    ProdJob j{};
    const TileShape tile = choose_tile(ceil_div(g.rows, kBM), x.rows, groups, ceil_div(ceil_div(g.cols, groups), kStepBytes / 2),
                                       g.rows > kBM, 64, sm_count(device));
    j.P = g.rows;
    j.Q = x.rows;
    j.K = g.cols;
    j.grouping = kContraction;
    j.groups = groups;
    j.off = off;
    j.a_mn = j.b_mn = 1;
    j.idesc = instruction(g, x, tile);
    j.out = out;
    j.out_type = out_type;
    j.out_ld = x.rows;
    j.out_batch = (long long)g.rows * x.rows;
    j.cols = x.rows;
    lay_tiles(j, tile);
    j.split = j.cluster = 1;
    j.out_vec = whole_rows(out, out_type, j.out_ld, j.out_batch);
    const long long tiles = ceil_div(g.rows, tile.rows()) * ceil_div(x.rows, tile.bn) * groups;
    const int lanes = sm_count(device) / tile.ctas;
    j.by_lanes = divider(lanes);
    j.balance = groups <= kDealGroups && tiles > lanes && lanes <= kThreads / 2 &&
                g.cols < (1 << 27);   // a CTA's steps and number share an int
    require(tiles < (1LL << 30), "matrix is too large");
    launch_shape<false>(tile, operand_map(g, 64), operand_map(x, 64), j, tiles, device, stream);
}

int product_status(int device) {
    OnDevice on(device);
    int code = 0, none = 0;
    AEISU_CUDA(cudaDeviceSynchronize());
    AEISU_CUDA(cudaMemcpyFromSymbol(&code, g_product_error, sizeof(code)));
    if (code) AEISU_CUDA(cudaMemcpyToSymbol(g_product_error, &none, sizeof(none)));
    return code;
}

}  // namespace aeisu
