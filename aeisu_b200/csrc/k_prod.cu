// Matrix products on tcgen05, D[p][q] = sum_k A[p][k] B[q][k]: block-scaled FP8 or 16-bit operands,
// dense, with the rows of one side grouped by expert, or with the contraction grouped by expert.
//
// One persistent, warp-specialised kernel.  A CTA takes output tiles of 128 x BN; per step of 128
// bytes of the contraction, warp 0 copies the operands' tiles by TMA into a ring of 128-byte
// swizzled stages, warp 1 issues four MMAs into FP32 accumulators in TMEM, warps 4..7 write the
// finished tile out (TMEM lane = row of A).  Warp 2 serves the form of the product:
//   * FP8: kind::mxf8f6f4.block_scale applies a power-of-two scale per row and 32 values inside the
//     tensor core; a block of 128 is four such steps with the same scale.  The scales of 128 rows and
//     four blocks form the 512-byte atom that tcgen05.cp spreads over the TMEM lanes (row r, block j at
//     (r % 32) * 16 + (r / 32) * 4 + j); warp 2 gathers it from global memory once per four steps and
//     the MMA names the byte j.  The accumulator never leaves TMEM before the tile is done.
//   * contraction grouped by expert: a group's last step may reach into the next group's rows; warp 2
//     zeroes those rows of both operands in shared memory before the MMA sees the stage.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "blockscale_host.h"
#include "tc.cuh"

namespace aeisu {
namespace {

using namespace tc;

constexpr int kBM = 128;              // rows of A per tile: the TMEM lanes
constexpr int kStepBytes = 128;       // contraction bytes per step: one swizzle row
constexpr int kThreads = 256;
constexpr int kRing = 200 * 1024;     // shared memory of the operand ring
constexpr int kErrWait = 1;           // error code: a wait ran out
constexpr int kAtom = 512;            // scales of 128 rows and four block columns

// What is grouped by the offsets.
enum Grouping { kDense = 0, kRowsA = 1, kRowsB = 2, kContraction = 3 };

__device__ int g_product_error;

struct ProdJob {
    int P, Q, K;                 // rows of A, rows of B, contraction (whole sides; per batch entry)
    int grouping, groups;
    const int* off;
    int a_mn, b_mn;              // operand stored with its rows contiguous (contraction strided)
    uint32_t idesc;
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
    int zero_outside, zero_rows;
    int after_quantize;          // starts while the quantiser of its float operand still runs; the other
                                 // operand and the offsets are older
};

template <bool FP8, int BN>
struct Shape {
    static constexpr int kATile = kBM * kStepBytes, kBTile = BN * kStepBytes;
    static constexpr int kAtomsB = (BN + 127) / 128;
    static constexpr int kScaleBytes = FP8 ? kAtom * (1 + kAtomsB) : 0;
    static constexpr int kStage = kATile + kBTile;
    static constexpr int kStages = kRing / (kStage + kScaleBytes);
    // Accumulators of two tiles where TMEM's 512 columns hold them beside the scales.
    static constexpr int kAccs = 2 * BN + (FP8 ? 64 : 0) <= 512 ? 2 : 1;
    static constexpr int kScaleCol = kAccs * BN;
    // Each stage has its own scale columns: they are written again only after the MMAs that read them
    // have been committed with the stage.
    static constexpr int kScaleCols = FP8 ? 4 * (1 + kAtomsB) : 0;
    static constexpr int kColsUsed = kAccs * BN + kStages * kScaleCols;
    static constexpr int kCols = kColsUsed <= 32 ? 32 : kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128
                                 : kColsUsed <= 256 ? 256 : 512;
    static constexpr int kBars = 3 * kStages + 2 * kAccs + 1;
    static constexpr size_t kSmem = 1024 + size_t(kStages) * (kStage + kScaleBytes) + kBars * 8 + 16;
};

// ---- PTX ---------------------------------------------------------------------------------------

// K-major operand tile, rows of 128 swizzled bytes: eight rows per 1024-byte atom.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Row-contiguous operand tile: chunks of 64 rows of the operand (128 swizzled bytes) by 64
// contraction values, 8192 bytes from chunk to chunk, 1024 from eight contraction values to the next.
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(8192 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
           (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

__device__ __forceinline__ void mma_block_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                                 uint32_t sfb, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
        :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc) : "memory");
}
// A 512-byte scale atom to four TMEM columns, repeated in the lanes of all four warps.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t saddr) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(taddr), "l"(sdesc(saddr, 128, 128))
                 : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t smem, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(smem), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar)) : "memory");
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
__device__ __forceinline__ float peer_float(uint32_t saddr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}\n"
                 : "=f"(v) : "r"(saddr), "r"(rank) : "memory");
    return v;
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
    return mbar_wait_bounded(bar, parity, &g_product_error, kErrWait);
}

// ---- tiles -------------------------------------------------------------------------------------

struct Tile {
    int e;               // batch entry of the grouped operand or output
    int p0, q0;          // first rows of A and B (absolute)
    int p1, q1;          // ends of the rows that are stored
    int k0, k1;          // contraction range (absolute)
    int part;            // part of a split contraction
};

// Cumulative row tiles of the groups, in shared memory; offsets are clamped to [0, rows] and to be
// no smaller than the one before, so that no value of theirs leads out of the tensors.
struct Groups {
    const int* bound;    // [groups + 1]
    const int* cum;      // [groups + 1] row tiles before each group
};

template <int BN>
__device__ __forceinline__ int tile_count(const ProdJob& j, const Groups& g) {
    const int tp = (j.P + kBM - 1) / kBM, tq = (j.Q + BN - 1) / BN;
    if (j.grouping == kDense) return tp * tq * j.split;
    if (j.grouping == kContraction) return tp * tq * j.groups;
    return g.cum[j.groups] * (j.grouping == kRowsA ? tq : tp);
}

template <int BN>
__device__ __forceinline__ Tile tile_at(const ProdJob& j, const Groups& g, int t, int step) {
    const int tp = (j.P + kBM - 1) / kBM, tq = (j.Q + BN - 1) / BN;
    Tile x{0, 0, 0, j.P, j.Q, 0, j.K, 0};
    if (j.grouping == kDense) {
        // Bands of 16 row tiles, walked column by column: CTAs that run at the same time share both
        // operands' tiles in L2.
        x.part = t / (tp * tq);
        t -= x.part * tp * tq;
        const int band = t / (16 * tq), first = band * 16, high = min(16, tp - first), in = t - band * 16 * tq;
        x.p0 = (first + in % high) * kBM;
        x.q0 = (in / high) * BN;
        x.k0 = x.part * j.steps_per_split * step;
        x.k1 = min(j.K, x.k0 + j.steps_per_split * step);
    } else if (j.grouping == kContraction) {
        x.e = t / (tp * tq);
        t -= x.e * tp * tq;
        x.p0 = (t % tp) * kBM;
        x.q0 = (t / tp) * BN;
        x.k0 = g.bound[x.e];
        x.k1 = g.bound[x.e + 1];
    } else {
        const int other = j.grouping == kRowsA ? tq : tp;
        int lo = 0, hi = j.groups - 1;       // last group whose tiles start at or before t
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (g.cum[mid] * other <= t) lo = mid;
            else hi = mid - 1;
        }
        x.e = lo;
        const int own = g.cum[lo + 1] - g.cum[lo], in = t - g.cum[lo] * other;
        if (j.grouping == kRowsA) {
            x.p0 = g.bound[lo] + (in % own) * kBM;
            x.p1 = g.bound[lo + 1];
            x.q0 = (in / own) * BN;
        } else {
            x.q0 = g.bound[lo] + (in % own) * BN;
            x.q1 = g.bound[lo + 1];
            x.p0 = (in / own) * kBM;
        }
    }
    return x;
}

// ---- scales ------------------------------------------------------------------------------------

// This lane's 16 bytes of the atom of rows row0 .. row0 + 127 and block columns kb .. kb + 3: word w
// holds row 32 w + lane.  Rows past the end repeat the last one, block columns past the end are
// not used by any MMA.
__device__ __forceinline__ uint4 gather_scales(const ScaleRef& s, int e, int row0, int rows, int kb, int blocks) {
    const uint8_t* base = s.ptr + e * s.batch_stride;
    const int lane = threadIdx.x & 31;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = min(row0 + 32 * i + lane, rows - 1) >> s.shift;
        w[i] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
            w[i] |= uint32_t(__ldg(base + (long long)min(kb + b, blocks - 1) * s.ld + at)) << (8 * b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
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
__device__ __forceinline__ uint32_t pack2(int type, float a, float b) {
    if (type == kF16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// `n` of up to W consecutive values at element index i; whole 16-byte stores where they fit.
template <int W>
__device__ __forceinline__ void store_run(void* p, int type, long long i, const float* v, int n) {
    if (n >= W) {
        if (type == kF32) {
            float* q = static_cast<float*>(p) + i;
            if ((reinterpret_cast<uintptr_t>(q) & 15) == 0) {
#pragma unroll
                for (int c = 0; c < W; c += 4)
                    *reinterpret_cast<float4*>(q + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
                return;
            }
        } else {
            uint16_t* q = static_cast<uint16_t*>(p) + i;
            if ((reinterpret_cast<uintptr_t>(q) & 15) == 0) {
#pragma unroll
                for (int c = 0; c < W; c += 8)
                    *reinterpret_cast<uint4*>(q + c) =
                        make_uint4(pack2(type, v[c], v[c + 1]), pack2(type, v[c + 2], v[c + 3]),
                                   pack2(type, v[c + 4], v[c + 5]), pack2(type, v[c + 6], v[c + 7]));
                return;
            }
        }
    }
#pragma unroll
    for (int c = 0; c < W; ++c)
        if (c < n) store_elem(p, type, i + c, v[c]);
}

template <int W>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float (&v)[W]);
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t taddr, float (&v)[32]) { tmem_ld32(taddr, v); }
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ---- the kernel --------------------------------------------------------------------------------

template <bool FP8, int BN>
__global__ void __launch_bounds__(kThreads, 1)
k_product(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
          const __grid_constant__ ProdJob j) {
    using S = Shape<FP8, BN>;
    constexpr int kStep = FP8 ? kStepBytes : kStepBytes / 2;   // contraction values per step
    extern __shared__ uint8_t raw[];
    __shared__ uint32_t tmem_slot;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* scales = ring + S::kStages * S::kStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(scales + S::kStages * S::kScaleBytes);
    uint64_t* empty = full + S::kStages;
    uint64_t* fixed = empty + S::kStages;
    uint64_t* acc_full = fixed + S::kStages;
    uint64_t* acc_empty = acc_full + S::kAccs;
    uint64_t* drain = acc_empty + S::kAccs;
    int* bound = reinterpret_cast<int*>(drain + 1);
    int* cum = bound + j.groups + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (warp == 3) tmem_alloc(&tmem_slot, S::kCols);
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            mbar_init(full + i, FP8 ? 2 : 1);
            mbar_init(empty + i, 1);
            mbar_init(fixed + i, 1);
        }
        for (int i = 0; i < S::kAccs; ++i) {
            mbar_init(acc_full + i, 1);
            mbar_init(acc_empty + i, 128);
        }
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    const Groups g{bound, cum};
    if (j.grouping != kDense) {
        const int rows = j.grouping == kContraction ? j.K : j.grouping == kRowsA ? j.P : j.Q;
        const int high = j.grouping == kRowsB ? BN : kBM;
        for (int i = threadIdx.x; i <= j.groups; i += kThreads) bound[i] = min(max(j.off[i], 0), rows);
        __syncthreads();
        if (threadIdx.x == 0) {
            int tiles = 0;
            cum[0] = 0;
            for (int i = 0; i < j.groups; ++i) {
                bound[i + 1] = max(bound[i + 1], bound[i]);
                tiles += (bound[i + 1] - bound[i] + high - 1) / high;
                cum[i + 1] = tiles;
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_slot;
    const int tiles = tile_count<BN>(j, g);
    // A cluster takes one tile, each of its CTAs a part of the contraction.
    const int rank = j.cluster > 1 ? int(cluster_rank()) : 0;
    const int first_tile = j.cluster > 1 ? rank * (tiles / j.split) + int(blockIdx.x) / j.cluster : int(blockIdx.x);
    const int stride = j.cluster > 1 ? tiles : int(gridDim.x);

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            long long issued = 0;
            if (j.after_quantize) grid_dep_wait();
            for (int t = first_tile; ok && t < tiles; t += stride) {
                const Tile x = tile_at<BN>(j, g, t, kStep);
                const int ea = j.grouping == kRowsB ? x.e : 0, eb = j.grouping == kRowsA ? x.e : 0;
                for (int k = x.k0; k < x.k1; k += kStep) {
                    if (!(ok = wait(empty + stage, phase ^ 1))) break;
                    const uint32_t a = smem_addr(ring + stage * S::kStage), b = a + S::kATile;
                    mbar_arrive_expect_tx(full + stage, S::kStage);
                    if (j.a_mn) {
                        for (int c = 0; c < kBM / 64; ++c) tma_3d(a + c * 8192, &ma, x.p0 + c * 64, k, ea, full + stage);
                    } else {
                        tma_3d(a, &ma, k, x.p0, ea, full + stage);
                    }
                    if (j.b_mn) {
                        for (int c = 0; c < BN / 64; ++c) tma_3d(b + c * 8192, &mb, x.q0 + c * 64, k, eb, full + stage);
                    } else {
                        tma_3d(b, &mb, k, x.q0, eb, full + stage);
                    }
                    ++issued;
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
            }
            // Every copy has landed before the CTA may end: those that no MMA waited for are waited for here.
            for (int i = 0; !ok && i < S::kStages && issued - i > 0; ++i) {
                const long long n = issued - 1 - i;
                wait(full + n % S::kStages, uint32_t(n / S::kStages) & 1);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            uint64_t* ready = j.grouping == kContraction ? fixed : full;
            const uint32_t a_k = (j.a_mn ? 2048 : 32) >> 4, b_k = (j.b_mn ? 2048 : 32) >> 4;
            for (int t = first_tile; ok && t < tiles; t += stride) {
                const Tile x = tile_at<BN>(j, g, t, kStep);
                if (!(ok = wait(acc_empty + acc, acc_phase ^ 1))) break;
                fence_after_sync();
                const uint32_t d = tmem + acc * BN;
                uint32_t first = 0;
                int step = 0;
                for (int k = x.k0; k < x.k1; k += kStep, ++step) {
                    if (!(ok = wait(ready + stage, phase))) break;
                    fence_after_sync();
                    const uint32_t sa = smem_addr(ring + stage * S::kStage), sb = sa + S::kATile;
                    const uint64_t da = j.a_mn ? desc_mnmajor(sa) : desc_kmajor(sa);
                    const uint64_t db = j.b_mn ? desc_mnmajor(sb) : desc_kmajor(sb);
                    if constexpr (FP8) {
                        const uint32_t sf = tmem + S::kScaleCol + stage * S::kScaleCols;
                        const uint32_t src = smem_addr(scales + stage * S::kScaleBytes);
#pragma unroll
                        for (int i = 0; i <= S::kAtomsB; ++i) scales_to_tmem(sf + 4 * i, src + i * kAtom);
                        const uint32_t id = j.idesc | (uint32_t(step & 3) << 4) | (uint32_t(step & 3) << 29);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_block_scaled(d, da + i * 2, db + i * 2, id, sf, sf + 4, first);
                            first = 1;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_f16(d, da + i * a_k, db + i * b_k, j.idesc, first);
                            first = 1;
                        }
                    }
                    commit(empty + stage);
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
                commit(acc_full + acc);
                if (++acc == S::kAccs) acc = 0, acc_phase ^= 1;
            }
            if (!ok) {   // let the MMAs in flight land before TMEM goes
                commit(drain);
                wait(drain, 0);
            }
        }
    } else if (warp == 2) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        if constexpr (FP8) {
            if (j.after_quantize) grid_dep_wait();
            const int blocks = (j.K + kBlock - 1) / kBlock;
            for (int t = first_tile; ok && t < tiles; t += stride) {
                const Tile x = tile_at<BN>(j, g, t, kStep);
                const int ea = j.grouping == kRowsB ? x.e : 0, eb = j.grouping == kRowsA ? x.e : 0;
                int step = 0;
                uint4 s[1 + S::kAtomsB];
                for (int k = x.k0; ok && k < x.k1; k += kStep, ++step) {
                    if ((step & 3) == 0) {
                        const int kb = k / kBlock;
                        s[0] = gather_scales(j.sa, ea, x.p0, j.a_rows, kb, blocks);
#pragma unroll
                        for (int i = 0; i < S::kAtomsB; ++i)
                            s[1 + i] = gather_scales(j.sb, eb, x.q0 + 128 * i, j.b_rows, kb, blocks);
                    }
                    ok = wait(empty + stage, phase ^ 1);
                    if (!ok) break;
                    uint4* dst = reinterpret_cast<uint4*>(scales + stage * S::kScaleBytes);
#pragma unroll
                    for (int i = 0; i <= S::kAtomsB; ++i) dst[i * 32 + lane] = s[i];
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + stage);
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
            }
        } else if (j.grouping == kContraction) {
            for (int t = first_tile; ok && t < tiles; t += stride) {
                const Tile x = tile_at<BN>(j, g, t, kStep);
                for (int k = x.k0; k < x.k1; k += kStep) {
                    if (!(ok = wait(full + stage, phase))) break;
                    const int rows = x.k1 - k;
                    if (rows < kStep) {
                        uint8_t* base = ring + stage * S::kStage;
                        const int tail = (kStep - rows) * 8;   // 16-byte pieces per chunk
                        for (int i = lane; i < tail * (S::kStage / 8192); i += 32)
                            *reinterpret_cast<uint4*>(base + (i / tail) * 8192 + rows * 128 + (i % tail) * 16) =
                                make_uint4(0, 0, 0, 0);
                        fence_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(fixed + stage);
                    if (++stage == S::kStages) stage = 0, phase ^= 1;
                }
            }
        }
    } else if (warp >= 4) {
        constexpr int W = BN < 32 ? BN : 32;
        const int quad = warp & 3, row = quad * 32 + lane;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = first_tile; t < tiles; t += stride) {
            const Tile x = tile_at<BN>(j, g, t, kStep);
            if (!wait(acc_full + acc, acc_phase)) break;
            fence_after_sync();
            const bool any = x.k0 < x.k1;
            const int p = x.p0 + row;
            const long long base = x.part * j.split_stride + (j.grouping == kContraction ? x.e * j.out_batch : 0);
#pragma unroll
            for (int c = 0; c < BN; c += W) {
                float v[W];
                if (any) {
                    tmem_load<W>(tmem + (uint32_t(quad * 32) << 16) + acc * BN + c, v);
                } else {
#pragma unroll
                    for (int i = 0; i < W; ++i) v[i] = 0.f;
                }
                const int q = x.q0 + c, n = x.q1 - q;
                if (j.cluster > 1) {
                    // every MMA of this CTA is done with the ring: it takes the tile, column by column
#pragma unroll
                    for (int i = 0; i < W; ++i) reinterpret_cast<float*>(ring)[(c + i) * kBM + row] = v[i];
                } else if (p < x.p1 && n > 0) {
                    if (!j.swapped) {
                        if (j.bias)
#pragma unroll
                            for (int i = 0; i < W; ++i)
                                if (i < n) v[i] += load_elem(j.bias, j.bias_type, q + i);
                        store_run<W>(j.out, j.out_type, base + p * j.out_ld + q, v, n);
                    } else {
                        const float b = j.bias ? load_elem(j.bias, j.bias_type, p) : 0.f;
#pragma unroll
                        for (int i = 0; i < W; ++i)
                            if (i < n) store_elem(j.out, j.out_type, base + (q + i) * j.out_ld + p, v[i] + b);
                    }
                }
                __syncwarp();
            }
            fence_before_sync();
            mbar_arrive(acc_empty + acc);
            if (++acc == S::kAccs) acc = 0, acc_phase ^= 1;
        }
        if (j.zero_outside) {
            const int before = bound[0], after = bound[j.groups], skip = after - before;
            const long long todo = (long long)(j.zero_rows - skip) * j.cols;
            for (long long i = (long long)blockIdx.x * 128 + (threadIdx.x - 128); i < todo; i += (long long)gridDim.x * 128) {
                const int r = int(i / j.cols), at = r < before ? r : r + skip;
                store_elem(j.out, j.out_type, at * j.out_ld + i % j.cols, 0.f);
            }
        }
    }
    if (j.cluster > 1) {
        // The parts are added in their order, each CTA taking its share of the columns.
        cluster_sync();
        if (warp >= 4 && first_tile < tiles) {
            const Tile x = tile_at<BN>(j, g, first_tile, kStep);
            const int row = threadIdx.x - 128, p = x.p0 + row, share = BN / j.cluster;
            const float pb = j.bias && j.swapped && p < x.p1 ? load_elem(j.bias, j.bias_type, p) : 0.f;
            for (int c = rank * share; c < (rank + 1) * share; ++c) {
                const int q = x.q0 + c;
                if (p >= x.p1 || q >= x.q1) continue;
                float v = 0.f;
                for (int r = 0; r < j.cluster; ++r) v += peer_float(smem_addr(ring) + (c * kBM + row) * 4, r);
                if (j.swapped) store_elem(j.out, j.out_type, q * j.out_ld + p, v + pb);
                else store_elem(j.out, j.out_type, p * j.out_ld + q, v + (j.bias ? load_elem(j.bias, j.bias_type, q) : 0.f));
            }
        }
        cluster_sync();
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 3) tmem_free(tmem, S::kCols);
}

// out = sum of the parts in order, plus the bias of the column.
__global__ void __launch_bounds__(256) k_join_parts(const float* part, int parts, long long stride, int rows, int cols,
                                                    void* out, int out_type, long long out_ld, const void* bias,
                                                    int bias_type) {
    const long long n = (long long)rows * cols;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = 0.f;
        for (int k = 0; k < parts; ++k) s += part[k * stride + i];
        const int r = int(i / cols), c = int(i % cols);
        if (bias) s += load_elem(bias, bias_type, c);
        store_elem(out, out_type, r * out_ld + c, s);
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

// Operand map: innermost the contiguous direction in boxes of 128 bytes, `high` of the other.
CUtensorMap operand_map(const MatrixRef& m, int high) {
    const int eb = elem_bytes(m.type);
    const int inner = m.trans ? m.rows : m.cols, outer = m.trans ? m.cols : m.rows;
    CUtensorMap map{};
    const cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(outer), cuuint64_t(m.batch)};
    const long long batch = m.batch > 1 ? m.batch_stride : ((m.ld * outer * eb + 15) / 16 * 16) / eb;
    const cuuint64_t strides[2] = {cuuint64_t(m.ld) * eb, cuuint64_t(batch) * eb};
    const cuuint32_t box[3] = {cuuint32_t(kStepBytes / eb), cuuint32_t(high), 1};
    const cuuint32_t one[3] = {1, 1, 1};
    const CUtensorMapDataType type = m.type == kF16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : m.type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const CUresult r = encoder()(&map, type, 3, const_cast<void*>(m.ptr), dims, strides, box, one,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
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

template <bool FP8, int BN>
void launch(const CUtensorMap& a, const CUtensorMap& b, const ProdJob& j, long long tiles, int device,
            cudaStream_t stream) {
    using S = Shape<FP8, BN>;
    const size_t smem = S::kSmem + (j.grouping == kDense ? 0 : 2 * size_t(j.groups + 1) * sizeof(int));
    static std::mutex mu;
    static bool ready[64] = {};
    const int sms = sm_count(device);
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[device]) {
            AEISU_CUDA(cudaFuncSetAttribute(k_product<FP8, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            int(S::kSmem + 2 * (kMaxGroups + 1) * sizeof(int))));
            ready[device] = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(j.cluster > 1 ? tiles : std::min<long long>(tiles, sms)), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = j.after_quantize;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(j.cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = j.cluster > 1 ? 2 : 1;
    AEISU_CUDA(cudaLaunchKernelEx(&cfg, k_product<FP8, BN>, a, b, j));
}

template <bool FP8>
void launch_width(int bn, const CUtensorMap& a, const CUtensorMap& b, const ProdJob& j, long long tiles, int device,
                  cudaStream_t stream) {
    switch (bn) {
        case 16: return launch<FP8, 16>(a, b, j, tiles, device, stream);
        case 32: return launch<FP8, 32>(a, b, j, tiles, device, stream);
        case 64: return launch<FP8, 64>(a, b, j, tiles, device, stream);
        case 128: return launch<FP8, 128>(a, b, j, tiles, device, stream);
        default: return launch<FP8, 256>(a, b, j, tiles, device, stream);
    }
}

uint32_t instruction(const MatrixRef& a, const MatrixRef& b, int bn) {
    const uint32_t size = (uint32_t(bn >> 3) << 17) | (uint32_t(kBM >> 4) << 24);
    if (is_code(a.type))
        return size | (uint32_t(a.type == kE5M2) << 7) | (uint32_t(b.type == kE5M2) << 10) | (1u << 23);
    const uint32_t f = a.type == kBF16 ? 1 : 0;
    return size | (1u << 4) | (f << 7) | (f << 10) | (uint32_t(a.trans) << 15) | (uint32_t(b.trans) << 16);
}

int width_for(int rows, bool trans) {
    const int least = trans ? 64 : 16;
    for (int w = least; w < 256; w *= 2)
        if (rows <= w) return w;
    return 256;
}

// How a dense product is cut: which side lies along the TMEM lanes, the tile width and the parts of
// the contraction.
struct Plan {
    bool swap;
    int bn, split, steps;   // steps of the contraction per part
    int cluster;
};

Plan plan_dense(int m, int n, int k, bool fp8, int sms) {
    Plan p{};
    const int step = fp8 ? kStepBytes : kStepBytes / 2, steps = (k + step - 1) / step;
    // Few rows: the weights take the 128 lanes, so that no lane idles, and the rows the columns.
    p.swap = m <= 64 && n > m;
    const int P = p.swap ? n : m, Q = p.swap ? m : n;
    p.bn = width_for(Q, false);
    auto tiles = [&](int bn) { return (long long)((P + kBM - 1) / kBM) * ((Q + bn - 1) / bn); };
    while (p.bn > 64 && tiles(p.bn) < sms) p.bn /= 2;
    // While SMs are left over, the contraction is cut: into 2, 4 or 8 parts of at least two steps, the CTAs
    // of a cluster, which need no second kernel; where that fills less than half of the SMs and the
    // contraction is long, into as many parts as fill them, of at least eight steps, joined by a kernel.
    const long long t = tiles(p.bn);
    p.cluster = p.split = 1;
    p.steps = steps;
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
    return p;
}

}  // namespace

size_t product_workspace(int m, int n, int k, bool fp8, int device) {
    const Plan p = plan_dense(m, n, k, fp8, sm_count(device));
    return p.split > p.cluster ? size_t(p.split) * m * n * sizeof(float) : 0;
}

void product(const MatrixRef& a, const ScaleRef* sa, const MatrixRef& b, const ScaleRef* sb, const ProductOut& out,
             void* workspace, size_t workspace_bytes, bool after_quantize, int device, cudaStream_t stream) {
    check_operand(a, sa);
    check_operand(b, sb);
    require(a.batch == 1 && b.batch == 1 && !a.trans && !b.trans && a.cols == b.cols, "contraction sizes differ");
    require((sa != nullptr) == (sb != nullptr) && (sa || a.type == b.type), "operand types do not go together");
    require(out.ptr && out.type >= kF32 && out.type <= kBF16 && out.ld >= b.rows, "output is out of range");
    OnDevice on(device);
    const bool fp8 = sa != nullptr;
    const Plan pl = plan_dense(a.rows, b.rows, a.cols, fp8, sm_count(device));
    const size_t need = pl.split > pl.cluster ? size_t(pl.split) * a.rows * b.rows * sizeof(float) : 0;
    require(need == 0 || (workspace && workspace_bytes >= need), "workspace is too small");
    const MatrixRef& A = pl.swap ? b : a;
    const MatrixRef& B = pl.swap ? a : b;
    ProdJob j{};
    j.P = A.rows;
    j.Q = B.rows;
    j.K = A.cols;
    j.a_mn = A.trans;
    j.b_mn = B.trans;
    j.idesc = instruction(A, B, pl.bn);
    if (fp8) {
        j.sa = pl.swap ? *sb : *sa;
        j.sb = pl.swap ? *sa : *sb;
    }
    j.a_rows = A.rows;
    j.b_rows = B.rows;
    j.swapped = pl.swap;
    j.cols = b.rows;
    j.split = pl.split;
    j.steps_per_split = pl.steps;
    j.cluster = pl.cluster;
    j.after_quantize = after_quantize;
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
    const long long tiles = (long long)((j.P + kBM - 1) / kBM) * ((j.Q + pl.bn - 1) / pl.bn) * pl.split;
    require(tiles < (1LL << 30), "matrix is too large");
    const CUtensorMap ma = operand_map(A, A.trans ? 64 : kBM), mb = operand_map(B, B.trans ? 64 : pl.bn);
    if (fp8) launch_width<true>(pl.bn, ma, mb, j, tiles, device, stream);
    else launch_width<false>(pl.bn, ma, mb, j, tiles, device, stream);
    if (pl.split > pl.cluster) {
        const long long n = (long long)a.rows * b.rows;
        k_join_parts<<<unsigned(std::min<long long>((n + 255) / 256, 148 * 8)), 256, 0, stream>>>(
            static_cast<const float*>(workspace), pl.split, j.split_stride, a.rows, b.rows, out.ptr, out.type, out.ld,
            out.bias, out.bias_type);
        AEISU_CUDA(cudaGetLastError());
    }
}

void grouped_product(const MatrixRef& x, const ScaleRef* sx, const MatrixRef& b, const ScaleRef* sb, const int* off,
                     const ProductOut& out, bool zero_outside, bool after_quantize, int device, cudaStream_t stream) {
    check_operand(x, sx);
    check_operand(b, sb);
    require(x.batch == 1 && !x.trans && x.cols == b.cols, "contraction sizes differ");
    require((sx != nullptr) == (sb != nullptr) && (sx || x.type == b.type), "operand types do not go together");
    require(off && b.batch <= kMaxGroups, "a grouped product has offsets and at most 1024 groups");
    require(out.ptr && out.type >= kF32 && out.type <= kBF16 && out.ld >= b.rows && !out.bias, "output is out of range");
    OnDevice on(device);
    const bool fp8 = sx != nullptr;
    // Few rows per group on average: as for a dense product, the weights take the lanes.
    const int mean = (x.rows + b.batch - 1) / b.batch;
    const bool swap = mean <= 64 && b.rows >= kBM;
    ProdJob j{};
    const MatrixRef& A = swap ? b : x;
    const MatrixRef& B = swap ? x : b;
    int bn = swap ? width_for(mean, false) : width_for(b.rows, b.trans);
    if (!swap) {
        const long long rows = (x.rows + kBM - 1) / kBM;
        while (bn > 64 && rows * ((b.rows + bn - 1) / bn) < sm_count(device)) bn /= 2;
    }
    j.P = A.rows;
    j.Q = B.rows;
    j.K = A.cols;
    j.grouping = swap ? kRowsB : kRowsA;
    j.groups = b.batch;
    j.off = off;
    j.a_mn = A.trans;
    j.b_mn = B.trans;
    j.idesc = instruction(A, B, bn);
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
    j.split = j.cluster = 1;
    j.after_quantize = after_quantize;
    j.zero_outside = zero_outside;
    j.zero_rows = x.rows;
    const int high = swap ? bn : kBM, wide = swap ? kBM : bn;
    // Each group has at most one partly filled row tile.
    const long long tiles = ((long long)(x.rows + high - 1) / high + std::min(b.batch, x.rows)) *
                            ((b.rows + wide - 1) / wide);
    require(tiles < (1LL << 30), "matrix is too large");
    const CUtensorMap ma = operand_map(A, A.trans ? 64 : kBM), mb = operand_map(B, B.trans ? 64 : bn);
    if (fp8) launch_width<true>(bn, ma, mb, j, tiles, device, stream);
    else launch_width<false>(bn, ma, mb, j, tiles, device, stream);
}

void grouped_weight_gradient(const MatrixRef& g, const MatrixRef& x, const int* off, int groups, void* out,
                             int out_type, int device, cudaStream_t stream) {
    check_operand(g, nullptr);
    check_operand(x, nullptr);
    require(g.batch == 1 && x.batch == 1 && g.trans && x.trans && g.cols == x.cols && g.type == x.type,
            "contraction sizes differ");
    require(off && groups >= 1 && groups <= kMaxGroups, "a grouped product has offsets and at most 1024 groups");
    require(out && out_type >= kF32 && out_type <= kBF16, "output is out of range");
    OnDevice on(device);
    ProdJob j{};
    int bn = width_for(x.rows, true);
    auto count = [&](int w) { return (long long)((g.rows + kBM - 1) / kBM) * ((x.rows + w - 1) / w) * groups; };
    while (bn > 64 && count(bn) < sm_count(device)) bn /= 2;
    j.P = g.rows;
    j.Q = x.rows;
    j.K = g.cols;
    j.grouping = kContraction;
    j.groups = groups;
    j.off = off;
    j.a_mn = j.b_mn = 1;
    j.idesc = instruction(g, x, bn);
    j.out = out;
    j.out_type = out_type;
    j.out_ld = x.rows;
    j.out_batch = (long long)g.rows * x.rows;
    j.cols = x.rows;
    j.split = j.cluster = 1;
    require(count(bn) < (1LL << 30), "matrix is too large");
    launch_width<false>(bn, operand_map(g, 64), operand_map(x, 64), j, count(bn), device, stream);
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
