// Block-scaled FP8 quantisation: codes E4M3 or E5M2, one power-of-two scale (E8M0) for each block
// of 128 values of a row (block_rows 1) or of 128 x 128 values (block_rows 128).
//
// With amax the largest finite magnitude of a block and top the largest finite code (448 or
// 57344), the scale is the smallest power of two s with amax / s <= top (1 for a block of zeros),
// and a code is x / s rounded to nearest even.  Division by a power of two is exact, so the one
// rounding of a code is the rounding to 8 bits, and the result is defined bit for bit.  Infinities
// and NaN become NaN codes and take no part in amax: they spoil what they would spoil in the
// product, and nothing else.
#include <algorithm>

#include "blockscale_dev.cuh"
#include "blockscale_host.h"

namespace aeisu {
namespace {

using namespace blockq;

constexpr int kThreads = 256;

template <typename T>
struct QuantJob {
    const T* x;
    int rows, cols;
    long long ld, batch_stride;
    uint8_t* codes;
    long long codes_ld, codes_batch;
    uint8_t* scales;           // [batch][col blocks][row blocks]
    uint8_t* t_codes;          // codes of the transpose [batch][cols][rows], or null
    long long t_ld, t_batch;
    uint8_t* t_scales;         // [batch][row blocks of 128][col blocks or cols]
    float* sums;               // column sums of each 128 rows [row blocks][cols], or null
};

// The product that reads the codes may start its set-up now; it waits for this kernel's end.
__device__ __forceinline__ void let_dependents_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// One scale per row and block column, no transpose.  Eight lanes share a block (two loads of eight
// values each), a warp takes CB neighbouring blocks of 4 / CB rows at a time, four times, a CTA 128 of these
// blocks; the scales leave through shared memory as contiguous bytes of a block column.  CB is 4 where
// rows are long, so that a warp reads whole runs of them; fewer leave no lane idle on short rows (165,888 x 128
// bfloat16: 29 us with 4).
template <typename T, bool E5M2, bool VEC, int CB>
__global__ void __launch_bounds__(kThreads) k_quant_rows(QuantJob<T> j) {
    constexpr int kRows = kBlock / CB;
    __shared__ uint8_t sh[CB][kRows];
    let_dependents_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col_groups = (j.cols + CB * kBlock - 1) / (CB * kBlock);
    const int r0 = int(blockIdx.x / col_groups) * kRows, c0 = int(blockIdx.x % col_groups) * CB * kBlock;
    const T* x = j.x + blockIdx.y * j.batch_stride;
    uint8_t* codes = j.codes + blockIdx.y * j.codes_batch;
    const int b = (lane >> 3) % CB, c = c0 + b * kBlock + (lane & 7) * 16;
    const int first = warp * (kRows / 8) + (lane >> 3) / CB;   // rows first + i * 4 / CB
    Vals<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + first + i * (4 / CB);
        v[i] = {};
        if (r < j.rows) {
            load8<T, VEC>(v[i], 0, x + r * j.ld, c, j.cols);
            load8<T, VEC>(v[i], 1, x + r * j.ld, c + 8, j.cols);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + first + i * (4 / CB);
        float amax = finite_max(v[i]);
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, d));
        const uint32_t s = scale_of<E5M2>(amax);
        const float inv = inverse_scale(s);
        if ((lane & 7) == 0) sh[b][first + i * (4 / CB)] = uint8_t(s);
        if (r < j.rows && c < j.cols) {
            uint4 q;
            uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = codes4<E5M2>(v[i].get(4 * k) * inv, v[i].get(4 * k + 1) * inv, v[i].get(4 * k + 2) * inv,
                                    v[i].get(4 * k + 3) * inv);
            *reinterpret_cast<uint4*>(codes + r * j.codes_ld + c) = q;
        }
    }
    __syncthreads();
    if (threadIdx.x < kBlock) {
        const int block = threadIdx.x / kRows, r = threadIdx.x % kRows, col_blocks = (j.cols + kBlock - 1) / kBlock;
        if (r0 + r < j.rows && c0 / kBlock + block < col_blocks)
            j.scales[(size_t(blockIdx.y) * col_blocks + c0 / kBlock + block) * j.rows + r0 + r] = sh[block][r];
    }
}

// A 128 x 128 tile per CTA: codes with one scale per row or per tile and, with BOTH, the codes of the
// transpose too, from one read of x.  A lane holds four consecutive rows of two runs of eight
// columns: row maxima over eight lanes, column maxima over a lane's rows, four lanes and eight warps,
// pairs of 16-bit values at a time.  The transposed codes (four rows to a word) turn in shared memory; the
// 16-byte chunk of a column is exclusive-or'ed with the column's octet, so that a warp's 32 words
// fall in 32 banks.
// NARROW (at most 64 columns, one scale per row, both ways): the second run of eight columns is instead the same
// columns 128 rows on, so that no lane idles: a CTA takes 256 rows, two blocks of the transpose.
template <typename T, bool E5M2, bool VEC, bool TILE_SCALE, bool BOTH, bool NARROW = false>
__global__ void __launch_bounds__(kThreads, !BOTH ? (sizeof(T) == 2 ? 4 : 3) : sizeof(T) == 4 && !TILE_SCALE ? 2 : 3)
k_quant_tile(QuantJob<T> j) {
    static_assert(!NARROW || (BOTH && !TILE_SCALE), "narrow matrices have a form of their own one way and by tiles");
    using P = typename Pair<T>::type;
    constexpr int kPairs = sizeof(Vals<T>) / 4, kPer = 16 / kPairs;   // pairs of a lane's row, values in one
    __shared__ P col_max[8][kBlock / kPer];
    __shared__ __align__(16) float col_inv[kBlock];
    __shared__ uint8_t row_s[NARROW ? 2 * kBlock : kBlock];
    __shared__ float col_sum[TILE_SCALE || !BOTH ? 1 : 8][kBlock];
    __shared__ float tile_max[8];
    __shared__ __align__(16) uint32_t turn[BOTH ? kBlock * 32 : 4];
    let_dependents_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, oct = lane & 7, sub = lane >> 3;
    const int col_blocks = (j.cols + kBlock - 1) / kBlock, row_blocks = (j.rows + kBlock - 1) / kBlock;
    const int rb = int(blockIdx.x / col_blocks), cb = int(blockIdx.x % col_blocks);
    const int r0 = rb * (NARROW ? 2 * kBlock : kBlock), c0 = cb * kBlock, rw = warp * 16 + sub * 4;
    constexpr int kDown = NARROW ? kBlock : 0, kAside = NARROW ? 0 : 64;   // from a lane's first run to its second
    const T* x = j.x + blockIdx.y * j.batch_stride;
    Vals<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + rw + i;
        v[i] = {};
        if (r < j.rows) load8<T, VEC>(v[i], 0, x + r * j.ld, c0 + oct * 8, j.cols);
        if (r + kDown < j.rows) load8<T, VEC>(v[i], 1, x + (r + kDown) * j.ld, c0 + kAside + oct * 8, j.cols);
    }
    if constexpr (!TILE_SCALE && BOTH) {
        if (j.sums) {   // of the values as they are, infinities too
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                float s = (v[0].get(k) + v[1].get(k)) + (v[2].get(k) + v[3].get(k));
                s += __shfl_xor_sync(~0u, s, 8);
                s += __shfl_xor_sync(~0u, s, 16);
                if (sub == 0) col_sum[warp][(k >> 3) * 64 + oct * 8 + (k & 7)] = s;
            }
        }
    }
    float amax[4];
    [[maybe_unused]] float amax2[4];   // NARROW: of the second run
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (NARROW) finite_max2(v[i], amax[i], amax2[i]);
        else amax[i] = finite_max(v[i]);
    }
    if constexpr (TILE_SCALE) {
        float m = fmaxf(fmaxf(amax[0], amax[1]), fmaxf(amax[2], amax[3]));
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
        if (lane == 0) tile_max[warp] = m;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) amax[i] = fmaxf(amax[i], __shfl_xor_sync(~0u, amax[i], d));
            if (oct == 0) row_s[rw + i] = uint8_t(scale_of<E5M2>(amax[i]));
            if constexpr (NARROW) {
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) amax2[i] = fmaxf(amax2[i], __shfl_xor_sync(~0u, amax2[i], d));
                if (oct == 0) row_s[kBlock + rw + i] = uint8_t(scale_of<E5M2>(amax2[i]));
            }
        }
        if constexpr (BOTH) {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                P m = larger<T>(larger<T>(v[0].w[k], v[1].w[k]), larger<T>(v[2].w[k], v[3].w[k]));
                m = larger<T>(m, __shfl_xor_sync(~0u, m, 8));
                m = larger<T>(m, __shfl_xor_sync(~0u, m, 16));
                if (sub == 0) col_max[warp][(k / (kPairs / 2)) * (64 / kPer) + oct * (8 / kPer) + k % (kPairs / 2)] = m;
            }
        }
    }
    __syncthreads();
    uint32_t tile_s = 0;
    if constexpr (TILE_SCALE) {
        float m = tile_max[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = fmaxf(m, tile_max[w]);
        tile_s = scale_of<E5M2>(m);
        if (threadIdx.x == 0) {
            j.scales[(size_t(blockIdx.y) * col_blocks + cb) * row_blocks + rb] = uint8_t(tile_s);
            if (BOTH) j.t_scales[(size_t(blockIdx.y) * row_blocks + rb) * col_blocks + cb] = uint8_t(tile_s);
        }
    } else {
        if (threadIdx.x < kBlock) {
            if (r0 + int(threadIdx.x) < j.rows)
                j.scales[(size_t(blockIdx.y) * col_blocks + cb) * j.rows + r0 + threadIdx.x] = row_s[threadIdx.x];
            if (NARROW && r0 + kBlock + int(threadIdx.x) < j.rows)
                j.scales[size_t(blockIdx.y) * j.rows + r0 + kBlock + threadIdx.x] = row_s[kBlock + threadIdx.x];
        } else if constexpr (BOTH) {
            const int c = threadIdx.x - kBlock;
            P m = col_max[0][c / kPer];
#pragma unroll
            for (int w = 1; w < 8; ++w) m = larger<T>(m, col_max[w][c / kPer]);
            const uint32_t s = scale_of<E5M2>(kPer == 2 && (c & 1) ? second_of<T>(m) : first_of<T>(larger<T>(m, m)));
            col_inv[c] = inverse_scale(s);
            const int block = NARROW ? 2 * rb + c / 64 : rb, column = NARROW ? c % 64 : c0 + c;
            if (column < j.cols && block < row_blocks) {
                j.t_scales[(size_t(blockIdx.y) * row_blocks + block) * j.cols + column] = uint8_t(s);
                if (j.sums) {
                    float t = 0.f;
#pragma unroll
                    for (int w = 0; w < 8; ++w) t += col_sum[w][c];
                    j.sums[size_t(block) * j.cols + column] = t;
                }
            }
        }
    }
    uint8_t* codes = j.codes + blockIdx.y * j.codes_batch;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = r0 + rw + i + h * kDown, c = c0 + h * kAside + oct * 8;
            const float inv = inverse_scale(TILE_SCALE ? tile_s : scale_of<E5M2>(NARROW && h ? amax2[i] : amax[i]));
            auto at = [&](int k) { return v[i].get(8 * h + k) * inv; };
            const uint2 q = make_uint2(codes4<E5M2>(at(0), at(1), at(2), at(3)), codes4<E5M2>(at(4), at(5), at(6), at(7)));
            if (r < j.rows && c < j.cols) *reinterpret_cast<uint2*>(codes + r * j.codes_ld + c) = q;
        }
    }
    if constexpr (BOTH) {
        if constexpr (!TILE_SCALE) __syncthreads();   // col_inv
        const float tile_inv = inverse_scale(tile_s);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float inv[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) inv[k] = TILE_SCALE ? tile_inv : col_inv[h * 64 + oct * 8 + k];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                turn[(h * 64 + oct * 8 + k) * 32 + ((rw >> 2) ^ (oct << 2))] =
                    codes4<E5M2>(v[0].get(8 * h + k) * inv[k], v[1].get(8 * h + k) * inv[k], v[2].get(8 * h + k) * inv[k],
                                 v[3].get(8 * h + k) * inv[k]);
        }
        __syncthreads();
        uint8_t* t_codes = j.t_codes + blockIdx.y * j.t_batch;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = i * kThreads + threadIdx.x, c = at >> 3, chunk = at & 7;
            const uint4 q = *reinterpret_cast<const uint4*>(turn + c * 32 + ((chunk ^ ((c >> 3) & 7)) << 2));
            const int column = NARROW ? c % 64 : c0 + c, row = r0 + (NARROW ? c / 64 * kBlock : 0) + chunk * 16;
            if (column < j.cols && row < j.rows)
                *reinterpret_cast<uint4*>(t_codes + column * j.t_ld + row) = q;
        }
    }
}

// Column sums: each CTA adds a run of rows of 64 columns (lanes: eight columns of every fourth row of a
// warp's), then the runs are added in order.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) k_column_runs(const T* x, int rows, int cols, long long ld, int run,
                                                          float* partial) {
    __shared__ float sh[32][65];
    const int part = threadIdx.x >> 3, oct = threadIdx.x & 7, c = int(blockIdx.x) * 64 + oct * 8;
    const int r1 = min(rows, int(blockIdx.y + 1) * run);
    float a[8] = {};
#pragma unroll 4
    for (int r = int(blockIdx.y) * run + part; r < r1; r += 32) {
        Vals<T> v;
        load8<T, VEC>(v, 0, x + r * ld, c, cols);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] += v.get(i);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sh[part][oct * 8 + i] = a[i];
    __syncthreads();
    if (threadIdx.x < 64 && int(blockIdx.x) * 64 + int(threadIdx.x) < cols) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 32; ++w) s += sh[w][threadIdx.x];
        partial[size_t(blockIdx.y) * cols + blockIdx.x * 64 + threadIdx.x] = s;
    }
}

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A CTA takes eight columns; a thread adds every 128th run of one, then the threads' sums are added in order
// (1,296 runs of 64 columns: 3.1 us; with a warp for 32 columns and eight loads at a time 4.4).
template <typename T>
__global__ void __launch_bounds__(1024) k_column_join(const float* partial, int runs, int cols, T* out) {
    __shared__ float sh[128][9];
    const int col = threadIdx.x & 7, part = threadIdx.x >> 3, c = int(blockIdx.x) * 8 + col;
    float a = 0.f;
    for (int r0 = part; c < cols && r0 < runs; r0 += 128 * 12) {   // twelve loads at a time, of the last ones too
        float v[12];
#pragma unroll
        for (int i = 0; i < 12; ++i) v[i] = r0 + i * 128 < runs ? partial[size_t(r0 + i * 128) * cols + c] : 0.f;
#pragma unroll
        for (int i = 0; i < 12; ++i) a += v[i];
    }
    sh[part][col] = a;
    __syncthreads();
    if (threadIdx.x < 256) {   // a warp per column
        const int column = threadIdx.x >> 5, lane = threadIdx.x & 31;
        float s = (sh[lane][column] + sh[lane + 32][column]) + (sh[lane + 64][column] + sh[lane + 96][column]);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
        if (lane == 0 && int(blockIdx.x) * 8 + column < cols) out[int(blockIdx.x) * 8 + column] = from_f32<T>(s);
    }
}

// Rows of one run: runs of at least 64 rows, at most 592 (four CTAs on each of 148 SMs) of them.
int column_run(int rows) { return std::max(64, (rows + 591) / 592); }

template <typename T, bool E5M2, bool VEC>
void launch_quant(const QuantJob<T>& j, int block_rows, int batch, cudaStream_t stream) {
    const long long rows128 = (j.rows + 127) / 128, col_blocks = (j.cols + 127) / 128;
    const int cb = col_blocks >= 3 ? 4 : int(col_blocks);
    // 256 rows to a CTA where 128 would make more CTAs than three on each of 148 SMs.  Both ways, 128 rows to a CTA
    // and 256, us: bfloat16, 56,960 rows of 8 columns 6.6 and 4.7, of 64 7.2 and 5.4; 165,888 rows of 8 13.6 and 9.4, of
    // 32 13.9 and 9.6, of 64 14.2 and 10.1; float32, 165,888 rows of 8 14.6 and 11.2, of 64 15.9 and 13.2.  Fewer rows lose:
    // bfloat16, 18,944 rows of 64 3.6 and 4.1.
    const bool narrow = block_rows == 1 && j.t_codes && j.cols <= 64 && rows128 > 3 * 148;
    const long long grid = block_rows == 1 && !j.t_codes
                               ? (j.rows * (long long)cb + 127) / 128 * ((col_blocks + cb - 1) / cb)
                           : narrow ? (rows128 + 1) / 2 : rows128 * col_blocks;
    require(grid < (1LL << 31), "matrix is too large");
    const dim3 g(unsigned(grid), unsigned(batch), 1);
    if (block_rows == 1 && !j.t_codes) {
        if (cb == 4) k_quant_rows<T, E5M2, VEC, 4><<<g, kThreads, 0, stream>>>(j);
        else if (cb == 2) k_quant_rows<T, E5M2, VEC, 2><<<g, kThreads, 0, stream>>>(j);
        else k_quant_rows<T, E5M2, VEC, 1><<<g, kThreads, 0, stream>>>(j);
    } else if (narrow) {
        k_quant_tile<T, E5M2, VEC, false, true, true><<<g, kThreads, 0, stream>>>(j);
    } else if (block_rows == 1) {
        k_quant_tile<T, E5M2, VEC, false, true><<<g, kThreads, 0, stream>>>(j);
    } else {
        if (!j.t_codes) k_quant_tile<T, E5M2, VEC, true, false><<<g, kThreads, 0, stream>>>(j);
        else k_quant_tile<T, E5M2, VEC, true, true><<<g, kThreads, 0, stream>>>(j);
    }
    AEISU_CUDA(cudaGetLastError());
}

template <typename T>
void quantize_as(const MatrixRef& x, int block_rows, int code_type, void* codes, long long ld, long long batch_stride,
                 uint8_t* scales, void* t_codes, long long t_ld, long long t_batch, uint8_t* t_scales, float* sums,
                 cudaStream_t stream) {
    QuantJob<T> j{static_cast<const T*>(x.ptr), x.rows, x.cols, x.ld, x.batch_stride, static_cast<uint8_t*>(codes), ld,
                  batch_stride, scales, static_cast<uint8_t*>(t_codes), t_ld, t_batch, t_scales, sums};
    constexpr int n = Vals<T>::n;
    const bool vec = aligned(x.ptr, 16) && x.ld % n == 0 && x.cols % n == 0 && (x.batch == 1 || x.batch_stride % n == 0);
    if (code_type == kE5M2) {
        if (vec) launch_quant<T, true, true>(j, block_rows, x.batch, stream);
        else launch_quant<T, true, false>(j, block_rows, x.batch, stream);
    } else {
        if (vec) launch_quant<T, false, true>(j, block_rows, x.batch, stream);
        else launch_quant<T, false, false>(j, block_rows, x.batch, stream);
    }
}

}  // namespace

void block_quantize(const MatrixRef& x, int block_rows, int code_type, void* codes, long long ld,
                    long long batch_stride, uint8_t* scales, void* t_codes, long long t_ld, long long t_batch_stride,
                    uint8_t* t_scales, float* sums, int device, cudaStream_t stream) {
    require(!sums || (t_codes && block_rows == 1 && x.batch == 1), "column sums come with the codes of the transpose");
    require(x.ptr && codes && scales && (!t_codes || t_scales), "tensor pointer is null");
    require(x.rows >= 1 && x.cols >= 1 && x.batch >= 1 && x.batch <= 65535 && x.ld >= x.cols && !x.trans,
            "matrix sizes are out of range");
    require(block_rows == 1 || block_rows == kBlock, "blocks have 1 or 128 rows");
    require(is_code(code_type), "codes are E4M3 or E5M2");
    require(ld >= x.cols && ld % 16 == 0 && batch_stride % 16 == 0 && aligned(codes, 16),
            "code rows must start on 16-byte boundaries");
    require(!t_codes || (t_ld >= x.rows && t_ld % 16 == 0 && t_batch_stride % 16 == 0 && aligned(t_codes, 16)),
            "code rows of the transpose must start on 16-byte boundaries");
    OnDevice on(device);
    auto go = [&](auto t) {
        quantize_as<decltype(t)>(x, block_rows, code_type, codes, ld, batch_stride, scales, t_codes, t_ld,
                                 t_batch_stride, t_scales, sums, stream);
    };
    if (x.type == kF32) go(float{});
    else if (x.type == kF16) go(__half{});
    else if (x.type == kBF16) go(__nv_bfloat16{});
    else fail(AEISU_ERR_INVALID_ARG, "values must be float32, float16 or bfloat16");
}

void join_sums(const float* partial, int runs, int cols, void* out, int out_type, cudaStream_t stream) {
    auto join = [&](auto t) {
        using T = decltype(t);
        k_column_join<T><<<unsigned((cols + 7) / 8), 1024, 0, stream>>>(partial, runs, cols, static_cast<T*>(out));
    };
    if (out_type == kF32) join(float{});
    else if (out_type == kF16) join(__half{});
    else if (out_type == kBF16) join(__nv_bfloat16{});
    else fail(AEISU_ERR_INVALID_ARG, "sums must be float32, float16 or bfloat16");
    AEISU_CUDA(cudaGetLastError());
}

size_t column_sum_partials(int rows, int cols) {
    const int run = column_run(rows);
    return size_t((rows + run - 1) / run) * cols;
}

void column_sum(const MatrixRef& x, void* out, int out_type, float* partial, int device, cudaStream_t stream) {
    require(x.ptr && out && partial, "tensor pointer is null");
    require(x.rows >= 1 && x.cols >= 1 && x.ld >= x.cols && x.batch == 1 && !x.trans, "matrix sizes are out of range");
    OnDevice on(device);
    const int run = column_run(x.rows), runs = (x.rows + run - 1) / run;
    const dim3 grid(unsigned((x.cols + 63) / 64), unsigned(runs), 1);
    auto in = [&](auto t) {
        using T = decltype(t);
        const T* p = static_cast<const T*>(x.ptr);
        constexpr int n = Vals<T>::n;
        if (aligned(p, 16) && x.ld % n == 0 && x.cols % n == 0)
            k_column_runs<T, true><<<grid, kThreads, 0, stream>>>(p, x.rows, x.cols, x.ld, run, partial);
        else
            k_column_runs<T, false><<<grid, kThreads, 0, stream>>>(p, x.rows, x.cols, x.ld, run, partial);
    };
    if (x.type == kF32) in(float{});
    else if (x.type == kF16) in(__half{});
    else if (x.type == kBF16) in(__nv_bfloat16{});
    else fail(AEISU_ERR_INVALID_ARG, "values must be float32, float16 or bfloat16");
    AEISU_CUDA(cudaGetLastError());
    join_sums(partial, runs, x.cols, out, out_type, stream);
}

}  // namespace aeisu
