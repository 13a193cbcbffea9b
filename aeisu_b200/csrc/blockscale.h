// Block-scaled FP8 operands and matrix products, dense and grouped by expert (k_blockq.cu,
// k_prod.cu).  All entry points enqueue on `stream` and return; pointers are device pointers.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace aeisu {

// Element types of the C boundary (AEISU_TYPE_* of aeisu.h).
enum ElemType : int { kF32 = 0, kF16 = 1, kBF16 = 2, kE4M3 = 3, kE5M2 = 4 };
inline int elem_bytes(int t) { return t == kF32 ? 4 : t <= kBF16 ? 2 : 1; }

constexpr int kBlock = 128;        // values per scale along a row
constexpr int kMaxSide = 0x7fffffff - 1024;   // rows or columns of a matrix
constexpr int kMaxGroups = 1024;   // groups of one grouped product (offsets live in shared memory)

// A batch of matrices [batch][rows][cols], cols contiguous unless `trans` (then rows are:
// element (r, c) sits at c * ld + r).
struct MatrixRef {
    const void* ptr;
    int type;
    int rows, cols;
    long long ld;
    int batch;
    long long batch_stride;
    bool trans;
};

// Scales of an FP8 operand: one E8M0 byte per (block column, row >> shift), block column major.
struct ScaleRef {
    const uint8_t* ptr;
    int shift;               // 0: one scale per row; 7: one per 128 rows
    int ld;                  // scales per block column
    long long batch_stride;
};

// `sums` (null, or with t_codes and single rows): the column sums of every 128 rows, [row blocks][cols].
void block_quantize(const MatrixRef& x, int block_rows, int code_type, void* codes, long long ld,
                    long long batch_stride, uint8_t* scales, void* t_codes, long long t_ld, long long t_batch_stride,
                    uint8_t* t_scales, float* sums, int device, cudaStream_t stream);

// out[c] = sum over rows of x[r][c], added in 32 bits in a fixed order; `partial` holds
// column_sum_partials(rows, cols) floats.
void join_sums(const float* partial, int runs, int cols, void* out, int out_type, cudaStream_t stream);
size_t column_sum_partials(int rows, int cols);
void column_sum(const MatrixRef& x, void* out, int out_type, float* partial, int device, cudaStream_t stream);

// out[m][n] = sum_k a[m][k] b[n][k] (+ bias[n]) of FP8 operands.
struct ProductOut {
    void* ptr;
    int type;
    long long ld;
    const void* bias;        // n values of bias_type, or null
    int bias_type;
};
size_t product_workspace(int m, int n, int k, int device);
// after_quantize: the kernel enqueued just before on `stream` is the quantiser of an operand, and the
// product may start while it runs.
void product(const MatrixRef& a, const ScaleRef& sa, const MatrixRef& b, const ScaleRef& sb, const ProductOut& out,
             void* workspace, size_t workspace_bytes, bool after_quantize, int device, cudaStream_t stream);

// The same with float rows x, which the product quantises to E4M3 in blocks of 1 x 128 itself; false, and
// nothing done, where there are too many or their type or alignment does not allow it.
bool product_of_values(const MatrixRef& x, const MatrixRef& b, const ScaleRef& sb, const ProductOut& out,
                       void* workspace, size_t workspace_bytes, int device, cudaStream_t stream);

// Rows t in [off[e], off[e + 1]) of x [rows][k] times b[e] [n][k]: out[t][n].  Rows outside every
// group are zeroed when zero_outside is set, otherwise left as they were.
void grouped_product(const MatrixRef& x, const ScaleRef* sx, const MatrixRef& b, const ScaleRef* sb, const int* off,
                     const ProductOut& out, bool zero_outside, bool after_quantize, int device, cudaStream_t stream);
bool grouped_product_of_values(const MatrixRef& x, const MatrixRef& b, const ScaleRef& sb, const int* off,
                               const ProductOut& out, bool zero_outside, int device, cudaStream_t stream);
// out[e][n][k] = sum over t in group e of g[t][n] x[t][k].
void grouped_weight_gradient(const MatrixRef& g, const MatrixRef& x, const int* off, int groups, void* out,
                             int out_type, int device, cudaStream_t stream);
// The linear layer in block-scaled FP8 (linear.cpp): quantiser and products in one call, operands
// and partial results carved out of one workspace.
enum LinearPass { kServe = 0, kTrainForward = 1, kTrainBackward = 2 };
size_t linear_workspace(int m, int n, int k, int pass, int device);
size_t transposed_codes_bytes(int rows, int cols, int block_rows);   // codes and scales of the transpose
void linear_serve(const MatrixRef& x, const MatrixRef& w, const ScaleRef& sw, const ProductOut& out, void* workspace,
                  size_t workspace_bytes, int device, cudaStream_t stream);
void linear_train_forward(const MatrixRef& x, const MatrixRef& w, const ProductOut& out, void* kept_x, void* kept_w,
                          void* workspace, size_t workspace_bytes, int device, cudaStream_t stream);
void linear_train_backward(const MatrixRef& grad, int k, int code_type, const void* kept_x, const void* kept_w,
                           void* gx, int gx_type, void* gw, int gw_type, void* gb, int gb_type, void* workspace,
                           size_t workspace_bytes, int device, cudaStream_t stream);
size_t grouped_linear_workspace(int rows, int k);
void grouped_linear(const MatrixRef& x, const MatrixRef& w, const ScaleRef& sw, const int* off, const ProductOut& out,
                    bool zero_outside, void* workspace, size_t workspace_bytes, int device, cudaStream_t stream);

// The error code that a product kernel left behind on `device` (0: none), cleared; waits for the device.
int product_status(int device);

}  // namespace aeisu
