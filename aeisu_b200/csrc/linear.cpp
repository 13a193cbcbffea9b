// The linear layer in block-scaled FP8 as single calls: forward for serving, forward and backward for
// training, and the rows of a grouped product.  Each call quantises its float operands into the
// caller's workspace and multiplies; between calls of a training step only the transposed codes of
// input and weight are kept, in buffers that the caller owns too.
#include <algorithm>

#include "blockscale_host.h"

namespace aeisu {
namespace {

constexpr size_t kAlign = 256;
size_t padded(size_t n) { return (n + kAlign - 1) / kAlign * kAlign; }
long long code_ld(int cols) { return (cols + 15) / 16 * 16LL; }

// An FP8 operand laid out in a buffer: codes, then scales.
struct Operand {
    MatrixRef m;
    ScaleRef s;
};
size_t operand_bytes(int rows, int cols, int block_rows) {
    return padded(size_t(rows) * code_ld(cols)) +
           padded(size_t((cols + kBlock - 1) / kBlock) * ((rows + block_rows - 1) / block_rows));
}
Operand operand_at(const void* buffer, int type, int rows, int cols, int block_rows) {
    const uint8_t* p = static_cast<const uint8_t*>(buffer);
    const int per = (rows + block_rows - 1) / block_rows;
    return {{p, type, rows, cols, code_ld(cols), 1, 0, false},
            {p + padded(size_t(rows) * code_ld(cols)), block_rows == 1 ? 0 : 7, per, 0}};
}
// Partial sums of the bias gradient.
size_t sums_bytes(int m, int n) {
    return padded(std::max(column_sum_partials(m, n), size_t((m + kBlock - 1) / kBlock) * n) * sizeof(float));
}
void* codes_of(const Operand& o) { return const_cast<void*>(o.m.ptr); }
uint8_t* scales_of(const Operand& o) { return const_cast<uint8_t*>(o.s.ptr); }

// Quantises x into `o` and its transpose into `t` (null: not wanted).
void quantize_into(const MatrixRef& x, int block_rows, const Operand& o, const Operand* t, float* sums, int device,
                   cudaStream_t stream) {
    block_quantize(x, block_rows, o.m.type, codes_of(o), o.m.ld, 0, scales_of(o), t ? codes_of(*t) : nullptr,
                   t ? t->m.ld : 0, 0, t ? scales_of(*t) : nullptr, sums, device, stream);
}

void check_workspace(const void* workspace, size_t have, size_t need) {
    require(need == 0 || (workspace && have >= need && aligned(workspace, 16)), "workspace is too small");
}

}  // namespace

size_t transposed_codes_bytes(int rows, int cols, int block_rows) { return operand_bytes(cols, rows, block_rows); }

size_t linear_workspace(int m, int n, int k, int pass, int device) {
    if (pass == kServe) return operand_bytes(m, k, 1) + product_workspace(m, n, k, device);
    if (pass == kTrainForward)
        return operand_bytes(m, k, 1) + operand_bytes(n, k, kBlock) + product_workspace(m, n, k, device);
    return operand_bytes(m, n, 1) + operand_bytes(n, m, 1) + sums_bytes(m, n) +
           std::max(product_workspace(m, k, n, device), product_workspace(n, k, m, device));
}

void linear_serve(const MatrixRef& x, const MatrixRef& w, const ScaleRef& sw, const ProductOut& out, void* workspace,
                  size_t workspace_bytes, int device, cudaStream_t stream) {
    check_workspace(workspace, workspace_bytes, linear_workspace(x.rows, w.rows, x.cols, kServe, device));
    // Few rows: one kernel does both (one token through 4,096 x 4,096, weights at hand as BlockFP8: 12 us from one
    // Python call to the next instead of 16, of which the GPU takes 9.5 either way).
    if (product_of_values(x, w, sw, out, workspace, workspace_bytes, device, stream)) return;
    const Operand q = operand_at(workspace, kE4M3, x.rows, x.cols, 1);
    const size_t used = operand_bytes(x.rows, x.cols, 1);
    quantize_into(x, 1, q, nullptr, nullptr, device, stream);
    product(q.m, q.s, w, sw, out, static_cast<uint8_t*>(workspace) + used, workspace_bytes - used, true, device, stream);
}

void linear_train_forward(const MatrixRef& x, const MatrixRef& w, const ProductOut& out, void* kept_x, void* kept_w,
                          void* workspace, size_t workspace_bytes, int device, cudaStream_t stream) {
    check_workspace(workspace, workspace_bytes, linear_workspace(x.rows, w.rows, x.cols, kTrainForward, device));
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const Operand q = operand_at(ws, kE4M3, x.rows, x.cols, 1);
    ws += operand_bytes(x.rows, x.cols, 1);
    const Operand r = operand_at(ws, kE4M3, w.rows, w.cols, kBlock);
    ws += operand_bytes(w.rows, w.cols, kBlock);
    const Operand qt = operand_at(kept_x, kE4M3, x.cols, x.rows, 1), rt = operand_at(kept_w, kE4M3, w.cols, w.rows, kBlock);
    quantize_into(w, kBlock, r, kept_w ? &rt : nullptr, nullptr, device, stream);
    quantize_into(x, 1, q, kept_x ? &qt : nullptr, nullptr, device, stream);
    product(q.m, q.s, r.m, r.s, out, ws, workspace_bytes - size_t(ws - static_cast<uint8_t*>(workspace)), true, device,
            stream);
}

void linear_train_backward(const MatrixRef& grad, int k, int code_type, const void* kept_x, const void* kept_w,
                           void* gx, int gx_type, void* gw, int gw_type, void* gb, int gb_type, void* workspace,
                           size_t workspace_bytes, int device, cudaStream_t stream) {
    const int m = grad.rows, n = grad.cols;
    require(k >= 1 && (!gx || kept_w) && (!gw || kept_x), "kept codes are missing");
    require(is_code(code_type), "codes are E4M3 or E5M2");
    check_workspace(workspace, workspace_bytes, linear_workspace(m, n, k, kTrainBackward, device));
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const Operand g = operand_at(ws, code_type, m, n, 1);
    ws += operand_bytes(m, n, 1);
    const Operand gt = operand_at(ws, code_type, n, m, 1);
    ws += operand_bytes(n, m, 1);
    // The bias gradient comes out of the pass that quantises both ways, and is joined when the products, which
    // start under that pass, are on their way; or it has a pass of its own.
    float* sums = reinterpret_cast<float*>(ws);
    ws += sums_bytes(m, n);
    const size_t left = workspace_bytes - size_t(ws - static_cast<uint8_t*>(workspace));
    if (gb && !gw) column_sum(grad, gb, gb_type, sums, device, stream);
    if (gx || gw) quantize_into(grad, 1, g, gw ? &gt : nullptr, gb && gw ? sums : nullptr, device, stream);
    if (gx) {
        const Operand wt = operand_at(kept_w, kE4M3, k, n, kBlock);
        product(g.m, g.s, wt.m, wt.s, {gx, gx_type, k, nullptr, 0}, ws, left, true, device, stream);
    }
    if (gw) {
        const Operand xt = operand_at(kept_x, kE4M3, k, m, 1);
        product(gt.m, gt.s, xt.m, xt.s, {gw, gw_type, k, nullptr, 0}, ws, left, !gx, device, stream);
    }
    if (gb && gw) {
        OnDevice on(device);
        join_sums(sums, (m + kBlock - 1) / kBlock, n, gb, gb_type, stream);
    }
}

size_t grouped_linear_workspace(int rows, int k) { return operand_bytes(rows, k, 1); }

void grouped_linear(const MatrixRef& x, const MatrixRef& w, const ScaleRef& sw, const int* off, const ProductOut& out,
                    bool zero_outside, void* workspace, size_t workspace_bytes, int device, cudaStream_t stream) {
    check_workspace(workspace, workspace_bytes, grouped_linear_workspace(x.rows, x.cols));
    if (grouped_product_of_values(x, w, sw, off, out, zero_outside, device, stream)) return;
    const Operand q = operand_at(workspace, kE4M3, x.rows, x.cols, 1);
    quantize_into(x, 1, q, nullptr, nullptr, device, stream);
    grouped_product(q.m, &q.s, w, &sw, off, out, zero_outside, true, device, stream);
}

}  // namespace aeisu
