// 4-bit floating-point matrices: what the host and the kernels share about their layout.
//
// A matrix of `rows` x `cols` is kept as
//   values  e2m1 numbers (sign, two exponent bits, one mantissa bit: 0 0.5 1 1.5 2 3 4 6), two to a byte, the lower half
//           first, rows of `pitch` bytes (a multiple of 16), zeros behind the last column;
//   scales  one byte per block of a row: nvfp4 e4m3 for 16 values, mxfp4 a power of two (e8m0) for 32.  128 rows x 4
//           scales lie in 512 bytes, row r's four at (r % 32) * 16 + (r / 32) * 4 - the order in which one copy brings
//           them to the tensor memory columns that the block-scaled MMA reads - row block by row block, with zeros where the
//           matrix ends inside a block;
//   tensor_scale  one fp32 number, a power of two (1 for mxfp4).
// The kernels are launched with programmatic serialization (launch_after) and read what a kernel before them may have written, inputs of the
// caller's included: by ordinary loads only, with no pointer that promises the compiler data which nobody writes, and after their wait for that kernel.
// The reference has no 4-bit form (src/common.h:14-43: fp16 and tf32).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/b200_spmm.h"

namespace b200spmm {
namespace fp4 {

struct Layout {
    uint32_t pitch;       // bytes of a row of values
    uint32_t groups;      // blocks of four scales along a row
    uint32_t row_blocks;  // of 128 rows
};

constexpr int block_of(int format) { return format == B200SPMM_MXFP4 ? 32 : 16; }

inline Layout layout_of(uint64_t rows, uint64_t cols, int format) {
    const uint64_t blk = (uint64_t)block_of(format);
    return {(uint32_t)((cols + 31) / 32 * 16), (uint32_t)((cols + 4 * blk - 1) / (4 * blk)), (uint32_t)((rows + 127) / 128)};
}

constexpr uint32_t kAmaxBlocks = 1024;  // partial maxima of a tensor that one quantisation may leave in its workspace

// The device a call works on is current while this exists.
struct DeviceGuard {
    int before = -1;
    cudaError_t status;
    explicit DeviceGuard(int device) {
        int now = 0;
        status = cudaGetDevice(&now);
        if (status == cudaSuccess && now != device) {
            status = cudaSetDevice(device);
            if (status == cudaSuccess) before = now;
        }
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
    DeviceGuard(const DeviceGuard &) = delete;
};

// Launches, after the entry points' checks of the arguments; the device is current.
int launch_quantize(const void *x, int64_t ldx, int x_dtype, uint64_t x_rows, uint64_t x_cols, const float *tensor_scale,
                    const b200spmm_fp4_t *by_rows, const b200spmm_fp4_t *by_cols, float *workspace, cudaStream_t stream);
int launch_dequantize(const b200spmm_fp4_t *a, void *x, int64_t ldx, int x_dtype, cudaStream_t stream);
int launch_product(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, void *c, int64_t ldc, int c_dtype, bool c_transposed,
                   float *workspace, uint64_t workspace_bytes, cudaStream_t stream);
int product_workspace(const b200spmm_fp4_t *a, int64_t n, uint64_t *bytes);
int launch_dense_product(const b200spmm_fp4_t *a, const void *b, int64_t ldb, int64_t n, int b_dtype, bool b_transposed, void *c,
                         int64_t ldc, int c_dtype, bool c_transposed, uint8_t *workspace, uint64_t workspace_bytes, cudaStream_t stream);
int dense_product_workspace(const b200spmm_fp4_t *a, const void *b, int64_t ldb, int64_t n, bool b_transposed, uint64_t *bytes);

constexpr int kMaxDevices = 64;
// The word in which kernels count waits that ran out, on the current device, for a launch on `stream` by this thread.
cudaError_t status_of_launch(cudaStream_t stream, uint32_t **word);
// Multiprocessors of the current device.
int sm_count();

// How long waits of a product that this thread launches may last, and the rows of the box that a stage of A (operand 0) or B (1) arrives in:
// two seconds and `rows`, but for b200spmm_kat_fp4_starve.
unsigned long long wait_limit_ns();
uint32_t rows_of_box(int operand, uint32_t rows);

}  // namespace fp4
}  // namespace b200spmm
