// What the C entry points of dense operators share: checks of arguments, the device of a call.
#pragma once

#include "common.hpp"
#include "fp4.hpp"

namespace b200spmm {
namespace fp4 {

// B200SPMM_OK where `device` is one that the kernels run on.
int check_device(int device);

// Calls that a capturing thread may not make otherwise (they touch no stream).
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

inline bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline bool is_type(int t) { return t == B200SPMM_T_F32 || t == B200SPMM_T_F16 || t == B200SPMM_T_BF16; }
inline uintptr_t size_of(int t) { return t == B200SPMM_T_F32 ? 4 : t == B200SPMM_T_E4M3 ? 1 : 2; }

// A dense matrix of rows x cols, rows `ld` elements apart.
inline int check_dense(const void *p, int type, uint64_t rows, uint64_t cols, int64_t ld) {
    if (!is_type(type)) return B200SPMM_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return B200SPMM_OK;
    if (!p || (rows > 1 && ld < (int64_t)cols) || !aligned(p, size_of(type))) return B200SPMM_ERR_INVALID_ARG;
    return B200SPMM_OK;
}

inline int zero_output(void *c, int64_t ldc, int type, uint64_t rows, uint64_t cols, cudaStream_t stream) {
    const size_t esz = size_of(type), width = cols * esz;
    B200_CUDA_TRY(cudaMemset2DAsync(c, rows > 1 ? (size_t)ldc * esz : width, 0, width, rows, stream));
    return B200SPMM_OK;
}

template <class Fn>
int on_device(int device, Fn &&body) {
    return guarded([&]() -> int {
        const int st = check_device(device);
        if (st != B200SPMM_OK) return st;
        const DeviceGuard guard(device);
        B200_CUDA_TRY(guard.status);
        const RelaxedCapture relaxed;
        return body();
    });
}

}  // namespace fp4
}  // namespace b200spmm
