// C entry points of the 4-bit matrices (include/b200_spmm.h): argument checks, the device, the status word.
#include <atomic>
#include <map>
#include <utility>

#include "../../include/b200_spmm_kat.h"
#include "common.hpp"
#include "fp4.hpp"

namespace b200spmm {
namespace fp4 {
namespace {

// Waits that ran out on each device that loads the library.  Only counted up: whoever asks compares with what it was told last, so that nobody's
// asking hides a failure from others.
__device__ uint32_t g_status;

std::atomic<uint32_t *> g_status_word[kMaxDevices];
std::atomic<uint32_t> g_counted[kMaxDevices];  // the largest count that anybody has read
std::atomic<int> g_sms[kMaxDevices];

// What this thread knows of a device's count, each one more than that (0: it has not come to the device yet): `first`, what anybody had read when
// it came; `told`, the most it was told since.  And for each stream that it launches to or asks for, by device and handle, what it goes by
// there: at the first launch what it had been told by then, later what it was told there.  (A handle that comes back as another stream finds
// an older count: that may say a failure twice, and hides none.)
struct Known {
    uint64_t first, told;
};
thread_local Known t_known[kMaxDevices];
thread_local std::map<std::pair<int, cudaStream_t>, uint32_t> t_streams;

void come(int device) {
    if (!t_known[device].first) t_known[device].first = t_known[device].told = 1ull + g_counted[device].load();
}

// What b200spmm_kat_fp4_starve asked for; a limit of 0 is none.
thread_local unsigned long long t_starve_ns = 0;
thread_local int t_starve_operand = 0;

// Calls that a capturing thread may not make otherwise (they touch no stream).
struct RelaxedCapture {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
    ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

int check_device(int device) {
    if (device < 0 || device >= kMaxDevices) return B200SPMM_ERR_NO_DEVICE;
    if (g_sms[device].load(std::memory_order_relaxed) > 0) return B200SPMM_OK;
    int n_dev = 0, major = 0, sms = 0;
    if (cudaGetDeviceCount(&n_dev) != cudaSuccess || device >= n_dev) {
        cudaGetLastError();
        return B200SPMM_ERR_NO_DEVICE;
    }
    B200_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
    if (major != 10) return B200SPMM_ERR_NO_DEVICE;
    B200_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    g_sms[device].store(sms, std::memory_order_relaxed);
    return B200SPMM_OK;
}

bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool is_type(int t) { return t == B200SPMM_T_F32 || t == B200SPMM_T_F16 || t == B200SPMM_T_BF16; }
uintptr_t size_of(int t) { return t == B200SPMM_T_F32 ? 4 : 2; }
bool is_empty(const b200spmm_fp4_t *m) { return m->rows == 0 || m->cols == 0; }

int check_matrix(const b200spmm_fp4_t *m) {
    if (!m || (m->format != B200SPMM_NVFP4 && m->format != B200SPMM_MXFP4)) return B200SPMM_ERR_INVALID_ARG;
    if (m->rows > 0x7FFFFFFFull - 128 || m->cols > 0x7FFFFFFFull - 256) return B200SPMM_ERR_UNSUPPORTED;
    if (!m->tensor_scale || !aligned(m->tensor_scale, 4)) return B200SPMM_ERR_INVALID_ARG;
    if (is_empty(m)) return B200SPMM_OK;
    if (!m->values || !m->scales) return B200SPMM_ERR_INVALID_ARG;
    if (!aligned(m->values, 16) || !aligned(m->scales, 16)) return B200SPMM_ERR_UNSUPPORTED;
    return B200SPMM_OK;
}

// A dense matrix of rows x cols, rows `ld` elements apart.
int check_dense(const void *p, int type, uint64_t rows, uint64_t cols, int64_t ld) {
    if (!is_type(type)) return B200SPMM_ERR_INVALID_ARG;
    if (rows == 0 || cols == 0) return B200SPMM_OK;
    if (!p || (rows > 1 && ld < (int64_t)cols) || !aligned(p, size_of(type))) return B200SPMM_ERR_INVALID_ARG;
    return B200SPMM_OK;
}

int zero_output(void *c, int64_t ldc, int type, uint64_t rows, uint64_t cols, cudaStream_t stream) {
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

// The word of the device, which is current.
cudaError_t status_word(int device, uint32_t **word) {
    *word = g_status_word[device].load(std::memory_order_relaxed);
    if (*word) return cudaSuccess;
    void *p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, g_status);
    if (e != cudaSuccess) return e;
    *word = static_cast<uint32_t *>(p);
    g_status_word[device].store(*word, std::memory_order_relaxed);
    return cudaSuccess;
}

int quantize(const void *x, int64_t ldx, int x_dtype, const float *tensor_scale, const b200spmm_fp4_t *by_rows, const b200spmm_fp4_t *by_cols,
             float *workspace, void *stream) {
    for (const b200spmm_fp4_t *m : {by_rows, by_cols})
        if (m) {
            const int st = check_matrix(m);
            if (st != B200SPMM_OK) return st;
        }
    const b200spmm_fp4_t *one = by_rows ? by_rows : by_cols;
    const uint64_t rows = by_rows ? by_rows->rows : by_cols->cols, cols = by_rows ? by_rows->cols : by_cols->rows;
    if (by_rows && by_cols && (by_cols->cols != rows || by_cols->rows != cols || by_rows->format != by_cols->format || by_rows->device != by_cols->device))
        return B200SPMM_ERR_INVALID_ARG;
    const int st = check_dense(x, x_dtype, rows, cols, ldx);
    if (st != B200SPMM_OK) return st;
    if (one->format == B200SPMM_NVFP4 && !tensor_scale && !workspace) return B200SPMM_ERR_INVALID_ARG;
    if (!aligned(tensor_scale, 4) || !aligned(workspace, 4)) return B200SPMM_ERR_INVALID_ARG;
    return on_device(one->device, [&]() -> int {
        return launch_quantize(x, ldx, x_dtype, rows, cols, one->format == B200SPMM_NVFP4 ? tensor_scale : nullptr, by_rows, by_cols, workspace,
                               static_cast<cudaStream_t>(stream));
    });
}

}  // namespace

int sm_count() {
    int device = 0;
    cudaGetDevice(&device);
    return device >= 0 && device < kMaxDevices && g_sms[device] > 0 ? g_sms[device].load() : 148;
}

unsigned long long wait_limit_ns() { return t_starve_ns ? t_starve_ns : kDeviceWaitLimitNs; }
uint32_t rows_of_box(int operand, uint32_t rows) { return t_starve_ns && operand == t_starve_operand ? rows / 2u : rows; }

cudaError_t status_of_launch(cudaStream_t stream, uint32_t **word) {
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    come(device);
    t_streams.try_emplace({device, stream}, (uint32_t)(t_known[device].told - 1u));
    return status_word(device, word);
}

}  // namespace fp4
}  // namespace b200spmm

using namespace b200spmm;
using namespace b200spmm::fp4;

extern "C" {

int b200spmm_fp4_sizes(uint64_t rows, uint64_t cols, int format, uint64_t *pitch, uint64_t *values_bytes, uint64_t *scales_bytes, uint64_t *workspace_bytes) {
    if (format != B200SPMM_NVFP4 && format != B200SPMM_MXFP4) return B200SPMM_ERR_INVALID_ARG;
    if (rows > 0x7FFFFFFFull - 128 || cols > 0x7FFFFFFFull - 256) return B200SPMM_ERR_UNSUPPORTED;
    const Layout l = layout_of(rows, cols, format);
    if (pitch) *pitch = l.pitch;
    if (values_bytes) *values_bytes = rows * l.pitch;
    if (scales_bytes) *scales_bytes = (uint64_t)l.row_blocks * l.groups * 512u;
    if (workspace_bytes) *workspace_bytes = kAmaxBlocks * sizeof(float);
    return B200SPMM_OK;
}

int b200spmm_fp4_quantize(const void *d_X, int64_t ldx, int x_dtype, int transposed, const float *d_tensor_scale, const b200spmm_fp4_t *out,
                          void *workspace, void *stream) {
    if (!out) return B200SPMM_ERR_INVALID_ARG;
    return quantize(d_X, ldx, x_dtype, d_tensor_scale, transposed ? nullptr : out, transposed ? out : nullptr, static_cast<float *>(workspace), stream);
}

int b200spmm_fp4_quantize_both(const void *d_X, int64_t ldx, int x_dtype, const float *d_tensor_scale, const b200spmm_fp4_t *by_rows,
                               const b200spmm_fp4_t *by_cols, void *workspace, void *stream) {
    if (!by_rows || !by_cols) return B200SPMM_ERR_INVALID_ARG;
    return quantize(d_X, ldx, x_dtype, d_tensor_scale, by_rows, by_cols, static_cast<float *>(workspace), stream);
}

int b200spmm_fp4_dequantize(const b200spmm_fp4_t *a, void *d_X, int64_t ldx, int x_dtype, void *stream) {
    int st = check_matrix(a);
    if (st == B200SPMM_OK) st = check_dense(d_X, x_dtype, a->rows, a->cols, ldx);
    if (st != B200SPMM_OK) return st;
    return on_device(a->device, [&]() -> int { return is_empty(a) ? B200SPMM_OK : launch_dequantize(a, d_X, ldx, x_dtype, static_cast<cudaStream_t>(stream)); });
}

int b200spmm_fp4_product_workspace(const b200spmm_fp4_t *a, const void *d_B, int64_t ldb, int64_t n, int b_transposed, uint64_t *bytes) {
    if (!bytes || n < 0) return B200SPMM_ERR_INVALID_ARG;
    *bytes = 0;
    const int st = check_matrix(a);
    if (st != B200SPMM_OK) return st;
    if (n > 0x7FFFFFFF - 256) return B200SPMM_ERR_UNSUPPORTED;
    return on_device(a->device, [&]() -> int {
        if (is_empty(a) || n == 0) return B200SPMM_OK;
        return d_B ? dense_product_workspace(a, d_B, ldb, n, b_transposed != 0, bytes) : product_workspace(a, n, bytes);
    });
}

int b200spmm_fp4_product(const b200spmm_fp4_t *a, const b200spmm_fp4_t *b, void *d_C, int64_t ldc, int c_dtype, int c_transposed, void *workspace,
                         uint64_t workspace_bytes, void *stream) {
    int st = check_matrix(a);
    if (st == B200SPMM_OK) st = check_matrix(b);
    if (st != B200SPMM_OK) return st;
    if (a->cols != b->cols || a->device != b->device) return B200SPMM_ERR_INVALID_ARG;
    if (!aligned(workspace, 16)) return B200SPMM_ERR_INVALID_ARG;
    if (a->format != b->format) return B200SPMM_ERR_UNSUPPORTED;
    const uint64_t rows = c_transposed ? b->rows : a->rows, cols = c_transposed ? a->rows : b->rows;
    st = check_dense(d_C, c_dtype, rows, cols, ldc);
    if (st != B200SPMM_OK) return st;
    return on_device(a->device, [&]() -> int {
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (rows == 0 || cols == 0) return B200SPMM_OK;
        if (a->cols == 0) return zero_output(d_C, ldc, c_dtype, rows, cols, s);
        return launch_product(a, b, d_C, ldc, c_dtype, c_transposed != 0, static_cast<float *>(workspace), workspace_bytes, s);
    });
}

int b200spmm_fp4_dense_product(const b200spmm_fp4_t *a, const void *d_B, int64_t ldb, int64_t n, int b_dtype, int b_transposed, void *d_C, int64_t ldc,
                               int c_dtype, int c_transposed, void *workspace, uint64_t workspace_bytes, void *stream) {
    int st = check_matrix(a);
    if (st != B200SPMM_OK) return st;
    if (n < 0) return B200SPMM_ERR_INVALID_ARG;
    if (n > 0x7FFFFFFF - 256) return B200SPMM_ERR_UNSUPPORTED;
    st = check_dense(d_B, b_dtype, b_transposed ? (uint64_t)n : a->cols, b_transposed ? a->cols : (uint64_t)n, ldb);
    if (st != B200SPMM_OK) return st;
    if (!aligned(workspace, 16)) return B200SPMM_ERR_INVALID_ARG;
    if (b_dtype == B200SPMM_T_F32 || (a->format == B200SPMM_MXFP4 && b_dtype != B200SPMM_T_BF16)) return B200SPMM_ERR_UNSUPPORTED;
    const uint64_t rows = c_transposed ? (uint64_t)n : a->rows, cols = c_transposed ? a->rows : (uint64_t)n;
    st = check_dense(d_C, c_dtype, rows, cols, ldc);
    if (st != B200SPMM_OK) return st;
    return on_device(a->device, [&]() -> int {
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (rows == 0 || cols == 0) return B200SPMM_OK;
        if (a->cols == 0) return zero_output(d_C, ldc, c_dtype, rows, cols, s);
        return launch_dense_product(a, d_B, ldb, n, b_dtype, b_transposed != 0, d_C, ldc, c_dtype, c_transposed != 0, static_cast<uint8_t *>(workspace), workspace_bytes, s);
    });
}

int b200spmm_fp4_status(int device, void *stream_v) {
    return on_device(device, [&]() -> int {
        const cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
        if (is_captured(stream)) return B200SPMM_ERR_UNSUPPORTED;
        uint32_t *word = nullptr, count = 0;
        come(device);
        B200_CUDA_TRY(status_word(device, &word));
        B200_CUDA_TRY(cudaMemcpyAsync(&count, word, sizeof(count), cudaMemcpyDeviceToHost, stream));
        B200_CUDA_TRY(cudaStreamSynchronize(stream));
        if (count == 0) return B200SPMM_OK;
        for (uint32_t most = g_counted[device].load(); most < count && !g_counted[device].compare_exchange_weak(most, count);) {}
        uint32_t &known = t_streams.try_emplace({device, stream}, (uint32_t)(t_known[device].first - 1u)).first->second;
        if (known == count) return B200SPMM_OK;
        known = count;
        t_known[device].told = 1ull + count;
        return B200SPMM_ERR_DEVICE_TIMEOUT;
    });
}

/* Declared in b200_spmm_kat.h: products whose stages can never be complete. */
int b200spmm_kat_fp4_starve(unsigned long long limit_ns, int operand) {
    if (limit_ns > kDeviceWaitLimitNs || (operand != 0 && operand != 1)) return B200SPMM_ERR_INVALID_ARG;
    t_starve_ns = limit_ns;
    t_starve_operand = operand;
    return B200SPMM_OK;
}

}  // extern "C"
