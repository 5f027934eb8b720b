// Matrices of 4-bit integers on the host's side: checks of a b200spmm_int4_t, and what kernels get of it.
#pragma once

#include <atomic>

#include "entry.hpp"
#include "narrow.cuh"

namespace b200spmm {
namespace narrow {

inline int check_int4(const b200spmm_int4_t *m) {
    if (!m || (m->scale_dtype != B200SPMM_T_F16 && m->scale_dtype != B200SPMM_T_BF16)) return B200SPMM_ERR_INVALID_ARG;
    if (m->group != 0 && (m->group < 32 || (m->group & (m->group - 1)) != 0)) return B200SPMM_ERR_INVALID_ARG;
    if (m->rows > 0x7FFFFFFFull - 256 || m->cols > 0x7FFFFFFFull - 512) return B200SPMM_ERR_UNSUPPORTED;
    if (m->group && m->rows * ((m->cols + m->group - 1) / m->group) > 0xFFFFFFFFull) return B200SPMM_ERR_UNSUPPORTED;  // (kernels count scales in 32 bits)
    if (m->rows == 0 || m->cols == 0) return B200SPMM_OK;
    if (!m->values || !m->scales || !fp4::aligned(m->scales, 2)) return B200SPMM_ERR_INVALID_ARG;
    if (!fp4::aligned(m->values, 16)) return B200SPMM_ERR_UNSUPPORTED;
    return B200SPMM_OK;
}

inline uint32_t shift_of(int group) {
    uint32_t s = kWholeGroup;
    if (group)
        for (s = 0; (1 << s) < group; ++s) {}
    return s;
}
// The widest span of columns that has one scale and that kernels are made for.
inline uint32_t span_of(const b200spmm_int4_t *m) { return m->group ? std::min(m->group, 128) : 128; }

inline Matrix matrix_of(const b200spmm_int4_t *m) {
    Matrix out{};
    out.values = static_cast<const uint8_t *>(m->values);
    out.pitch = (m->cols + 31) / 32 * 16;
    out.row_bytes = (uint32_t)out.pitch;
    out.shift = shift_of(m->group);
    out.groups = m->group ? (uint32_t)((m->cols + m->group - 1) / m->group) : 1;
    out.rows = (uint32_t)m->rows;
    out.scales = static_cast<const uint16_t *>(m->scales);
    out.zeros = m->zeros ? m->zeros : static_cast<const uint8_t *>(m->scales);
    out.zero_mask = m->zeros ? 15u : 0u;
    out.zero_else = m->zeros ? 0u : 8u;
    out.bf16_scales = m->scale_dtype == B200SPMM_T_BF16;
    return out;
}

// How many of `steps` of `cols` columns there is room for beside `taken` bytes of a block's shared memory; a column has `scales` bytes of them for each step.
template <class W>
uint32_t steps_that_fit(uint32_t steps, uint32_t cols, uint32_t scales, uint64_t taken) {
    static_assert(W::kUnits * 16u % 128u == 0, "a column's steps are multiples of what it is rounded up to");
    if (taken >= kMaxSmem) return 0;
    const uint64_t room = (kMaxSmem - taken) / cols;  // bytes that a column may take
    if (room < column_pitch<W>(0)) return 0;
    return (uint32_t)std::min<uint64_t>((room - column_pitch<W>(0)) / (W::kUnits * 16u + scales), steps);
}

// Lets a kernel have so much shared memory, once for each device; `allowed` keeps which.
template <typename... P>
cudaError_t allow_smem(void (*kernel)(P...), std::atomic<uint64_t> &allowed, uint32_t bytes = kMaxSmem) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (allowed.load(std::memory_order_relaxed) >> device & 1u)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) allowed.fetch_or(1ull << device);
    return e;
}

}  // namespace narrow
}  // namespace b200spmm
