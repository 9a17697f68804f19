// The epilogue steps for one output at a time, and their argument checks:
// used by the 4-bit products and the products grouped by expert, whose
// threads hold one column and many rows (fused_gemm.cu's kernels hold one row
// and many columns; gemm_common.cuh).
#pragma once

#include <cstring>

#include "internal.h"

namespace mxb {

struct CellEpilogue {
    EpStepDev steps[MXB_MAX_EPILOGUE];
    int n_steps;
    int n_cols;  // the modulo rule's row length
};

namespace {

// Output (row, col) of group `group`: ADD_ROW steps take row `group` of their
// operand when they have a pitch (grouped products), else its only row.
__device__ __forceinline__ float apply_cell(float v, long long row, int col, int group, const CellEpilogue& e) {
    for (int s = 0; s < e.n_steps; ++s) {
        const EpStepDev& st = e.steps[s];
        switch (st.kind) {
            case MXB_EP_RELU: v = v > 0.0f ? v : 0.0f; break;
            case MXB_EP_SCALE: v = v * st.scale; break;
            case MXB_EP_ADD_FULL: v += __ldcs(st.ptr + row * st.ld_or_size + col); break;
            case MXB_EP_ADD_ROW: v += ld_global(st.ptr + group * st.ld_or_size + col); break;
            case MXB_EP_ADD_MOD:
                v += ld_global(st.ptr + (static_cast<unsigned long long>(row) * e.n_cols + col) %
                                             static_cast<unsigned long long>(st.ld_or_size));
                break;
            case MXB_EP_RELU_GRAD: v = __ldcs(st.ptr + row * st.ld_or_size + col) > 0.0f ? v : 0.0f; break;
            default: break;
        }
    }
    return v;
}

// The steps for W outputs of column `col` (rows row .. row + W - 1, the first `n` of them wanted).
template <int W>
__device__ __forceinline__ void apply_column(float (&v)[W], long long row, int n, int col, int group,
                                             const CellEpilogue& e) {
    for (int s = 0; s < e.n_steps; ++s) {
        const EpStepDev& st = e.steps[s];
        if (st.kind == MXB_EP_RELU) {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = v[i] > 0.0f ? v[i] : 0.0f;
        } else if (st.kind == MXB_EP_SCALE) {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = v[i] * st.scale;
        } else if (st.kind == MXB_EP_ADD_ROW) {
            const float b = ld_global(st.ptr + group * st.ld_or_size + col);
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] += b;
        } else if (st.kind == MXB_EP_ADD_MOD) {
            const unsigned long long size = static_cast<unsigned long long>(st.ld_or_size);
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (i < n) v[i] += ld_global(st.ptr + (static_cast<unsigned long long>(row + i) * e.n_cols + col) % size);
        } else {  // ADD_FULL, RELU_GRAD (plain loads: the operand may be the output itself)
            const float* src = st.ptr + row * st.ld_or_size + col;
            float c[W];
#pragma unroll
            for (int i = 0; i < W; ++i) c[i] = i < n ? __ldcs(src + i * st.ld_or_size) : 0.0f;
            if (st.kind == MXB_EP_ADD_FULL) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] += c[i];
            } else {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] = c[i] > 0.0f ? v[i] : 0.0f;
            }
        }
    }
}

// Checks `steps` for an output of n_cols columns and copies them.  `grouped`:
// the steps of the grouped products (RELU_GRAD, ADD_ROW with a pitch between
// groups, no modulo rule); else those of mxb_fused_gemm.
inline bool take_cell_steps(const char* fn, const mxb_ep_step* steps, int n_steps, int n_cols, bool grouped,
                            CellEpilogue& e) {
    e.n_steps = n_steps;
    e.n_cols = n_cols;
    for (int i = 0; i < n_steps; ++i) {
        const mxb_ep_step& s = steps[i];
        bool ok = false;
        switch (s.kind) {
            case MXB_EP_RELU:
            case MXB_EP_SCALE: ok = true; break;
            case MXB_EP_ADD_FULL: ok = s.operand && s.ld_or_size >= n_cols; break;
            case MXB_EP_ADD_ROW: ok = s.operand && (!grouped || s.ld_or_size == 0 || s.ld_or_size >= n_cols); break;
            case MXB_EP_ADD_MOD: ok = !grouped && s.operand && s.ld_or_size >= 1; break;
            case MXB_EP_RELU_GRAD: ok = grouped && s.operand && s.ld_or_size >= n_cols; break;
            default: break;
        }
        if (!ok) {
            set_error("%s: invalid epilogue step %d", fn, i);
            return false;
        }
        memcpy(&e.steps[i], &s, sizeof(s));
        if (s.kind == MXB_EP_ADD_ROW && !grouped) e.steps[i].ld_or_size = 0;  // one row, whatever the field holds
    }
    return true;
}

}  // namespace
}  // namespace mxb
