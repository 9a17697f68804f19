// Products grouped by expert (mxb_grouped_gemm and its gradients): rows
// offsets[e] .. offsets[e+1] - 1 belong to group e and meet its own matrix.
//   forward  out[r, n]   = epi(sum over k of A[r, k] * B_e[k, n])
//   grad_a   dA[r, k]    = epi(sum over n of dY[r, n] * B_e[k, n])
//   grad_b   dB_e[k, n]  = sum over the group's rows r of A[r, k] * dY[r, n],  dbias[e, n] = sum over r of dY[r, n]
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>

#include "epilogue_cell.cuh"
#include "runtime_internal.h"

namespace mxb {

namespace {

enum GroupedMode : int { kForward, kGradA, kGradB };

struct GroupedParams {
    int mode;
    const float* x;      // forward: A; grad_a: dY; grad_b: A          (row matrix)
    long long ldx;
    const float* w;      // forward, grad_a: B; grad_b: dY             (weights, or the other row matrix)
    long long ldw, w_stride;
    const int* offsets;
    int groups, rows;
    float* out;          // out, dA, or dB
    long long ldo, out_stride;
    float* dbias;
    int N, K;
    CellEpilogue epi;
};

// Group e's rows [r0, r1), whatever offsets holds: 0 <= r0 <= r1 <= rows.
__device__ __forceinline__ void group_rows(const GroupedParams& p, int e, int& r0, int& r1) {
    r0 = min(max(__ldg(p.offsets + e), 0), p.rows);
    r1 = min(max(__ldg(p.offsets + e + 1), r0), p.rows);
}

// 32 x 32 outputs per block, one group per blockIdx.z; the row tiles of a
// group are walked by the blocks of blockIdx.y in turn.
__global__ void __launch_bounds__(1024) grouped_simple_kernel(const __grid_constant__ GroupedParams p) {
    __shared__ float left[32][33], right[32][33];
    const int e = blockIdx.z, tx = threadIdx.x, ty = threadIdx.y;
    int r0, r1;
    group_rows(p, e, r0, r1);
    const int out_rows = p.mode == kGradB ? p.K : r1 - r0;
    const int out_cols = p.mode == kGradA ? p.K : p.N;
    const int len = p.mode == kForward ? p.K : p.mode == kGradA ? p.N : r1 - r0;
    const int c = blockIdx.x * 32 + tx;
    const float* w = p.w + (p.mode == kGradB ? r0 * p.ldw : e * p.w_stride);
    for (int i0 = blockIdx.y * 32; i0 < out_rows; i0 += gridDim.y * 32) {
        const int i = i0 + ty;
        float acc = 0.0f, colsum = 0.0f;
        for (int l0 = 0; l0 < len; l0 += 32) {
            // left[i][l], right[l][c]
            float a = 0.0f, b = 0.0f;
            if (p.mode == kGradB) {
                if (i0 + tx < out_rows && l0 + ty < len) a = __ldg(p.x + (r0 + l0 + ty) * p.ldx + i0 + tx);
                left[tx][ty] = a;
                if (c < out_cols && l0 + ty < len) b = __ldg(w + (l0 + ty) * p.ldw + c);
                right[ty][tx] = b;
            } else {
                if (i < out_rows && l0 + tx < len) a = __ldg(p.x + (r0 + i) * p.ldx + l0 + tx);
                left[ty][tx] = a;
                if (p.mode == kForward) {
                    if (c < out_cols && l0 + ty < len) b = __ldg(w + (l0 + ty) * p.ldw + c);
                    right[ty][tx] = b;
                } else {
                    const int cc = blockIdx.x * 32 + ty;
                    if (cc < out_cols && l0 + tx < len) b = __ldg(w + cc * p.ldw + l0 + tx);
                    right[tx][ty] = b;
                }
            }
            __syncthreads();
            for (int l = 0; l < 32; ++l) {
                acc += left[ty][l] * right[l][tx];
                colsum += right[l][tx];
            }
            __syncthreads();
        }
        if (i >= out_rows || c >= out_cols) continue;
        if (p.mode == kGradB) {
            p.out[e * p.out_stride + i * p.ldo + c] = acc;
            if (p.dbias && i == 0) p.dbias[static_cast<long long>(e) * p.N + c] = colsum;
        } else {
            p.out[(r0 + i) * p.ldo + c] = apply_cell(acc, r0 + i, c, e, p.epi);
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int grouped_gemm(const char* fn, GpuCtx* ctx, GroupedParams& p, const mxb_ep_step* steps, int n_steps, int precision,
                 void* stream) {
    const bool grad_b = p.mode == kGradB;
    const int x_cols = p.mode == kGradA ? p.N : p.K, out_cols = p.mode == kGradA ? p.K : p.N;
    const long long w_cols = p.N;
    if (!ctx || !p.offsets || p.groups < 1 || p.groups > MXB_MAX_GROUPS || p.rows < 0 || p.N < 1 || p.K < 1 ||
        p.ldx < x_cols || p.ldw < w_cols || p.ldo < out_cols || n_steps < 0 || n_steps > MXB_MAX_EPILOGUE ||
        (n_steps > 0 && !steps) || (precision != GPU_PRECISION_TF32 && precision != GPU_PRECISION_3XTF32) ||
        ((p.rows > 0 || grad_b) && !p.out) || (p.rows > 0 && (!p.x || !p.w))) {
        set_error("%s: invalid arguments", fn);
        return MXB_E_ARG;
    }
    if (p.groups > 1 && ((!grad_b && p.w_stride < (p.K - 1) * p.ldw + p.N) ||
                         (grad_b && p.out_stride < (p.K - 1) * p.ldo + p.N))) {
        set_error("%s: the groups' matrices overlap", fn);
        return MXB_E_ARG;
    }
    if (p.ldx % 4 || p.ldw % 4 || (!grad_b && p.groups > 1 && p.w_stride % 4) || !aligned16(p.x) || !aligned16(p.w)) {
        set_error("%s: the operands need 16-byte aligned bases, pitches and group strides (multiples of 4)", fn);
        return MXB_E_ARG;
    }
    if (!take_cell_steps(fn, steps, n_steps, out_cols, true, p.epi)) return MXB_E_ARG;
    if (p.rows == 0 && !grad_b) return MXB_OK;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    const int tiles = ((grad_b ? p.K : p.rows) + 31) / 32;
    grouped_simple_kernel<<<dim3((out_cols + 31) / 32, std::min(tiles, 64), p.groups), dim3(32, 32), 0, st>>>(p);
    note_launch();
    return cuda_ok(cudaGetLastError(), "grouped product launch") ? MXB_OK : MXB_E_CUDA;
}

}  // namespace
}  // namespace mxb

extern "C" {

int mxb_grouped_gemm(GpuCtx* ctx, const float* A, long long lda, const float* B, long long ldb, long long b_stride,
                     const int* offsets, int groups, float* out, long long ldo, int rows, int N, int K,
                     const mxb_ep_step* steps, int n_steps, int precision, void* stream) {
    mxb::GroupedParams p{mxb::kForward, A, lda, B, ldb, b_stride, offsets, groups, rows, out, ldo, 0, nullptr, N, K, {}};
    return mxb::grouped_gemm("mxb_grouped_gemm", ctx, p, steps, n_steps, precision, stream);
}

int mxb_grouped_gemm_grad_a(GpuCtx* ctx, const float* dY, long long lddy, const float* B, long long ldb,
                            long long b_stride, const int* offsets, int groups, float* dA, long long ldda, int rows,
                            int N, int K, const mxb_ep_step* steps, int n_steps, int precision, void* stream) {
    mxb::GroupedParams p{mxb::kGradA, dY, lddy, B, ldb, b_stride, offsets, groups, rows, dA, ldda, 0, nullptr, N, K, {}};
    return mxb::grouped_gemm("mxb_grouped_gemm_grad_a", ctx, p, steps, n_steps, precision, stream);
}

int mxb_grouped_gemm_grad_b(GpuCtx* ctx, const float* A, long long lda, const float* dY, long long lddy,
                            const int* offsets, int groups, float* dB, long long lddb, long long db_stride,
                            float* dbias, int rows, int N, int K, int precision, void* stream) {
    mxb::GroupedParams p{mxb::kGradB, A, lda, dY, lddy, 0, offsets, groups, rows, dB, lddb, db_stride, dbias, N, K, {}};
    return mxb::grouped_gemm("mxb_grouped_gemm_grad_b", ctx, p, nullptr, 0, precision, stream);
}

}  // extern "C"
