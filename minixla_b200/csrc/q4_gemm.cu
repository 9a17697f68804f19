// Products with 4-bit weights and group scales (mxb_q4_gemm):
//   out[m, n] = epi(sum over groups g of s[n, g] * sum over k in g of A[m, k] * (q[n, k] - z[n, g])).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>

#include "epilogue_cell.cuh"
#include "runtime_internal.h"

namespace mxb {

namespace {

struct Q4Params {
    const float* a;
    long long lda;
    const unsigned char* q;
    long long ldq;
    const void* scales;
    const unsigned char* zeros;
    long long lds;
    int scale_type, group;
    float* out;
    long long ldo;
    int M, N, K;
    CellEpilogue epi;
};

__device__ __forceinline__ float load_scale(const Q4Params& p, long long at) {
    if (p.scale_type == MXB_SCALE_F32) return __ldg(static_cast<const float*>(p.scales) + at);
    const unsigned short raw = __ldg(static_cast<const unsigned short*>(p.scales) + at);
    return p.scale_type == MXB_SCALE_F16 ? __half2float(__ushort_as_half(raw))
                                         : __bfloat162float(__ushort_as_bfloat16(raw));
}

// A warp per output column and up to kRows rows of A: lane l takes the 8
// values of word l, l + 32, ... of the column's weights.
constexpr int kRows = 8, kWarps = 8;

__global__ void __launch_bounds__(32 * kWarps) q4_simple_kernel(const __grid_constant__ Q4Params p) {
    const int lane = threadIdx.x & 31;
    const int n = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int m0 = blockIdx.y * kRows, rows = min(kRows, p.M - m0);
    if (n >= p.N) return;
    float acc[kRows] = {};
    const unsigned* q = reinterpret_cast<const unsigned*>(p.q + n * p.ldq);
    for (int k0 = lane * 8; k0 < p.K; k0 += 256) {
        const unsigned w = __ldg(q + k0 / 8);
        const long long g = n * p.lds + k0 / p.group;
        const float s = load_scale(p, g);
        const float z = p.zeros ? static_cast<float>(__ldg(p.zeros + g) & 15) : 8.0f;
        float part[kRows] = {};
        for (int i = 0; i < 8 && k0 + i < p.K; ++i) {
            const float v = static_cast<float>((w >> (4 * i)) & 15u) - z;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (r < rows) part[r] += v * __ldg(p.a + (m0 + r) * p.lda + k0 + i);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) acc[r] += s * part[r];
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == 0 && r < rows) p.out[(m0 + r) * p.ldo + n] = apply_cell(acc[r], m0 + r, n, 0, p.epi);
    }
}

int q4_gemm(GpuCtx* ctx, Q4Params& p, const mxb_ep_step* steps, int n_steps, void* stream) {
    if (!ctx || !p.a || !p.q || !p.scales || !p.out || p.M < 1 || p.N < 1 || p.K < 1 || p.lda < p.K || p.ldo < p.N ||
        p.group < 32 || p.group % 32 || n_steps < 0 || n_steps > MXB_MAX_EPILOGUE || (n_steps > 0 && !steps) ||
        p.scale_type < MXB_SCALE_F32 || p.scale_type > MXB_SCALE_BF16) {
        set_error("mxb_q4_gemm: invalid arguments");
        return MXB_E_ARG;
    }
    if (p.ldq < (static_cast<long long>(p.K) + 1) / 2 || p.lds < (static_cast<long long>(p.K) + p.group - 1) / p.group) {
        set_error("mxb_q4_gemm: a weight row needs (K + 1) / 2 bytes and ceil(K / group) scales");
        return MXB_E_ARG;
    }
    const uintptr_t scale_mask = p.scale_type == MXB_SCALE_F32 ? 3 : 1;
    if (p.lda % 4 || (reinterpret_cast<uintptr_t>(p.a) & 15) || p.ldq % 16 || (reinterpret_cast<uintptr_t>(p.q) & 15) ||
        (reinterpret_cast<uintptr_t>(p.scales) & scale_mask)) {
        set_error("mxb_q4_gemm: A and Q need 16-byte aligned bases and row pitches (lda %% 4 == 0, ldq %% 16 == 0)");
        return MXB_E_ARG;
    }
    if (!take_cell_steps("mxb_q4_gemm", steps, n_steps, p.N, false, p.epi)) return MXB_E_ARG;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    const dim3 grid((p.N + kWarps - 1) / kWarps, (p.M + kRows - 1) / kRows);
    q4_simple_kernel<<<grid, 32 * kWarps, 0, st>>>(p);
    note_launch();
    return cuda_ok(cudaGetLastError(), "4-bit product launch") ? MXB_OK : MXB_E_CUDA;
}

}  // namespace
}  // namespace mxb

extern "C" int mxb_q4_gemm(GpuCtx* ctx, const float* A, long long lda, const unsigned char* Q, long long ldq,
                           const void* scales, int scale_type, const unsigned char* zeros, long long lds, int group,
                           float* out, long long ldo, int M, int N, int K, const mxb_ep_step* steps, int n_steps,
                           void* stream) {
    try {
        mxb::Q4Params p{A, lda, Q, ldq, scales, zeros, lds, scale_type, group, out, ldo, M, N, K, {}};
        return mxb::q4_gemm(ctx, p, steps, n_steps, stream);
    } catch (const std::exception& e) {  // host allocations of the pool's lists
        mxb::set_error("mxb_q4_gemm: %s", e.what());
        return MXB_E_NOMEM;
    }
}
