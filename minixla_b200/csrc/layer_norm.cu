// Layer norm and its backward pass (mxb_layer_norm, mxb_layer_norm_backward).
//
// Forward, row by row: mean = sum(x) / C, var = sum((x - mean)^2) / C,
// rstd = 1 / sqrt(var + eps), y = (x - mean) * rstd * gamma + beta.
// Backward, with v = dy * gamma and xhat = (x - mean) * rstd:
//   dx = rstd * (v - sum(v) / C - xhat * sum(v * xhat) / C),
//   dgamma = sum over rows of dy * xhat, dbeta = sum over rows of dy.
// Everything is fp32; the variance is taken around the mean (a second pass
// over the registers), never as a difference of two large sums.
//
// Bound by HBM: x in, y out (backward: x and dy in, dx out), each once.  A
// row is held in registers between its sums and its output, by one warp up
// to 1024 columns and by a block beyond; only rows longer than a block can
// hold are read again (from L2).  The gradients of gamma and beta are summed
// per thread over the rows its block walks through, then stored as one
// partial row per block and summed by a second small kernel in block order,
// so the result does not depend on timing.
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>

#include "runtime_internal.h"

namespace mxb {

namespace {

struct NormParams {
    const float* x;
    long long ldx;
    const float* gamma;
    const float* beta;
    float eps;
    float* y;
    long long ldy;
    float* mean;
    float* rstd;
    long long rows;
    int cols;
};

struct NormGradParams {
    const float* dy;
    long long lddy;
    const float* x;
    long long ldx;
    const float* gamma;
    const float* mean;
    const float* rstd;
    float* dx;
    long long lddx;
    float* partial;   // [block][2][cols]: dgamma, dbeta (nullptr: neither is wanted)
    long long rows;
    int cols;
};

// W consecutive floats at p + c, zeros from column `cols` on.
template <int W>
__device__ __forceinline__ void load_unit(float (&v)[W], const float* p, int c, int cols) {
    if (W == 4 && c + W <= cols) {
        const float4 t = __ldcs(reinterpret_cast<const float4*>(p + c));
        v[0] = t.x;
        v[W > 1 ? 1 : 0] = t.y;
        v[W > 2 ? 2 : 0] = t.z;
        v[W > 3 ? 3 : 0] = t.w;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = c + i < cols ? __ldcs(p + c + i) : 0.0f;
    }
}

// The same for a vector that every row reads (gamma, beta): cached; `absent` where there is none.
template <int W>
__device__ __forceinline__ void load_param(float (&v)[W], const float* p, int c, int cols, float absent) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = absent;
    } else if (W == 4 && c + W <= cols) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(p + c));
        v[0] = t.x;
        v[W > 1 ? 1 : 0] = t.y;
        v[W > 2 ? 2 : 0] = t.z;
        v[W > 3 ? 3 : 0] = t.w;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = c + i < cols ? __ldg(p + c + i) : 0.0f;
    }
}

template <int W>
__device__ __forceinline__ void store_unit(const float (&v)[W], float* p, int c, int cols) {
    if (W == 4 && c + W <= cols) {
        __stcs(reinterpret_cast<float4*>(p + c), make_float4(v[0], v[W > 1 ? 1 : 0], v[W > 2 ? 2 : 0], v[W > 3 ? 3 : 0]));
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (c + i < cols) __stcs(p + c + i, v[i]);
    }
}

__device__ __forceinline__ float2 warp_sum(float2 s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    return s;
}

// Sums over the threads of a row: one warp, or the block.  Two buffers take
// turns, so one barrier per sum is enough: a thread writes a buffer again
// only after the barrier of the sum in between, which every reader of the
// earlier values has reached.
template <bool WARP>
struct RowSum {
    float2 (*buf)[32];
    int turn = 0;
    __device__ __forceinline__ float2 operator()(float2 s) {
        s = warp_sum(s);
        if (WARP) return s;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) buf[turn][warp] = s;
        __syncthreads();
        s = lane < static_cast<int>(blockDim.x >> 5) ? buf[turn][lane] : make_float2(0.0f, 0.0f);
        turn ^= 1;
        return warp_sum(s);
    }
};

constexpr int kWarpRowThreads = 256;  // blocks of eight warps, a row each

// Each thread holds NV units of W floats of its row, unit u at columns
// (u * threads + t) * W.
template <int W, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRowThreads : 1024)
    layer_norm_kernel(const NormParams p) {
    __shared__ float2 buf[2][32];
    RowSum<WARP> row_sum{buf};
    const int threads = WARP ? 32 : blockDim.x;
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const long long rows_at_once = static_cast<long long>(gridDim.x) * (WARP ? kWarpRowThreads / 32 : 1);
    long long row = WARP ? blockIdx.x * static_cast<long long>(kWarpRowThreads / 32) + (threadIdx.x >> 5) : blockIdx.x;
    const float inv = 1.0f / static_cast<float>(p.cols);
    for (; row < p.rows; row += rows_at_once) {
        const float* x = p.x + row * p.ldx;
        float v[NV][W];
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < NV; ++u) load_unit<W>(v[u], x, (u * threads + t) * W, p.cols);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) s.x += v[u][i];
        const float mean = row_sum(s).x * inv;
        s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float d = (u * threads + t) * W + i < p.cols ? v[u][i] - mean : 0.0f;
                s.x += d * d;
            }
        const float rstd = 1.0f / sqrtf(row_sum(s).x * inv + p.eps);
        if (t == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        float* y = p.y + row * p.ldy;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int c = (u * threads + t) * W;
            float g[W], b[W];
            load_param<W>(g, p.gamma, c, p.cols, 1.0f);
            load_param<W>(b, p.beta, c, p.cols, 0.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) v[u][i] = (v[u][i] - mean) * rstd * g[i] + b[i];
            store_unit<W>(v[u], y, c, p.cols);
        }
    }
}

// Rows too long for a block's registers: three passes over the row, the
// second and third from L2.
template <int W>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(const NormParams p) {
    __shared__ float2 buf[2][32];
    RowSum<false> row_sum{buf};
    const int step = blockDim.x * W;
    const float inv = 1.0f / static_cast<float>(p.cols);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float* x = p.x + row * p.ldx;
        float* y = p.y + row * p.ldy;
        float v[W];
        float2 s = make_float2(0.0f, 0.0f);
        for (long long c = threadIdx.x * W; c < p.cols; c += step) {
            load_unit<W>(v, x, static_cast<int>(c), p.cols);
#pragma unroll
            for (int i = 0; i < W; ++i) s.x += v[i];
        }
        const float mean = row_sum(s).x * inv;
        s = make_float2(0.0f, 0.0f);
        for (long long c = threadIdx.x * W; c < p.cols; c += step) {
            load_unit<W>(v, x, static_cast<int>(c), p.cols);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float d = c + i < p.cols ? v[i] - mean : 0.0f;
                s.x += d * d;
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum(s).x * inv + p.eps);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[row] = mean;
            if (p.rstd) p.rstd[row] = rstd;
        }
        for (long long c = threadIdx.x * W; c < p.cols; c += step) {
            float g[W], b[W];
            load_unit<W>(v, x, static_cast<int>(c), p.cols);
            load_param<W>(g, p.gamma, static_cast<int>(c), p.cols, 1.0f);
            load_param<W>(b, p.beta, static_cast<int>(c), p.cols, 0.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = (v[i] - mean) * rstd * g[i] + b[i];
            store_unit<W>(v, y, static_cast<int>(c), p.cols);
        }
    }
}

template <int W, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRowThreads : 512)
    layer_norm_grad_kernel(const NormGradParams p) {
    __shared__ float2 buf[2][32];
    extern __shared__ float block_acc[];  // WARP: [2][cols], the block's sums over its warps
    RowSum<WARP> row_sum{buf};
    const int threads = WARP ? 32 : blockDim.x;
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
    const long long rows_at_once = static_cast<long long>(gridDim.x) * (WARP ? kWarpRowThreads / 32 : 1);
    long long row = WARP ? blockIdx.x * static_cast<long long>(kWarpRowThreads / 32) + (threadIdx.x >> 5) : blockIdx.x;
    const float inv = 1.0f / static_cast<float>(p.cols);
    float dg[NV][W], db[NV][W], g[NV][W];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        load_param<W>(g[u], p.gamma, (u * threads + t) * W, p.cols, 1.0f);
#pragma unroll
        for (int i = 0; i < W; ++i) dg[u][i] = db[u][i] = 0.0f;
    }
    for (; row < p.rows; row += rows_at_once) {
        const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
        const float* x = p.x + row * p.ldx;
        const float* dy = p.dy + row * p.lddy;
        float xh[NV][W], d[NV][W];
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            load_unit<W>(xh[u], x, (u * threads + t) * W, p.cols);
            load_unit<W>(d[u], dy, (u * threads + t) * W, p.cols);
        }
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                // Columns past the row have d = 0: they add nothing to any sum.
                xh[u][i] = (xh[u][i] - mean) * rstd;
                dg[u][i] += d[u][i] * xh[u][i];
                db[u][i] += d[u][i];
                d[u][i] *= g[u][i];
                s.x += d[u][i];
                s.y += d[u][i] * xh[u][i];
            }
        if (!p.dx) continue;
        s = row_sum(s);
        const float m1 = s.x * inv, m2 = s.y * inv;
        float* dx = p.dx + row * p.lddx;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
#pragma unroll
            for (int i = 0; i < W; ++i) d[u][i] = rstd * (d[u][i] - m1 - xh[u][i] * m2);
            store_unit<W>(d[u], dx, (u * threads + t) * W, p.cols);
        }
    }
    if (!p.partial) return;
    float* out = p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols;
    if constexpr (!WARP) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int c = (u * threads + t) * W + i;
                if (c < p.cols) {
                    out[c] = dg[u][i];
                    out[p.cols + c] = db[u][i];
                }
            }
    } else {
        // The warps add their sums one after the other, in warp order.
        for (int w = 0; w < kWarpRowThreads / 32; ++w) {
            if (static_cast<int>(threadIdx.x >> 5) == w) {
#pragma unroll
                for (int u = 0; u < NV; ++u)
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        const int c = (u * 32 + t) * W + i;
                        if (c < p.cols) {
                            block_acc[c] = (w ? block_acc[c] : 0.0f) + dg[u][i];
                            block_acc[p.cols + c] = (w ? block_acc[p.cols + c] : 0.0f) + db[u][i];
                        }
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < 2 * p.cols; c += kWarpRowThreads) out[c] = block_acc[c];
    }
}

// Rows too long for a block's registers: x and dy are read twice, and the
// block's partial sums live in its own row of the workspace, each column
// touched by one thread only.
template <int W>
__global__ void __launch_bounds__(1024) layer_norm_grad_long_kernel(const NormGradParams p) {
    __shared__ float2 buf[2][32];
    RowSum<false> row_sum{buf};
    const int step = blockDim.x * W;
    const float inv = 1.0f / static_cast<float>(p.cols);
    float* acc = p.partial ? p.partial + static_cast<long long>(blockIdx.x) * 2 * p.cols : nullptr;
    bool first = true;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
        const float* x = p.x + row * p.ldx;
        const float* dy = p.dy + row * p.lddy;
        float xh[W], d[W], g[W];
        float2 s = make_float2(0.0f, 0.0f);
        for (long long cc = threadIdx.x * W; cc < p.cols; cc += step) {
            const int c = static_cast<int>(cc);
            load_unit<W>(xh, x, c, p.cols);
            load_unit<W>(d, dy, c, p.cols);
            load_param<W>(g, p.gamma, c, p.cols, 1.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                xh[i] = (xh[i] - mean) * rstd;
                if (acc && c + i < p.cols) {
                    acc[c + i] = (first ? 0.0f : acc[c + i]) + d[i] * xh[i];
                    acc[p.cols + c + i] = (first ? 0.0f : acc[p.cols + c + i]) + d[i];
                }
                s.x += d[i] * g[i];
                s.y += d[i] * g[i] * xh[i];
            }
        }
        first = false;
        if (!p.dx) continue;
        s = row_sum(s);
        const float m1 = s.x * inv, m2 = s.y * inv;
        float* dx = p.dx + row * p.lddx;
        for (long long cc = threadIdx.x * W; cc < p.cols; cc += step) {
            const int c = static_cast<int>(cc);
            load_unit<W>(xh, x, c, p.cols);
            load_unit<W>(d, dy, c, p.cols);
            load_param<W>(g, p.gamma, c, p.cols, 1.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                xh[i] = (xh[i] - mean) * rstd;
                d[i] = rstd * (d[i] * g[i] - m1 - xh[i] * m2);
            }
            store_unit<W>(d, dx, c, p.cols);
        }
    }
}

// dgamma[c] (blockIdx.y 0) or dbeta[c] (1): the blocks' partial rows, summed
// by 32 threads per column and then in thread order.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* partial, int blocks, int cols, float* dgamma,
                                                            float* dbeta) {
    __shared__ float part[32][33];
    float* out = blockIdx.y ? dbeta : dgamma;
    if (!out) return;
    const int c = blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (c < cols) {
        const float* src = partial + static_cast<long long>(blockIdx.y) * cols + c;
        for (int b = threadIdx.y; b < blocks; b += 32) s += src[static_cast<long long>(b) * 2 * cols];
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = warp_sum(make_float2(part[threadIdx.x][threadIdx.y], 0.0f)).x;
    const int cc = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && cc < cols) out[cc] = s;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a row is spread: `threads` threads (32: a warp, eight rows to a block)
// holding `units` units each; units == 0: the kernel for long rows.
struct RowPlan {
    int threads, units;
    bool warp;
};

// max_floats: what a thread may hold of one row; max_threads: of one block.
RowPlan plan_row(int cols, int width, long long rows, int num_sms, int max_floats, int max_threads) {
    const int total = (cols + width - 1) / width, max_units = max_floats / width;
    auto pow2 = [](int n) {
        int p = 1;
        while (p < n) p *= 2;
        return p;
    };
    // Few rows leave most SMs without one: the widest block shortens each thread's share of a row.
    const bool few = rows <= 2ll * num_sms;
    if (total <= 32 || (!few && total <= 32 * max_units)) return {32, pow2((total + 31) / 32), true};
    int threads = few ? max_threads : std::min(256, max_threads);
    while (threads < max_threads && total > threads * max_units) threads *= 2;
    while (few && threads / 2 >= total) threads /= 2;
    if (total > threads * max_units) return {max_threads, 0, false};
    return {threads, pow2((total + threads - 1) / threads), false};
}

template <typename Kernel>
int resident_blocks(Kernel kernel, int threads, size_t smem, int num_sms) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess || n < 1) {
        cudaGetLastError();
        n = 1;
    }
    return n * num_sms;
}

template <int W, int NV, bool WARP>
cudaError_t launch_norm(const NormParams& p, const RowPlan& plan, int num_sms, cudaStream_t stream) {
    const int threads = WARP ? kWarpRowThreads : plan.threads;
    const long long want = WARP ? (p.rows + kWarpRowThreads / 32 - 1) / (kWarpRowThreads / 32) : p.rows;
    const int blocks = static_cast<int>(
        std::min<long long>(want, resident_blocks(layer_norm_kernel<W, NV, WARP>, threads, 0, num_sms)));
    layer_norm_kernel<W, NV, WARP><<<blocks, threads, 0, stream>>>(p);
    note_launch();
    return cudaGetLastError();
}

template <int W, bool WARP>
cudaError_t launch_norm_units(const NormParams& p, const RowPlan& plan, int num_sms, cudaStream_t stream) {
    switch (plan.units) {
        case 1: return launch_norm<W, 1, WARP>(p, plan, num_sms, stream);
        case 2: return launch_norm<W, 2, WARP>(p, plan, num_sms, stream);
        case 4: return launch_norm<W, 4, WARP>(p, plan, num_sms, stream);
        case 8: return launch_norm<W, 8, WARP>(p, plan, num_sms, stream);
        case 16: return launch_norm<W, W == 1 ? 16 : 8, WARP>(p, plan, num_sms, stream);
        case 32: return launch_norm<W, W == 1 ? 32 : 8, WARP>(p, plan, num_sms, stream);
        default: return cudaErrorInvalidValue;
    }
}

constexpr int kNormFloats = 32;      // of a row per thread: 1024 columns per warp, 32768 per block
constexpr int kNormGradFloats = 16;  // x, dy and two sums for each: 512 columns per warp, 8192 per block

template <int W>
cudaError_t launch_norm_width(const NormParams& p, int num_sms, cudaStream_t stream) {
    const RowPlan plan = plan_row(p.cols, W, p.rows, num_sms, kNormFloats, 1024);
    if (plan.units == 0) {
        const int blocks = static_cast<int>(
            std::min<long long>(p.rows, resident_blocks(layer_norm_long_kernel<W>, plan.threads, 0, num_sms)));
        layer_norm_long_kernel<W><<<blocks, plan.threads, 0, stream>>>(p);
        note_launch();
        return cudaGetLastError();
    }
    return plan.warp ? launch_norm_units<W, true>(p, plan, num_sms, stream)
                     : launch_norm_units<W, false>(p, plan, num_sms, stream);
}

// One launch of the backward kernel, or (p == nullptr) the number of blocks it takes.
template <int W, int NV, bool WARP>
cudaError_t launch_norm_grad(const NormGradParams* p, const RowPlan& plan, long long rows, int cols, int num_sms,
                             int* blocks, cudaStream_t stream) {
    const int threads = WARP ? kWarpRowThreads : plan.threads;
    const size_t smem = WARP ? 2 * sizeof(float) * cols : 0;
    if (!p) {
        const long long want = WARP ? (rows + kWarpRowThreads / 32 - 1) / (kWarpRowThreads / 32) : rows;
        *blocks = static_cast<int>(
            std::min<long long>(want, resident_blocks(layer_norm_grad_kernel<W, NV, WARP>, threads, smem, num_sms)));
        return cudaSuccess;
    }
    layer_norm_grad_kernel<W, NV, WARP><<<*blocks, threads, smem, stream>>>(*p);
    note_launch();
    return cudaGetLastError();
}

template <int W, bool WARP>
cudaError_t launch_norm_grad_units(const NormGradParams* p, const RowPlan& plan, long long rows, int cols, int num_sms,
                                   int* blocks, cudaStream_t stream) {
    switch (plan.units) {
        case 1: return launch_norm_grad<W, 1, WARP>(p, plan, rows, cols, num_sms, blocks, stream);
        case 2: return launch_norm_grad<W, 2, WARP>(p, plan, rows, cols, num_sms, blocks, stream);
        case 4: return launch_norm_grad<W, 4, WARP>(p, plan, rows, cols, num_sms, blocks, stream);
        case 8: return launch_norm_grad<W, W == 1 ? 8 : 4, WARP>(p, plan, rows, cols, num_sms, blocks, stream);
        case 16: return launch_norm_grad<W, W == 1 ? 16 : 4, WARP>(p, plan, rows, cols, num_sms, blocks, stream);
        default: return cudaErrorInvalidValue;
    }
}

template <int W>
cudaError_t launch_norm_grad_width(const NormGradParams* p, long long rows, int cols, int num_sms, int* blocks,
                                   cudaStream_t stream) {
    const RowPlan plan = plan_row(cols, W, rows, num_sms, kNormGradFloats, 512);
    if (plan.units == 0) {
        if (!p) {
            *blocks = static_cast<int>(
                std::min<long long>(rows, resident_blocks(layer_norm_grad_long_kernel<W>, plan.threads, 0, num_sms)));
            return cudaSuccess;
        }
        layer_norm_grad_long_kernel<W><<<*blocks, plan.threads, 0, stream>>>(*p);
        note_launch();
        return cudaGetLastError();
    }
    return plan.warp ? launch_norm_grad_units<W, true>(p, plan, rows, cols, num_sms, blocks, stream)
                     : launch_norm_grad_units<W, false>(p, plan, rows, cols, num_sms, blocks, stream);
}

int layer_norm(GpuCtx* ctx, const NormParams& p, void* stream) {
    if (!ctx || p.rows < 0 || p.cols < 1 || p.ldx < p.cols || p.ldy < p.cols || (p.rows > 0 && (!p.x || !p.y))) {
        set_error("mxb_layer_norm: invalid arguments");
        return MXB_E_ARG;
    }
    if (p.x == p.y && p.ldx != p.ldy) {
        set_error("mxb_layer_norm: in place, x and y need the same pitch");
        return MXB_E_ARG;
    }
    if (p.rows == 0) return MXB_OK;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    const bool vec = aligned16(p.x) && aligned16(p.y) && aligned16(p.gamma) && aligned16(p.beta) && p.ldx % 4 == 0 &&
                     p.ldy % 4 == 0;
    const cudaError_t e = vec ? launch_norm_width<4>(p, ctx->num_sms, st) : launch_norm_width<1>(p, ctx->num_sms, st);
    return cuda_ok(e, "layer norm launch") ? MXB_OK : MXB_E_CUDA;
}

int layer_norm_backward(GpuCtx* ctx, NormGradParams p, float* dgamma, float* dbeta, void* stream) {
    if (!ctx || p.rows < 0 || p.cols < 1 || p.lddy < p.cols || p.ldx < p.cols || (p.dx && p.lddx < p.cols) ||
        (!p.dx && !dgamma && !dbeta) || (p.rows > 0 && (!p.dy || !p.x || !p.mean || !p.rstd))) {
        set_error("mxb_layer_norm_backward: invalid arguments");
        return MXB_E_ARG;
    }
    if ((p.dx == p.dy && p.lddx != p.lddy) || (p.dx == p.x && p.lddx != p.ldx)) {
        if (p.dx) {
            set_error("mxb_layer_norm_backward: in place, dx needs the pitch of the matrix that it replaces");
            return MXB_E_ARG;
        }
    }
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    if (p.rows == 0) {
        for (float* z : {dgamma, dbeta})
            if (z && !cuda_ok(cudaMemsetAsync(z, 0, sizeof(float) * p.cols, st), "layer norm gradient clear"))
                return MXB_E_CUDA;
        return MXB_OK;
    }
    const bool vec = aligned16(p.x) && aligned16(p.dy) && aligned16(p.dx) && aligned16(p.gamma) && p.ldx % 4 == 0 &&
                     p.lddy % 4 == 0 && (!p.dx || p.lddx % 4 == 0);
    auto run = [&](const NormGradParams* q, int* blocks) {
        return vec ? launch_norm_grad_width<4>(q, p.rows, p.cols, ctx->num_sms, blocks, st)
                   : launch_norm_grad_width<1>(q, p.rows, p.cols, ctx->num_sms, blocks, st);
    };
    int blocks = 0;
    if (!cuda_ok(run(nullptr, &blocks), "layer norm backward plan")) return MXB_E_CUDA;
    Scratch scratch(ctx, st);
    if (dgamma || dbeta) {
        p.partial = static_cast<float*>(scratch.alloc(sizeof(float) * 2 * p.cols * static_cast<size_t>(blocks)));
        if (!p.partial) return MXB_E_NOMEM;
    }
    if (!cuda_ok(run(&p, &blocks), "layer norm backward launch")) return MXB_E_CUDA;
    if (!p.partial) return MXB_OK;
    sum_partials_kernel<<<dim3((p.cols + 31) / 32, 2), dim3(32, 32), 0, st>>>(p.partial, blocks, p.cols, dgamma, dbeta);
    note_launch();
    return cuda_ok(cudaGetLastError(), "layer norm gradient sums launch") ? MXB_OK : MXB_E_CUDA;
}

}  // namespace
}  // namespace mxb

extern "C" {

int mxb_layer_norm(GpuCtx* ctx, const float* x, long long ldx, const float* gamma, const float* beta, float eps,
                   float* y, long long ldy, float* mean, float* rstd, long long rows, int cols, void* stream) {
    return mxb::layer_norm(ctx, mxb::NormParams{x, ldx, gamma, beta, eps, y, ldy, mean, rstd, rows, cols}, stream);
}

int mxb_layer_norm_backward(GpuCtx* ctx, const float* dy, long long lddy, const float* x, long long ldx,
                            const float* gamma, const float* mean, const float* rstd, float* dx, long long lddx,
                            float* dgamma, float* dbeta, long long rows, int cols, void* stream) {
    try {
        return mxb::layer_norm_backward(
            ctx, mxb::NormGradParams{dy, lddy, x, ldx, gamma, mean, rstd, dx, lddx, nullptr, rows, cols}, dgamma,
            dbeta, stream);
    } catch (const std::exception& e) {  // host allocations of the pool's lists
        mxb::set_error("mxb_layer_norm_backward: %s", e.what());
        return MXB_E_NOMEM;
    }
}

}  // extern "C"
