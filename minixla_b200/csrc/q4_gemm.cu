// Products with 4-bit weights and group scales (mxb_q4_gemm):
//   out[m, n] = epi(sum over groups g of s[n, g] * sum over k in g of A[m, k] * (q[n, k] - z[n, g])).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <exception>
#include <mutex>

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

// ---------------------------------------------------------------- few rows
//
// Up to 16 rows: bound by the weights' bytes.  One mma.sync.m16n8k16 (bf16,
// fp32 accumulate) takes 16 weight columns as its rows and activations as
// its eight columns.  q - z is exact in bf16; an activation is cut into three
// bf16 parts of eight bits each whose sum is exact, so nothing is rounded
// before the fp32 sums.  A warp takes every eighth run of 128 k for
// 16 * MT weight columns; lane (g, t) of the warp holds, for each 32 k, the
// eight values of word t of weight rows g and g + 8 -- the k order inside an
// MMA is free as long as weights and activations agree on it, so the words
// are used as they lie -- and the same eight k of activation row g, which it
// cuts itself.  All 16 k of an MMA lie in one group; the sums of a group (of
// the whole run, where the group is a multiple of 128) start from zero and
// are scaled in fp32.
//  PACK: one or two rows; the eight MMA columns hold the parts side by side
//        (column 3 m + part), one MMA instead of three.
//  RT:   row tiles of eight; their three parts go through three MMAs into
//        the same accumulators.
// Weights and activations come through a ring of cp.async units per warp.

constexpr int kFewWarps = 8;
constexpr int kRun = 128;  // k of one unit

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two q - z as a bf16 pair, from nibbles 0 and 4 of `w` and the pair (128 + z, 128 + z):
// 0x4300 | q is the bf16 number 128 + q, and the difference is exact.
__device__ __forceinline__ uint32_t weight_pair(uint32_t w, __nv_bfloat162 z128) {
    uint32_t v = (w & 0x000F000Fu) | 0x43004300u;
    __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), z128);
    return *reinterpret_cast<uint32_t*>(&h);
}

// The top eight bits of x and y as a bf16 pair; x and y keep the rest.
__device__ __forceinline__ uint32_t cut_pair(float& x, float& y) {
    const uint32_t ux = __float_as_uint(x), uy = __float_as_uint(y);
    x -= __uint_as_float(ux & 0xFFFF0000u);
    y -= __uint_as_float(uy & 0xFFFF0000u);
    return __byte_perm(ux, uy, 0x7632);
}

template <bool PACK, int RT, int MT>
struct FewCfg {
    static constexpr int kRows = PACK ? 2 : 8 * RT;
    static constexpr int kUnit = MT * 1024 + kRows * kRun * 4;
    static constexpr int kDepth = kUnit * kFewWarps * 4 <= 100 * 1024 ? 4 : kUnit * kFewWarps * 3 <= 110 * 1024 ? 3 : 2;
    static constexpr int kRing = kUnit * kFewWarps * kDepth;
    static constexpr int kReduce = kFewWarps * 16 * MT * (8 * RT) * 4;
    static constexpr int kSmem = kRing > kReduce ? kRing : kReduce;
};

template <bool PACK, int RT, int MT>
__global__ void __launch_bounds__(32 * kFewWarps)
    q4_few_rows_kernel(const __grid_constant__ Q4Params p) {
    using C = FewCfg<PACK, RT, MT>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16 * MT, m0 = blockIdx.y * C::kRows;
    const int rows = min(C::kRows, p.M - m0);
    const int runs = (p.K + kRun - 1) / kRun;
    uint8_t* ring = smem + warp * C::kDepth * C::kUnit;

    // Unit of run r into slot `slot`.  Weights: row i at 64 i, its 16-byte
    // chunk s (32 k) at position s ^ ((i >> 1) & 3); activations: row m at
    // 512 m, chunk c at c ^ (m & 1): both conflict-free for the reads below.
    auto issue = [&](int r, int slot) {
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring + slot * C::kUnit));
        const int k0 = r * kRun;
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) {
            const int i = j * 8 + g;
            const bool in = n0 + i < p.N && k0 / 2 + 16 * t < p.ldq;
            cp_async16(dst + i * 64 + ((t ^ ((i >> 1) & 3)) << 4),
                       in ? p.q + (n0 + i) * p.ldq + k0 / 2 + 16 * t : p.q, in ? 16 : 0);
        }
        for (int m = 0; m < rows; ++m) {
            const int left = min(max(p.K - k0 - 4 * lane, 0), 4);
            cp_async16(dst + MT * 1024 + m * 512 + ((lane ^ (m & 1)) << 4),
                       left ? p.a + (m0 + m) * p.lda + k0 + 4 * lane : p.a, 4 * left);
        }
    };
    const bool whole = p.group % kRun == 0;  // one group to a run
    // Lane t keeps the scale and zero point of 32-value piece t of a run (of the whole run), for its 2 MT weight rows.
    auto load_group = [&](int r, float (&s)[2 * MT], uint32_t (&z)[2 * MT]) {
        const int k = r * kRun + (whole ? 0 : 32 * t);
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) {
            const int n = n0 + j * 8 + g;
            const bool in = n < p.N && k < p.K;
            const long long at = n * p.lds + k / p.group;
            s[j] = in ? load_scale(p, at) : 0.0f;
            z[j] = in && p.zeros ? __ldg(p.zeros + at) & 15u : 8u;
        }
    };

    // This lane's activation row (PACK: row and part) of the MMA's column g.
    const int part = PACK ? g % 3 : 0;
    float tot[MT][RT][4] = {};
    float s_next[2 * MT];
    uint32_t z_next[2 * MT];
    int r = warp;
    if (r < runs) load_group(r, s_next, z_next);
#pragma unroll
    for (int d = 0; d < C::kDepth - 1; ++d) {
        if (r + d * kFewWarps < runs) issue(r + d * kFewWarps, d);
        cp_async_commit();
    }
    for (int slot = 0; r < runs; r += kFewWarps) {
        float s[2 * MT];
        uint32_t z[2 * MT];
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) {
            s[j] = s_next[j];
            z[j] = z_next[j];
        }
        if (r + kFewWarps < runs) load_group(r + kFewWarps, s_next, z_next);
        cp_async_wait<C::kDepth - 2>();
        __syncwarp();  // the unit is here for every lane, and the one before it is read by all
        const int ahead = r + (C::kDepth - 1) * kFewWarps;
        if (ahead < runs) issue(ahead, slot == 0 ? C::kDepth - 1 : slot - 1);
        cp_async_commit();
        const uint8_t* unit = ring + slot * C::kUnit;
        float acc[MT][RT][4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            // Parts of this lane's eight activations: pairs (k, k + 4) as the nibbles of a word pair up.
            uint32_t b[RT][PACK ? 1 : 3][4];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int m = PACK ? (g < 6 ? g / 3 : 0) : rt * 8 + g;
                const float4* x = reinterpret_cast<const float4*>(unit + MT * 1024 + m * 512);
                float4 lo = x[(c * 8 + 2 * t) ^ (m & 1)], hi = x[(c * 8 + 2 * t + 1) ^ (m & 1)];
                float u[4] = {lo.x, lo.y, lo.z, lo.w}, v[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t p0 = cut_pair(u[i], v[i]), p1 = cut_pair(u[i], v[i]);
                    const uint32_t p2 = __byte_perm(__float_as_uint(u[i]), __float_as_uint(v[i]), 0x7632);
                    if (PACK) {
                        b[rt][0][i] = part == 0 ? p0 : part == 1 ? p1 : p2;
                    } else {
                        b[rt][0][i] = p2;  // small parts first
                        b[rt][PACK ? 0 : 1][i] = p1;
                        b[rt][PACK ? 0 : 2][i] = p0;
                    }
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                uint32_t w[2], zz[2];
                float sc[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = mt * 16 + h * 8 + g, j = 2 * mt + h;
                    w[h] = *reinterpret_cast<const uint32_t*>(unit + i * 64 + ((c ^ ((i >> 1) & 3)) << 4) + 4 * t);
                    zz[h] = __shfl_sync(0xffffffffu, z[j], (lane & ~3) | c);
                    sc[h] = __shfl_sync(0xffffffffu, s[j], (lane & ~3) | c);
                }
                __nv_bfloat162 z128[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t pair = 0x43004300u | zz[h] | (zz[h] << 16);
                    z128[h] = *reinterpret_cast<const __nv_bfloat162*>(&pair);
                }
                const uint32_t a1[4] = {weight_pair(w[0], z128[0]), weight_pair(w[1], z128[1]),
                                        weight_pair(w[0] >> 4, z128[0]), weight_pair(w[1] >> 4, z128[1])};
                const uint32_t a2[4] = {weight_pair(w[0] >> 8, z128[0]), weight_pair(w[1] >> 8, z128[1]),
                                        weight_pair(w[0] >> 12, z128[0]), weight_pair(w[1] >> 12, z128[1])};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int q = 0; q < (PACK ? 1 : 3); ++q) {
                        mma_bf16(acc[mt][rt], a1, b[rt][q][0], b[rt][q][1]);
                        mma_bf16(acc[mt][rt], a2, b[rt][q][2], b[rt][q][3]);
                    }
                    if (!whole || c == 3) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            tot[mt][rt][i] += sc[i >> 1] * acc[mt][rt][i];
                            acc[mt][rt][i] = 0.0f;
                        }
                    }
                }
            }
        }
        if (++slot == C::kDepth) slot = 0;
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with the ring
    // The warps' sums: [warp][MMA column][weight column], added in warp order (PACK: small parts first).
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                red[(warp * 8 * RT + rt * 8 + 2 * t + (i & 1)) * 16 * MT + mt * 16 + (i >> 1) * 8 + g] = tot[mt][rt][i];
    __syncthreads();
    for (int i = threadIdx.x; i < rows * 16 * MT; i += 32 * kFewWarps) {
        const int m = i / (16 * MT), n = i % (16 * MT);
        if (n0 + n >= p.N) continue;
        float v = 0.0f;
#pragma unroll
        for (int q = PACK ? 2 : 0; q >= 0; --q)
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w)
                v += red[(w * 8 * RT + (PACK ? 3 * m + q : m)) * 16 * MT + n];
        p.out[(m0 + m) * p.ldo + n0 + n] = apply_cell(v, m0 + m, n0 + n, 0, p.epi);
    }
}

template <bool PACK, int RT, int MT>
cudaError_t run_few_rows(const Q4Params& p, cudaStream_t stream) {
    using C = FewCfg<PACK, RT, MT>;
    auto kernel = q4_few_rows_kernel<PACK, RT, MT>;
    static std::mutex mu;
    static uint64_t configured = 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (dev >= 64 || !(configured & (1ull << dev))) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
            if (e != cudaSuccess) return e;
            if (dev < 64) configured |= 1ull << dev;
        }
    }
    kernel<<<dim3((p.N + 16 * MT - 1) / (16 * MT), (p.M + C::kRows - 1) / C::kRows), 32 * kFewWarps, C::kSmem, stream>>>(p);
    note_launch();
    return cudaGetLastError();
}

template <bool PACK, int RT>
cudaError_t run_few_rows_width(const Q4Params& p, int num_sms, cudaStream_t stream) {
    // Wider warp tiles cut each activation for more weights; narrow ones fill the SMs.
    if (p.N >= 64 * num_sms && !PACK) return run_few_rows<PACK, RT, PACK ? 2 : 4>(p, stream);
    return p.N >= 32 * num_sms ? run_few_rows<PACK, RT, 2>(p, stream) : run_few_rows<PACK, RT, 1>(p, stream);
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
    const cudaError_t e = p.M <= 2   ? run_few_rows_width<true, 1>(p, ctx->num_sms, st)
                          : p.M <= 8 ? run_few_rows_width<false, 1>(p, ctx->num_sms, st)
                                     : run_few_rows_width<false, 2>(p, ctx->num_sms, st);
    return cuda_ok(e, "4-bit product launch") ? MXB_OK : MXB_E_CUDA;
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
