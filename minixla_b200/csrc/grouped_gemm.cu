// Products grouped by expert (mxb_grouped_gemm and its gradients): rows
// offsets[e] .. offsets[e+1] - 1 belong to group e and meet its own matrix.
//   forward  out[r, n]   = epi(sum over k of A[r, k] * B_e[k, n])
//   grad_a   dA[r, k]    = epi(sum over n of dY[r, n] * B_e[k, n])
//   grad_b   dB_e[k, n]  = sum over the group's rows r of A[r, k] * dY[r, n],  dbias[e, n] = sum over r of dY[r, n]
//
// Three tcgen05 kernels: pairs of CTAs with tiles of 256 x 256 where groups
// have many rows (all three products), a CTA with at most 64 rows to a tile
// where they have few (forward, grad_a), and a CTA with 128 x 128 for grad_b's
// small matrices.  plan_grouped has the rule.  The tile is turned around
// compared with the dense GEMMs: the dimension along which the result is contiguous
// (n, or k in grad_a) lies along the tensor core's 128 rows and TMEM lanes,
// the ragged dimension (the group's rows; k in grad_b) along its columns.
// A group with few rows then costs an MMA of 16 columns instead of 128 rows,
// the column count follows each tile's own rows at run time, and a warp
// stores 32 consecutive floats of one output row at a time whatever the
// pitch.  A lane-side tile of the weights is read where it lies: MN-major
// (forward, grad_b) or K-major (grad_a), by the MMA descriptor alone.
//
// Which tile belongs to which group is found on the device from `offsets`
// (a scan at the start of the kernel, a search per tile), so nothing is read
// back to the host and a captured call follows the offsets of each replay.
//
// 3xTF32: x = big + small, three TF32 products.  The tensor core itself cuts
// an fp32 operand to its upper 19 bits, so the tile that TMA loaded serves as
// big, and converter warps write small = x - big (rounded to the nearest TF32)
// to a second tile or to tensor memory: no pass over the weights beforehand, which would cost two to
// three times the bytes of the product where a group has few rows.  K is
// summed in segments of 64 or 128, each in a fresh accumulator, because the
// tensor core cuts its running sums toward zero; the epilogue warps add the
// segments in fp32 registers.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <exception>

#include "gemm_common.cuh"

#include "epilogue_cell.cuh"
#include "runtime_internal.h"

namespace mxb {

namespace {

enum GroupedMode : int { kForward = MXB_GROUPED_FORWARD, kGradA = MXB_GROUPED_GRAD_A, kGradB = MXB_GROUPED_GRAD_B };

struct GroupedCall {
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
};

struct GroupedParams {
    const int* offsets;
    int groups, rows;
    float* out;
    long long ldo, out_stride;  // out_stride: grad_b, between groups
    int lane_dim;               // columns of the result: N, or K in grad_a
    int col_dim;                // grad_b: K (else each group's rows)
    int sum_dim;                // forward: K, grad_a: N (grad_b: each group's rows)
    int lane_tiles;
    int split3;                 // 3xTF32
    float* dbias;               // grad_b, 3xTF32 CTA pairs: column sums of dY, [groups][lane_dim] (or nullptr)
    unsigned long long timeout_ns;
    int* err;
    CellEpilogue epi;
};

constexpr int kGroupedTableBytes = 20 * MXB_MAX_GROUPS + 128 * 4 + 16;

struct GroupedGradBCfg {
    static constexpr int kCols = 128;                 // columns of A that a tile takes
    static constexpr int kLaneBytes = 128 * kBK * 4;
    static constexpr int kColBytes = kCols * kBK * 4;
    static constexpr int kStageBytes = kLaneBytes + kColBytes;
    static constexpr int kStages = 4;                 // tiles as loaded
    static constexpr int kSmall = 2;                  // their small parts
    static constexpr int kEpiWarps = 8;
    static constexpr int kConvWarps = 8;
    static constexpr int kThreads = 32 * (kEpiWarps + kConvWarps + 4);  // and a warpgroup with TMA and MMA
    // Registers a thread: the launch has 640 x 96, given out in shares of 128 threads.
    static constexpr int kEpiRegs = 144, kConvRegs = 64, kIssueRegs = 64;
    static_assert(2 * kEpiRegs + 2 * kConvRegs + kIssueRegs <= 480, "more registers than the launch has");
    static constexpr int kTmemCols = 2 * kCols;          // two segment buffers
    static constexpr int kTotals = kCols * 4 / kEpiWarps;  // columns of one epilogue thread
    static constexpr int kSmallOffset = kStages * kStageBytes;
    static constexpr int kTableOffset = kSmallOffset + kSmall * kStageBytes;
    static constexpr int kBarOffset = kTableOffset + kGroupedTableBytes;
    static constexpr int kNumBars = 2 * kStages + 2 * kSmall + 4 + 1;
    static constexpr int kSmemBytes = 1024 + kBarOffset + kNumBars * 8 + 16;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
    static_assert(kTmemCols >= 32 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM columns come in powers of two");
};

// kind::tf32 with fp32 accumulation, operand majorness as given (1: MN-major).
__host__ __device__ constexpr uint32_t idesc_tf32_major(int m, int n, int a_mn, int b_mn) {
    return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(a_mn) << 15) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// The part of x below the upper 19 bits that the tensor core reads, rounded
// to the nearest TF32 (adding half a step; the tensor core cuts the rest).
// Non-finite x has none.
__device__ __forceinline__ float small_of(float x) {
    const float s = x - __uint_as_float(__float_as_uint(x) & 0xFFFFE000u);
    return s == s ? __uint_as_float(__float_as_uint(s) + 0x1000u) : 0.0f;
}

// The small parts of a staged k-block of n4 float4s (lane side, then column
// boxes), thread t0 of THREADS; the layout does not matter, both tiles have the
// same.  grad_b: of the 32 rows of every box (128 bytes each) only the first
// `valid` belong to the group; the others may hold anything and become zeros.
template <int MODE, int THREADS>
__device__ __forceinline__ void convert_tile(uint8_t* big, uint8_t* low, int t0, int n4, int valid, int split3) {
    float4* src = reinterpret_cast<float4*>(big);
    float4* dst = reinterpret_cast<float4*>(low);
    if (MODE == kGradB && valid < kBK) {
        for (int i = t0; i < n4; i += THREADS)
            if (((i >> 3) & 31) >= valid) src[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (!split3) return;
    // n4 is a multiple of THREADS (256).
#pragma unroll 4
    for (int i = t0; i < n4; i += THREADS) {
        const float4 v = src[i];
        dst[i] = make_float4(small_of(v.x), small_of(v.y), small_of(v.z), small_of(v.w));
    }
}

// grad_b's bias gradient, on the way: adds this k-block's rows of the staged lane side to the thread's 16 columns (four
// of each box).  Thread t0 of 256 has row t0 / 8 and 16-byte chunk t0 % 8 of every box; which columns those are
// depends on the row (32-byte chunks are swizzled by row % 4), but not on the k-block.
__device__ __forceinline__ void add_lane_columns(const uint8_t* staged, int t0, float (&sum)[16]) {
#pragma unroll
    for (int box = 0; box < 4; ++box) {
        const float4 v = reinterpret_cast<const float4*>(staged)[box * 256 + t0];
        sum[4 * box] += v.x;
        sum[4 * box + 1] += v.y;
        sum[4 * box + 2] += v.z;
        sum[4 * box + 3] += v.w;
    }
}
__device__ __forceinline__ void add_lane_columns(const uint8_t*, int, float (&)[1]) {}

// The warp's four rows of those sums added up, by column: dst[0 .. 127].
__device__ __forceinline__ void leave_lane_sums(const float (&sum)[16], float* dst, int lane) {
    const int block = (lane & 7) >> 1 ^ (lane >> 3), low = lane & 1;  // of this lane's columns within a box: 8 block + 4 low
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) v += __shfl_sync(0xffffffffu, sum[e], q * 8 + ((block ^ q) << 1 | low));
        if (lane < 8) dst[(e >> 2) * 32 + block * 8 + low * 4 + (e & 3)] = v;
    }
}
__device__ __forceinline__ void leave_lane_sums(const float (&)[1], float*, int) {}

// One tile of work.
struct GroupedTile {
    int group;
    int lane0;    // first result column
    int col0;     // first row of the group (grad_b: of dB) in this tile
    int cols;     // how many
    int row0;     // the group's first row
    int sum;      // length of the sum
};

// Which tile is which, written by each CTA from `offsets` at its start (every
// CTA the same: the order below depends on nothing else).  A group's column
// tiles are two entries, the whole tiles and the narrower last one; the entries
// are ordered by the cost of a tile, dearest first, in quarter octaves.  The
// CTAs (pairs) take tiles by their index, every other round backwards, so that
// the cheap tiles at the end even out what the dear ones left.
struct GroupedTable {
    int first_tile[2 * MXB_MAX_GROUPS];             // of each entry: the tiles before it
    unsigned short entry[2 * MXB_MAX_GROUPS];       // group * 2 + (0: whole tiles, 1: the last one)
    int row0[MXB_MAX_GROUPS], row1[MXB_MAX_GROUPS];
    int classes[128];
    int entries, total;
};
static_assert(sizeof(GroupedTable) <= kGroupedTableBytes && kGroupedTableBytes % 16 == 0, "table size");

// Tile t: inside an entry the column tiles vary fastest, so CTAs that run together share weights through L2.
template <int MODE, int BT, int LANES = 128>
__device__ __forceinline__ GroupedTile grouped_tile(const GroupedTable& tab, int t, const GroupedParams& p) {
    int lo = 0, hi = tab.entries - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tab.first_tile[mid] <= t) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    GroupedTile g;
    const int last = tab.entry[lo] & 1;
    g.group = tab.entry[lo] >> 1;
    g.row0 = tab.row0[g.group];
    const int rows = tab.row1[g.group] - g.row0;
    const int dim = MODE == kGradB ? p.col_dim : rows;
    const int i = t - tab.first_tile[lo], whole = dim / BT, col_tiles = last ? 1 : whole;
    g.lane0 = i / col_tiles * LANES;
    g.col0 = (last ? whole : i % col_tiles) * BT;
    g.cols = last ? dim - g.col0 : BT;
    g.sum = MODE == kGradB ? rows : p.sum_dim;
    return g;
}

// Tile of worker `me` of `n` in round `round`, or -1; -2 once no worker has one.
__device__ __forceinline__ int grouped_turn(int round, int me, int n, int total) {
    const long long first = static_cast<long long>(round) * n;
    if (first >= total) return -2;
    const long long t = first + (round & 1 ? n - 1 - me : me);
    return t < total ? static_cast<int>(t) : -1;
}

// Fills the table (one warp): group e's rows are clamped to 0 <= row0 <= row1 <= rows.
template <int MODE, int BT>
__device__ __forceinline__ void grouped_scan(GroupedTable& tab, const GroupedParams& p, int lane) {
    for (int c = lane; c < 128; c += 32) tab.classes[c] = 0;
    __syncwarp();
    // Entry i = 2 e + part: how many column tiles it has, and its class (127 - 4 log2(cost) or so; -1: no tile).
    auto look = [&](int i, int& tiles) -> int {
        tiles = 0;
        const int e = i >> 1;
        if (e >= p.groups) return -1;
        const int r0 = min(max(ld_global(p.offsets + e), 0), p.rows);
        const int r1 = min(max(ld_global(p.offsets + e + 1), r0), p.rows);
        if ((i & 1) == 0) {
            tab.row0[e] = r0;
            tab.row1[e] = r1;
        }
        const int dim = MODE == kGradB ? p.col_dim : r1 - r0;
        const int cols = i & 1 ? dim % BT : BT;
        tiles = i & 1 ? (cols ? 1 : 0) : dim / BT;
        if (!tiles) return -1;
        const unsigned cost = static_cast<unsigned>((cols + 15) / 16) *
                              static_cast<unsigned>(MODE == kGradB ? (r1 - r0) / kBK + 1 : 1);
        const int octave = 31 - __clz(cost);
        return 127 - (octave * 4 + static_cast<int>(octave >= 2 ? (cost >> (octave - 2)) & 3 : (cost << (2 - octave)) & 3));
    };
    const int n = 2 * p.groups;
    for (int i0 = 0; i0 < n; i0 += 32) {
        int tiles;
        const int c = look(i0 + lane, tiles);
        const unsigned same = __match_any_sync(0xffffffffu, c);
        if (c >= 0 && lane == __ffs(same) - 1) tab.classes[c] += __popc(same);
        __syncwarp();
    }
    // Classes' first places, by an exclusive scan of four counts a lane.
    int count[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        count[j] = sum;
        sum += tab.classes[4 * lane + j];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) tab.classes[4 * lane + j] = upto - sum + count[j];
    const int entries = __shfl_sync(0xffffffffu, upto, 31);
    __syncwarp();
    for (int i0 = 0; i0 < n; i0 += 32) {
        int tiles;
        const int c = look(i0 + lane, tiles);
        const unsigned same = __match_any_sync(0xffffffffu, c);
        const int place = c >= 0 ? tab.classes[c] + __popc(same & ((1u << lane) - 1)) : 0;
        __syncwarp();
        if (c >= 0) {
            tab.entry[place] = static_cast<unsigned short>(i0 + lane);
            tab.first_tile[place] = tiles * p.lane_tiles;
            if (lane == __ffs(same) - 1) tab.classes[c] += __popc(same);
        }
        __syncwarp();
    }
    // Sums end at 2^31 - 1 (an entry's own tiles are below 2^25, since the result has to be in memory): only groups that
    // decreasing offsets make overlap can have more tiles together, and those beyond are left out.
    auto add = [](unsigned a, unsigned b) { return min(a + b, 0x7FFFFFFFu); };
    unsigned base = 0;
    for (int i0 = 0; i0 < entries; i0 += 32) {
        unsigned upto_here = i0 + lane < entries ? tab.first_tile[i0 + lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned v = __shfl_up_sync(0xffffffffu, upto_here, o);
            if (lane >= o) upto_here = add(upto_here, v);
        }
        const unsigned before = __shfl_up_sync(0xffffffffu, upto_here, 1);
        if (i0 + lane < entries) tab.first_tile[i0 + lane] = static_cast<int>(lane ? add(base, before) : base);
        base = add(base, __shfl_sync(0xffffffffu, upto_here, 31));
    }
    if (lane == 0) {
        tab.entries = entries;
        tab.total = static_cast<int>(base);
    }
}

__device__ __forceinline__ void raise_grouped(const GroupedParams& p, volatile int* abort_flag, int bit) {
    atomicOr(p.err, bit);
    *abort_flag = 1;
}

constexpr int kGroupedSegKb = 2;  // k-blocks (of 32) to an accumulator

// grad_b with K too small for pairs, or too few tiles for all of them: 128 x
// 128 of dB_e to a CTA, or to a cluster that splits the group's rows, both
// operands MN-major as they lie.  Bound by shared memory (120 KB a k-block for
// 3xTF32) where there are many rows.
__global__ void __launch_bounds__(GroupedGradBCfg::kThreads, 1)
    grouped_grad_b_kernel(const __grid_constant__ CUtensorMap tm_lane, const __grid_constant__ CUtensorMap tm_col,
                        const __grid_constant__ GroupedParams p, const int splits) {
    using C = GroupedGradBCfg;
    constexpr int BT = C::kCols;
    extern __shared__ uint8_t smem_raw[];
    // (an offset, not a rounded pointer: the compiler then still knows that these are shared addresses)
    uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    GroupedTable& tab = *reinterpret_cast<GroupedTable*>(smem + C::kTableOffset);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };                         // TMA -> converter (whose arrival passes it on to the MMA)
    auto empty_bar = [&](int s) { return bar0 + 8u * (C::kStages + s); };         // MMA -> TMA
    auto conv_bar = [&](int s) { return bar0 + 8u * (2 * C::kStages + s); };      // converter -> MMA
    auto sfree_bar = [&](int s) { return bar0 + 8u * (2 * C::kStages + C::kSmall + s); };  // MMA -> converter
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + 2 + a); };
    const uint32_t drain_bar = bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kConvWarp = C::kEpiWarps, kTmaWarp = kConvWarp + C::kConvWarps, kMmaWarp = kTmaWarp + 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int s = 0; s < C::kSmall; ++s) {
            mbar_init(conv_bar(s), C::kConvWarps);
            mbar_init(sfree_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), C::kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_lane);
        tma_prefetch_desc(&tm_col);
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_addr(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    wait_for_previous_kernel();
    if (warp == kMmaWarp) let_next_kernel_in();  // behind this CTA's allocation
    if (warp == kConvWarp) grouped_scan<kGradB, BT>(tab, p, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = tab.total;
    const int team = blockIdx.x / splits, teams = gridDim.x / splits, rank = blockIdx.x - team * splits;
    // This CTA's k-blocks [first, second) of a tile's `num_kb`.
    auto my_part = [&](int num_kb, int& first) {
        first = static_cast<int>(static_cast<long long>(num_kb) * rank / splits);
        return static_cast<int>(static_cast<long long>(num_kb) * (rank + 1) / splits);
    };

    if (warp >= kTmaWarp) {
        fewer_registers<C::kIssueRegs>();
        if (warp == kTmaWarp) {
            // ------------------------------------------------------------ TMA producer
            if (lane == 0) {
                int stage = 0;
                uint32_t phase = 0;
                long long issued = 0;
                bool ok = true;
                for (int round = 0; ok; ++round) {
                    const int t = grouped_turn(round, team, teams, total_tiles);
                    if (t == -2) break;
                    if (t < 0) continue;
                    const GroupedTile g = grouped_tile<kGradB, BT>(tab, t, p);
                    const int col_boxes = (g.cols + 31) / 32;
                    int kb0;
                    const int kb1 = my_part((g.sum + kBK - 1) / kBK, kb0);
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (*abort_flag || !mbar_wait(empty_bar(stage), phase ^ 1u, p.timeout_ns)) {
                            raise_grouped(p, abort_flag, kErrProducer);
                            ok = false;
                            break;
                        }
                        const uint32_t st = smem_addr(smem + stage * C::kStageBytes);
                        const uint32_t fb = full_bar(stage);
                        mbar_arrive_expect_tx(fb, C::kLaneBytes + col_boxes * kBoxBytes);
                        const int q0 = kb * kBK;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tma_load_2d(st + j * kBoxBytes, &tm_lane, fb, g.lane0 + 32 * j, g.row0 + q0);
                        for (int j = 0; j < col_boxes; ++j)
                            tma_load_2d(st + C::kLaneBytes + j * kBoxBytes, &tm_col, fb, g.col0 + 32 * j, g.row0 + q0);
                        ++issued;
                        if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                    }
                }
                if (!ok) {
                    // Copies in flight land in this CTA's shared memory: wait for them before leaving.
                    const long long n = issued < C::kStages ? issued : C::kStages;
                    for (long long i = 1; i <= n; ++i) {
                        const long long idx = issued - i;
                        mbar_wait(full_bar(static_cast<int>(idx % C::kStages)),
                                  static_cast<uint32_t>((idx / C::kStages) & 1), p.timeout_ns);
                    }
                }
            }
        } else if (warp == kMmaWarp) {
            // ------------------------------------------------------------ MMA issuer
            constexpr uint32_t kHi = smem_desc_hi(512, kLayoutSW128Base32B), kStep = 64;  // 8 rows of 128 bytes
            const bool leader = elect_one();
            int stage = 0, small = 0, acc = 0;
            uint32_t small_phase = 0, acc_phase = 0;
            bool ok = true;
            for (int round = 0; ok; ++round) {
                const int t = grouped_turn(round, team, teams, total_tiles);
                if (t == -2) break;
                if (t < 0) continue;
                const GroupedTile g = grouped_tile<kGradB, BT>(tab, t, p);
                const uint32_t idesc = idesc_tf32_major(128, (g.cols + 15) & ~15, 1, 1);
                int kb0;
                const int kb1 = my_part((g.sum + kBK - 1) / kBK, kb0);
                int in_seg = 0;
                for (int kb = kb0; kb < kb1; ++kb) {
                    bool ready = *abort_flag == 0;
                    if (ready && in_seg == 0) ready = mbar_wait(tempty_bar(acc), acc_phase ^ 1u, p.timeout_ns);
                    if (!ready || !mbar_wait(conv_bar(small), small_phase, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const bool end_seg = ++in_seg == kGroupedSegKb || kb == kb1 - 1;
                    if (leader) {
                        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BT);
                        const uint32_t big = smem_addr(smem + stage * C::kStageBytes);
                        const uint32_t low = smem_addr(smem + C::kSmallOffset + small * C::kStageBytes);
                        const uint32_t bl = smem_desc_lo(big, kBoxBytes);
                        const uint32_t bc = smem_desc_lo(big + C::kLaneBytes, kBoxBytes);
                        const uint32_t sl = smem_desc_lo(low, kBoxBytes);
                        const uint32_t sc = smem_desc_lo(low + C::kLaneBytes, kBoxBytes);
                        // The last k-block ends with its own eighth: nothing past the sum is multiplied.
                        const int steps = min(4, (g.sum - kb * kBK + 7) / 8);
                        const uint32_t begun = in_seg > 1 ? 1u : 0u;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            if (kk >= steps) break;
                            const uint64_t da = smem_desc_of(kHi, bl + kk * kStep);
                            const uint64_t db = smem_desc_of(kHi, bc + kk * kStep);
                            if (p.split3) {
                                // Small cross terms first, the dominant product last.
                                mma_tf32(d, da, smem_desc_of(kHi, sc + kk * kStep), idesc, kk ? 1u : begun);
                                mma_tf32(d, smem_desc_of(kHi, sl + kk * kStep), db, idesc, 1u);
                                mma_tf32(d, da, db, idesc, 1u);
                            } else {
                                mma_tf32(d, da, db, idesc, kk ? 1u : begun);
                            }
                        }
                        mma_commit(empty_bar(stage));
                        mma_commit(sfree_bar(small));
                        if (end_seg) mma_commit(tfull_bar(acc));
                    }
                    if (++stage == C::kStages) stage = 0;
                    if (++small == C::kSmall) { small = 0; small_phase ^= 1u; }
                    if (end_seg) {
                        in_seg = 0;
                        acc ^= 1;
                        if (acc == 0) acc_phase ^= 1u;
                    }
                }
            }
            if (leader) {
                if (!ok) raise_grouped(p, abort_flag, kErrMma);
                mma_commit(drain_bar);
                if (!mbar_wait(drain_bar, 0, p.timeout_ns)) raise_grouped(p, abort_flag, kErrMma);
            }
            __syncwarp();
        }
    } else if (warp >= kConvWarp) {
        fewer_registers<C::kConvRegs>();
        // ------------------------------------------------------------ converter
        const int t0 = threadIdx.x - 32 * kConvWarp;
        int stage = 0, small = 0;
        uint32_t phase = 0, small_phase = 0;
        bool failed = false;
        for (int round = 0; !failed; ++round) {
            const int t = grouped_turn(round, team, teams, total_tiles);
            if (t == -2) break;
            if (t < 0) continue;
            const GroupedTile g = grouped_tile<kGradB, BT>(tab, t, p);
            const int col_boxes = (g.cols + 31) / 32;
            int kb0;
            const int kb1 = my_part((g.sum + kBK - 1) / kBK, kb0);
            for (int kb = kb0; kb < kb1; ++kb) {
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(full_bar(stage), phase, p.timeout_ns) &&
                                 mbar_wait(sfree_bar(small), small_phase ^ 1u, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_grouped(p, abort_flag, kErrProducer);
                    failed = true;
                    break;
                }
                convert_tile<kGradB, 32 * C::kConvWarps>(smem + stage * C::kStageBytes,
                                                         smem + C::kSmallOffset + small * C::kStageBytes, t0,
                                                         1024 + col_boxes * 256, g.sum - kb * kBK, p.split3);
                fence_proxy_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(conv_bar(small));
                if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                if (++small == C::kSmall) { small = 0; small_phase ^= 1u; }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue
        more_registers<C::kEpiRegs>();
        constexpr int W = 16;
        const int quad = warp & 3;
        const int first_col = (warp >> 2) * C::kTotals;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + first_col;
        int acc = 0;
        uint32_t acc_phase = 0;
        bool failed = false;
        for (int round = 0; !failed; ++round) {
            const int t = grouped_turn(round, team, teams, total_tiles);
            if (t == -2) break;
            if (t < 0) continue;
            const GroupedTile g = grouped_tile<kGradB, BT>(tab, t, p);
            int kb0;
            const int kb1 = my_part((g.sum + kBK - 1) / kBK, kb0);
            float total[C::kTotals];
#pragma unroll
            for (int i = 0; i < C::kTotals; ++i) total[i] = 0.0f;
            for (int k_begin = kb0; k_begin < kb1; k_begin += kGroupedSegKb) {
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(tfull_bar(acc), acc_phase, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_grouped(p, abort_flag, kErrEpilogue);
                    failed = true;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < C::kTotals; c += W) {
                    if (first_col + c < g.cols) {
                        uint32_t r[W];
                        tmem_ld_32x32b_x16(lane_base + static_cast<uint32_t>(acc * BT + c), r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < W; ++i) total[c + i] += __uint_as_float(r[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(acc));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (failed) break;
            const int col = g.lane0 + quad * 32 + lane;
            if (splits > 1) {
                // The one tile of this cluster: every copy and MMA of it is done, so the stages can hold the totals,
                // [tile column][result column].
                float* share = reinterpret_cast<float*>(smem) + first_col * 128 + quad * 32 + lane;
#pragma unroll
                for (int i = 0; i < C::kTotals; ++i) share[i * 128] = total[i];
                continue;
            }
            if (col < p.lane_dim) {
#pragma unroll
                for (int c = 0; c < C::kTotals; c += W) {
                    const int n = min(W, g.cols - first_col - c);
                    if (n <= 0) continue;
                    float v[W];
#pragma unroll
                    for (int i = 0; i < W; ++i) v[i] = total[c + i];
                    const long long row = g.col0 + first_col + c;
                    float* dst = p.out + row * p.ldo + col + g.group * p.out_stride;
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (i < n) __stcs(dst + i * p.ldo, v[i]);
                }
            }
        }
    }

    if (splits > 1) {
        __syncwarp();
        cluster_sync();  // the totals of every CTA of the tile are in place (or a CTA gave up)
        if (team < total_tiles && *abort_flag == 0) {
            const GroupedTile g = grouped_tile<kGradB, BT>(tab, team, p);
            // Every thread an output, this CTA the tile columns rank, rank + splits, ...
            const int share = (g.cols - rank + splits - 1) / splits;
            for (int i = threadIdx.x; i < share * 128; i += C::kThreads) {
                const int c = rank + (i >> 7) * splits, col = g.lane0 + (i & 127);
                if (col >= p.lane_dim) continue;
                const uint32_t at = smem_addr(smem) + static_cast<uint32_t>(c * 128 + (i & 127)) * 4;
                float v = 0.0f;
                for (int r = 0; r < splits; ++r) v += ld_shared_cluster_f32(mapa_shared(at, static_cast<uint32_t>(r)));
                p.out[(g.col0 + c) * p.ldo + col + g.group * p.out_stride] = v;
            }
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while another still reads its totals
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

// ------------------------------------------------------------------ few rows per group
//
// Groups with a handful of rows: bound by the weights' bytes.  What stands
// between a weight and HBM's rate is shared memory: every pass over the 128 x
// 32 tile costs 16 KB of its 128 bytes a clock.  So the tile is read as little
// as possible: by the MMA once for big, against big and small activations side
// by side (columns 0 .. n and n .. 2n of one MMA), and once by the
// converter, a thread to a weight column, which leaves the small parts in
// tensor memory, from where the second MMA takes them as its A operand (and
// adds to the columns of the other small term: the main columns then see
// a third of the sums that the tensor core cuts).  That is 72 KB a k-block (of
// 32) where small parts in shared memory would move 120.  Small parts as bf16
// pairs, half the tensor memory and MMAs, were no faster (92 us either way at
// 128 rows, 64 groups of 1024 x 2048) and less exact.  Tiles of 32 rows, with
// two stages more, were within 2% at 16 and 32 rows a group and behind from
// there (8 groups, 2048 x 4096: 24 rows 93 us against 70, 48 rows 108 against 100).
//
// Cold L2: 128 rows over 64 groups of 1024 x 2048, of which 45 have a row, 84 us
// (4.5 TB/s; five rounds of tiles and a start of 5 us), 16 rows of one group x
// 16384 x 18944 221 us (5.6 TB/s).
//
// With fewer tiles than SMs, a cluster of `splits` CTAs shares a tile, each
// summing its own stretch of the sum; the totals meet in distributed shared
// memory, added in CTA order.  A cluster has room for one tile's totals, and
// the grid has a cluster for every tile that non-decreasing offsets can give.
// Decreasing ones can give more (groups then overlap): every CTA sees that in
// its table and takes whole tiles for itself, in rounds.

struct GroupedFewCfg {
    static constexpr int kCols = 64;  // rows of the group that a tile takes
    static constexpr int kLaneBytes = 128 * kBK * 4;
    static constexpr int kColBytes = 2 * kCols * kBK * 4;  // activations, then their small parts
    static constexpr int kStageBytes = kLaneBytes + kColBytes;
    static constexpr int kStages = 6;
    static constexpr int kSmall = 4;                  // small weights in tensor memory: 32 columns each
    static constexpr int kEpiWarps = 4, kConvGroups = 3, kConvWarps = 4 * kConvGroups;
    static constexpr int kThreads = 32 * (kEpiWarps + kConvWarps + 4);  // and a warpgroup with TMA and MMA
    // Registers a thread: the launch has 640 x 96, given out in shares of 128 threads.
    static constexpr int kEpiRegs = 144, kConvRegs = 88, kIssueRegs = 72;
    static_assert(kEpiRegs + kConvGroups * kConvRegs + kIssueRegs <= 480, "more registers than the launch has");
    static constexpr int kSmallCol = 4 * kCols;       // first TMEM column behind the two accumulators of 2 kCols
    static constexpr int kTmemCols = 512;
    static constexpr int kSegKb = 4;                  // k-blocks to an accumulator: 16 sums into a main column
    static constexpr int kTableOffset = kStages * kStageBytes;
    static constexpr int kBarOffset = kTableOffset + kGroupedTableBytes;
    static constexpr int kNumBars = 2 * kStages + 2 * kSmall + 4 + 1;
    static constexpr int kSmemBytes = 1024 + kBarOffset + kNumBars * 8 + 16;
    static_assert(kSmallCol + 32 * kSmall <= kTmemCols, "tensor memory");
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

template <int MODE>
__global__ void __launch_bounds__(GroupedFewCfg::kThreads, 1)
    grouped_few_kernel(const __grid_constant__ CUtensorMap tm_lane, const __grid_constant__ CUtensorMap tm_col,
                       const __grid_constant__ GroupedParams p, const int cluster) {
    using C = GroupedFewCfg;
    constexpr int BT = C::kCols;
    static_assert(MODE != kGradB, "the rows are the columns here");
    constexpr bool kLaneMn = MODE == kForward;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    GroupedTable& tab = *reinterpret_cast<GroupedTable*>(smem + C::kTableOffset);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (C::kStages + s); };
    auto conv_bar = [&](int s) { return bar0 + 8u * (2 * C::kStages + s); };
    auto sfree_bar = [&](int s) { return bar0 + 8u * (2 * C::kStages + C::kSmall + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + 2 + a); };
    const uint32_t drain_bar = bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (the converter's warp w reads and writes TMEM lanes 32 (w % 4) ..: both roles start at a multiple of four)
    constexpr int kConvWarp = C::kEpiWarps, kTmaWarp = kConvWarp + C::kConvWarps, kMmaWarp = kTmaWarp + 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int s = 0; s < C::kSmall; ++s) {
            mbar_init(conv_bar(s), 4);  // a group of the converter
            mbar_init(sfree_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), C::kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_lane);
        tma_prefetch_desc(&tm_col);
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_addr(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    wait_for_previous_kernel();
    if (warp == kMmaWarp) let_next_kernel_in();  // behind this CTA's allocation
    if (warp == kConvWarp) grouped_scan<MODE, BT>(tab, p, lane);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = tab.total;
    const int splits = total_tiles > static_cast<int>(gridDim.x) / cluster ? 1 : cluster;
    const int team = blockIdx.x / splits, teams = gridDim.x / splits, rank = blockIdx.x - team * splits;
    // This CTA's k-blocks [kb0, kb1) of every tile (all sums are as long as sum_dim).
    const int all_kb = (p.sum_dim + kBK - 1) / kBK;
    const int kb0 = static_cast<int>(static_cast<long long>(all_kb) * rank / splits);
    const int kb1 = static_cast<int>(static_cast<long long>(all_kb) * (rank + 1) / splits);

    if (warp >= kTmaWarp) {
        fewer_registers<C::kIssueRegs>();
        if (warp == kTmaWarp) {
            // ------------------------------------------------------------ TMA producer
            const bool leader = elect_one();
            int stage = 0;
            uint32_t phase = 0;
            long long issued = 0;
            bool ok = true;
            for (int round = 0; ok; ++round) {
                const int t = grouped_turn(round, team, teams, total_tiles);
                if (t == -2) break;
                if (t < 0) continue;
                const GroupedTile g = grouped_tile<MODE, BT>(tab, t, p);
                const int col_boxes = (g.cols + 31) / 32;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (*abort_flag || !mbar_wait(empty_bar(stage), phase ^ 1u, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    if (leader) {
                        const uint32_t st = smem_addr(smem + stage * C::kStageBytes), fb = full_bar(stage);
                        mbar_arrive_expect_tx(fb, C::kLaneBytes + col_boxes * kBoxBytes);
                        const int q0 = kb * kBK;
                        if (MODE == kForward) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                tma_load_3d(st + j * kBoxBytes, &tm_lane, fb, g.lane0 + 32 * j, q0, g.group);
                        } else {
                            tma_load_3d(st, &tm_lane, fb, q0, g.lane0, g.group);
                        }
                        for (int j = 0; j < col_boxes; ++j)
                            tma_load_2d(st + C::kLaneBytes + j * kBoxBytes, &tm_col, fb, q0, g.row0 + g.col0 + 32 * j);
                    }
                    __syncwarp();
                    ++issued;
                    if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok && leader) {
                raise_grouped(p, abort_flag, kErrProducer);
                // Copies in flight land in this CTA's shared memory: wait for them before leaving.
                for (long long i = issued > C::kStages ? issued - C::kStages : 0; i < issued; ++i)
                    mbar_wait(full_bar(static_cast<int>(i % C::kStages)), static_cast<uint32_t>((i / C::kStages) & 1),
                              p.timeout_ns);
            }
            __syncwarp();
        } else if (warp == kMmaWarp) {
            // ------------------------------------------------------------ MMA issuer
            constexpr uint32_t kHiMn = smem_desc_hi(512, kLayoutSW128Base32B), kHiK = smem_desc_hi(1024, kLayoutSW128);
            constexpr uint32_t kLaneHi = kLaneMn ? kHiMn : kHiK, kLaneStep = kLaneMn ? 64 : 2;
            const uint32_t leader = elect_one();
            int stage = 0, small = 0, acc = 0;
            uint32_t small_phase = 0, acc_phase = 0;
            bool ok = true;
            for (int round = 0; ok; ++round) {
                const int t = grouped_turn(round, team, teams, total_tiles);
                if (t == -2) break;
                if (t < 0) continue;
                const GroupedTile g = grouped_tile<MODE, BT>(tab, t, p);
                const int n = (g.cols + 15) & ~15;
                const uint32_t both = idesc_tf32_major(128, p.split3 ? 2 * n : n, kLaneMn, 0);
                const uint32_t one = idesc_tf32_major(128, n, 0, 0);  // (A in tensor memory is K-major)
                int in_seg = 0;
                for (int kb = kb0; kb < kb1; ++kb) {
                    bool ready = *abort_flag == 0;
                    if (ready && in_seg == 0) ready = mbar_wait(tempty_bar(acc), acc_phase ^ 1u, p.timeout_ns);
                    if (!ready || !mbar_wait(conv_bar(small), small_phase, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const bool end_seg = ++in_seg == C::kSegKb || kb == kb1 - 1;
                    const uint32_t d = tmem_base + static_cast<uint32_t>(acc * 2 * BT);
                    const uint32_t a_small = tmem_base + static_cast<uint32_t>(C::kSmallCol + 32 * small);
                    const uint32_t big = smem_addr(smem + stage * C::kStageBytes);
                    const uint32_t bl = smem_desc_lo(big, kLaneMn ? kBoxBytes : 16);
                    const uint32_t bc = smem_desc_lo(big + C::kLaneBytes, 16);
                    const int steps = min(4, (g.sum - kb * kBK + 7) / 8);
                    const uint32_t begun = in_seg > 1 ? 1u : 0u;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (kk >= steps) break;
                        const uint64_t db = smem_desc_of(kHiK, bc + kk * 2);
                        mma_tf32_of(leader, d, smem_desc_of(kLaneHi, bl + kk * kLaneStep), db, both, kk ? 1u : begun);
                        if (p.split3) mma_tf32_ts_of(leader, d + n, a_small + kk * 8, db, one, 1u);
                    }
                    if (leader) {
                        mma_commit(empty_bar(stage));
                        mma_commit(sfree_bar(small));
                        if (end_seg) mma_commit(tfull_bar(acc));
                    }
                    __syncwarp();
                    if (++stage == C::kStages) stage = 0;
                    if (++small == C::kSmall) { small = 0; small_phase ^= 1u; }
                    if (end_seg) {
                        in_seg = 0;
                        acc ^= 1;
                        if (acc == 0) acc_phase ^= 1u;
                    }
                }
            }
            if (leader) {
                if (!ok) raise_grouped(p, abort_flag, kErrMma);
                mma_commit(drain_bar);
                if (!mbar_wait(drain_bar, 0, p.timeout_ns)) raise_grouped(p, abort_flag, kErrMma);
            }
            __syncwarp();
        }
    } else if (warp >= kConvWarp) {
        // ------------------------------------------------------------ converter: a weight column a thread
        fewer_registers<C::kConvRegs>();
        // Each group of four warps takes every kConvGroups-th k-block: what a k-block costs besides the work (three
        // waits of about 130 clocks) is then paid once for 32 k a thread.
        const int t0 = threadIdx.x - 32 * kConvWarp, row = t0 & 127, turn = t0 >> 7;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(row & ~31) << 16) + C::kSmallCol;
        unsigned count = 0;  // k-blocks so far
        bool failed = false;
        for (int round = 0; !failed; ++round) {
            const int t = grouped_turn(round, team, teams, total_tiles);
            if (t == -2) break;
            if (t < 0) continue;
            const GroupedTile g = grouped_tile<MODE, BT>(tab, t, p);
            const int n = (g.cols + 15) & ~15;
            for (int kb = kb0; kb < kb1; ++kb, ++count) {
                if (static_cast<int>(count % C::kConvGroups) != turn) continue;
                const int stage = static_cast<int>(count % C::kStages), small = static_cast<int>(count % C::kSmall);
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(full_bar(stage), (count / C::kStages) & 1u, p.timeout_ns) &&
                                 mbar_wait(sfree_bar(small), ((count / C::kSmall) & 1u) ^ 1u, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_grouped(p, abort_flag, kErrProducer);
                    failed = true;
                    break;
                }
                if (p.split3) {
                    tc_fence_after();
                    const uint8_t* st = smem + stage * C::kStageBytes;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // (16 k at a time: fewer registers)
                        uint32_t r[16];
                        if (kLaneMn) {
                            // [k][n]: box n / 32, 128 bytes a k, its 32-byte chunks swizzled by k % 4.
                            const uint8_t* src = st + (row >> 5) * kBoxBytes + half * 16 * 128 + (row & 7) * 4;
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                r[k] = __float_as_uint(small_of(
                                    *reinterpret_cast<const float*>(src + k * 128 + ((((row >> 3) & 3) ^ (k & 3)) << 5))));
                        } else {
                            // [n][k]: 128 bytes a weight column, 16-byte chunks swizzled by n % 8.
                            const uint8_t* src = st + row * 128;
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const float4 v = *reinterpret_cast<const float4*>(src + (((4 * half + c) ^ (row & 7)) << 4));
                                r[4 * c] = __float_as_uint(small_of(v.x));
                                r[4 * c + 1] = __float_as_uint(small_of(v.y));
                                r[4 * c + 2] = __float_as_uint(small_of(v.z));
                                r[4 * c + 3] = __float_as_uint(small_of(v.w));
                            }
                        }
                        tmem_st_32x32b_x16(lane_base + static_cast<uint32_t>(32 * small + 16 * half), r);
                    }
                    // The activations' small parts go behind them, to rows n .. 2n of the same swizzled tile.
                    float4* x = reinterpret_cast<float4*>(smem + stage * C::kStageBytes + C::kLaneBytes);
                    for (int i = row; i < n * 8; i += 128) {
                        const float4 v = x[i];
                        x[i + n * 8] = make_float4(small_of(v.x), small_of(v.y), small_of(v.z), small_of(v.w));
                    }
                    tmem_st_wait();
                    fence_proxy_async_shared();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(conv_bar(small));
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue: a result column and all rows a thread
        more_registers<C::kEpiRegs>();
        constexpr int W = 16;
        const int quad = warp & 3;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
        int acc = 0;
        uint32_t acc_phase = 0;
        bool failed = false;
        for (int round = 0; !failed; ++round) {
            const int t = grouped_turn(round, team, teams, total_tiles);
            if (t == -2) break;
            if (t < 0) continue;
            const GroupedTile g = grouped_tile<MODE, BT>(tab, t, p);
            const int n = (g.cols + 15) & ~15;
            float total[BT];
#pragma unroll
            for (int i = 0; i < BT; ++i) total[i] = 0.0f;
            for (int k_begin = kb0; k_begin < kb1; k_begin += C::kSegKb) {
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(tfull_bar(acc), acc_phase, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_grouped(p, abort_flag, kErrEpilogue);
                    failed = true;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < BT; c += W) {
                    if (c < n) {
                        uint32_t r[W], s[W];
                        tmem_ld_32x32b_x16(lane_base + static_cast<uint32_t>(acc * 2 * BT + c), r);
                        if (p.split3) tmem_ld_32x32b_x16(lane_base + static_cast<uint32_t>(acc * 2 * BT + n + c), s);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < W; ++i)
                            total[c + i] += p.split3 ? __uint_as_float(r[i]) + __uint_as_float(s[i]) : __uint_as_float(r[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(acc));
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (failed) break;
            const int col = g.lane0 + quad * 32 + lane;
            if (splits > 1) {
                // The one tile of this cluster: every copy and MMA of it is done, so stage 0 can hold the totals,
                // [row][column].
                float* share = reinterpret_cast<float*>(smem) + quad * 32 + lane;
#pragma unroll
                for (int i = 0; i < BT; ++i) share[i * 128] = total[i];
                continue;
            }
            if (col < p.lane_dim) {
#pragma unroll
                for (int c = 0; c < BT; c += W) {
                    const int m = min(W, g.cols - c);
                    if (m <= 0) continue;
                    float v[W];
#pragma unroll
                    for (int i = 0; i < W; ++i) v[i] = total[c + i];
                    const long long row = g.row0 + g.col0 + c;
                    apply_column<W>(v, row, m, col, g.group, p.epi);
                    float* dst = p.out + row * p.ldo + col;
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (i < m) __stcs(dst + i * p.ldo, v[i]);
                }
            }
        }
    }

    if (splits > 1) {
        __syncwarp();
        cluster_sync();  // the totals of every CTA of the tile are in place (or a CTA gave up)
        if (team < total_tiles && *abort_flag == 0) {
            const GroupedTile g = grouped_tile<MODE, BT>(tab, team, p);
            // Every thread an output, this CTA the rows rank, rank + splits, ...
            const int share = (g.cols - rank + splits - 1) / splits;
            for (int i = threadIdx.x; i < share * 128; i += C::kThreads) {
                const int row = rank + (i >> 7) * splits, col = g.lane0 + (i & 127);
                if (col >= p.lane_dim) continue;
                const uint32_t at = smem_addr(smem) + static_cast<uint32_t>(row * 128 + (i & 127)) * 4;
                float v = 0.0f;
                for (int r = 0; r < splits; ++r) v += ld_shared_cluster_f32(mapa_shared(at, static_cast<uint32_t>(r)));
                const long long out_row = g.row0 + g.col0 + row;
                p.out[out_row * p.ldo + col] = apply_cell(v, out_row, col, g.group, p.epi);
            }
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while another still reads its totals
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

// ------------------------------------------------------------------ CTA pairs
//
// Groups with many rows: bound by the tensor cores, and on one SM by shared
// memory, whose 128 bytes a clock the MMA (24 bytes per operand element and
// product triple, with the copies and the converter) would need 1.5 times.  Two
// CTAs share a tile of 256 lanes x 256 columns (cta_group::2): each stages
// 128 lanes and half the columns, converts them itself, and holds its
// lanes' accumulators; per byte staged the pair multiplies twice as much.
// The epilogue's 128 totals a thread need more registers than an even
// split gives: the other warps hand some over (setmaxnreg; the shares add up
// to the launch's 640 x 96).
//
// 8192 rows, 8 groups of 4096 x 4096: 1103 us in a burst, 249 TFLOP/s of fp32
// products (three TF32 products each), and 1270 us once the power limit has the
// clock at 1.57 GHz; 4096 rows of 4 groups keep the tensor cores 76% active.
// 8191 rows, 8 groups, 1024 x 4096: grad_b with dbias 305 us.  4001 rows of 16
// groups, 1024 x 4096: grad_a 220-235 us; of the 74 pairs 64 have a whole tile and
// some a tile of the few rows behind one as well (balance, not rate).

struct GroupedPairCfg {
    static constexpr int kCols = 256;
    static constexpr int kLaneBytes = 128 * kBK * 4;
    static constexpr int kColBytes = (kCols / 2) * kBK * 4;
    static constexpr int kStageBytes = kLaneBytes + kColBytes;
    static constexpr int kStages = 4, kSmall = 2;
    static constexpr int kEpiWarps = 8, kConvWarps = 8;
    static constexpr int kThreads = 640;              // epilogue, converter, and a warpgroup with TMA and MMA
    static constexpr int kTmemCols = 512;
    static constexpr int kTotals = 128;
    static constexpr int kSmallOffset = kStages * kStageBytes;
    static constexpr int kTableOffset = kSmallOffset + kSmall * kStageBytes;
    static constexpr int kSumBuffers = 3;             // of the converter warps' sums for dbias
    static constexpr int kSumsOffset = kTableOffset + kGroupedTableBytes;
    static constexpr int kBarOffset = kSumsOffset + kSumBuffers * kConvWarps * 128 * 4;
    static constexpr int kNumBars = 2 * kStages + 2 * kSmall + 4 + 1 + kSumBuffers;
    static constexpr int kSmemBytes = 1024 + kBarOffset + kNumBars * 8 + 16;
    static constexpr int kEpiRegs = 168, kConvRegs = 48, kIssueRegs = 48;
    static_assert(2 * kEpiRegs + 2 * kConvRegs + kIssueRegs <= 480, "more registers than the launch has");
    static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedPairCfg::kThreads, 1)
    grouped_pair_kernel(const __grid_constant__ CUtensorMap tm_lane, const __grid_constant__ CUtensorMap tm_col,
                        const __grid_constant__ GroupedParams p) {
    using C = GroupedPairCfg;
    constexpr int BT = C::kCols;
    constexpr bool kLaneMn = MODE != kGradA, kColMn = MODE == kGradB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    GroupedTable& tab = *reinterpret_cast<GroupedTable*>(smem + C::kTableOffset);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };                         // TMA -> converter (own CTA)
    auto empty_bar = [&](int s) { return bar0 + 8u * (C::kStages + s); };         // MMA -> TMA (both CTAs)
    auto conv_bar = [&](int s) { return bar0 + 8u * (2 * C::kStages + s); };      // both converters -> MMA (leader)
    auto sfree_bar = [&](int s) { return bar0 + 8u * (2 * C::kStages + C::kSmall + s); };  // MMA -> converter (both)
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + 2 + a); };
    const uint32_t drain_bar = bar0 + 8u * (2 * C::kStages + 2 * C::kSmall + 4);
    auto sums_bar = [&](int b) { return drain_bar + 8u * (1 + b); };              // converter warps -> the first of them

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    constexpr int kConvWarp = C::kEpiWarps, kTmaWarp = kConvWarp + C::kConvWarps, kMmaWarp = kTmaWarp + 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int s = 0; s < C::kSmall; ++s) {
            mbar_init(conv_bar(s), 2 * C::kConvWarps);
            mbar_init(sfree_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 2 * C::kEpiWarps);
        }
        mbar_init(drain_bar, 1);
        for (int b = 0; b < C::kSumBuffers; ++b) mbar_init(sums_bar(b), C::kConvWarps);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tm_lane);
        tma_prefetch_desc(&tm_col);
    }
    if (warp == kMmaWarp) {
        tmem_alloc_pair(smem_addr(tmem_slot), C::kTmemCols);
        tmem_relinquish_pair();
    }
    wait_for_previous_kernel();
    if (warp == kMmaWarp) let_next_kernel_in();  // behind this CTA's allocation
    if (warp == kConvWarp) grouped_scan<MODE, BT>(tab, p, lane);
    __syncwarp();
    tc_fence_before();
    cluster_sync();  // barriers initialised, TMEM allocated and the tables written in both CTAs
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int total_tiles = tab.total;
    // The pair's columns are rounded up to 32: each CTA stages half of them.
    auto half_cols = [](int cols) { return ((cols + 31) & ~31) / 2; };

    if (warp >= kTmaWarp) {
        fewer_registers<C::kIssueRegs>();
        if (warp == kTmaWarp) {
            // -------------------------------------------------------- TMA producer (both CTAs)
            const bool leader = elect_one();
            int stage = 0;
            uint32_t phase = 0;
            long long issued = 0;
            bool ok = true;
            for (int round = 0; ok; ++round) {
                const int t = grouped_turn(round, pair, num_pairs, total_tiles);
                if (t == -2) break;
                if (t < 0) continue;
                const GroupedTile g = grouped_tile<MODE, BT, 256>(tab, t, p);
                const int half = half_cols(g.cols), col_boxes = (half + 31) / 32;
                const int lane0 = g.lane0 + static_cast<int>(rank) * 128, col0 = g.col0 + static_cast<int>(rank) * half;
                const int num_kb = (g.sum + kBK - 1) / kBK;
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (*abort_flag || !mbar_wait_cluster(empty_bar(stage), phase ^ 1u, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    if (leader) {
                        const uint32_t st = smem_addr(smem + stage * C::kStageBytes), fb = full_bar(stage);
                        mbar_arrive_expect_tx(fb, C::kLaneBytes + col_boxes * kBoxBytes);
                        const int q0 = kb * kBK;
                        if (MODE == kForward) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                tma_load_3d(st + j * kBoxBytes, &tm_lane, fb, lane0 + 32 * j, q0, g.group);
                        } else if (MODE == kGradA) {
                            tma_load_3d(st, &tm_lane, fb, q0, lane0, g.group);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                tma_load_2d(st + j * kBoxBytes, &tm_lane, fb, lane0 + 32 * j, g.row0 + q0);
                        }
                        for (int j = 0; j < col_boxes; ++j) {
                            const uint32_t dst = st + C::kLaneBytes + j * kBoxBytes;
                            if (MODE == kGradB) {
                                tma_load_2d(dst, &tm_col, fb, col0 + 32 * j, g.row0 + q0);
                            } else {
                                tma_load_2d(dst, &tm_col, fb, q0, g.row0 + col0 + 32 * j);
                            }
                        }
                    }
                    __syncwarp();
                    ++issued;
                    if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok && leader) {
                raise_grouped(p, abort_flag, kErrProducer);
                // Copies in flight land in this CTA's shared memory: wait for them before leaving.
                for (long long i = issued > C::kStages ? issued - C::kStages : 0; i < issued; ++i)
                    mbar_wait(full_bar(static_cast<int>(i % C::kStages)), static_cast<uint32_t>((i / C::kStages) & 1),
                              p.timeout_ns);
            }
            __syncwarp();
        } else if (warp == kMmaWarp && rank == 0) {
            // -------------------------------------------------------- MMA issuer (leader only)
            constexpr uint32_t kHiMn = smem_desc_hi(512, kLayoutSW128Base32B), kHiK = smem_desc_hi(1024, kLayoutSW128);
            constexpr uint32_t kLaneHi = kLaneMn ? kHiMn : kHiK, kColHi = kColMn ? kHiMn : kHiK;
            constexpr uint32_t kLaneStep = kLaneMn ? 64 : 2, kColStep = kColMn ? 64 : 2;
            const bool leader = elect_one();
            int stage = 0, small = 0, acc = 0;
            uint32_t small_phase = 0, acc_phase = 0;
            bool ok = true;
            for (int round = 0; ok; ++round) {
                const int t = grouped_turn(round, pair, num_pairs, total_tiles);
                if (t == -2) break;
                if (t < 0) continue;
                const GroupedTile g = grouped_tile<MODE, BT, 256>(tab, t, p);
                const uint32_t idesc = idesc_tf32_major(256, 2 * half_cols(g.cols), kLaneMn, kColMn);
                const int num_kb = (g.sum + kBK - 1) / kBK;
                int in_seg = 0;
                for (int kb = 0; kb < num_kb; ++kb) {
                    bool ready = *abort_flag == 0;
                    if (ready && in_seg == 0) ready = mbar_wait_cluster(tempty_bar(acc), acc_phase ^ 1u, p.timeout_ns);
                    if (!ready || !mbar_wait_cluster(conv_bar(small), small_phase, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const bool end_seg = ++in_seg == kGroupedSegKb || kb == num_kb - 1;
                    if (leader) {
                        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BT);
                        const uint32_t big = smem_addr(smem + stage * C::kStageBytes);
                        const uint32_t low = smem_addr(smem + C::kSmallOffset + small * C::kStageBytes);
                        const uint32_t bl = smem_desc_lo(big, kLaneMn ? kBoxBytes : 16);
                        const uint32_t bc = smem_desc_lo(big + C::kLaneBytes, kColMn ? kBoxBytes : 16);
                        const uint32_t sl = smem_desc_lo(low, kLaneMn ? kBoxBytes : 16);
                        const uint32_t sc = smem_desc_lo(low + C::kLaneBytes, kColMn ? kBoxBytes : 16);
                        const int steps = min(4, (g.sum - kb * kBK + 7) / 8);
                        const uint32_t begun = in_seg > 1 ? 1u : 0u;
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            if (kk >= steps) break;
                            const uint64_t da = smem_desc_of(kLaneHi, bl + kk * kLaneStep);
                            const uint64_t db = smem_desc_of(kColHi, bc + kk * kColStep);
                            if (p.split3) {
                                // Small cross terms first, the dominant product last.
                                mma_tf32_pair(d, da, smem_desc_of(kColHi, sc + kk * kColStep), idesc, kk ? 1u : begun);
                                mma_tf32_pair(d, smem_desc_of(kLaneHi, sl + kk * kLaneStep), db, idesc, 1u);
                                mma_tf32_pair(d, da, db, idesc, 1u);
                            } else {
                                mma_tf32_pair(d, da, db, idesc, kk ? 1u : begun);
                            }
                        }
                        mma_commit_pair(empty_bar(stage), 0x3);
                        mma_commit_pair(sfree_bar(small), 0x3);
                        if (end_seg) mma_commit_pair(tfull_bar(acc), 0x3);
                    }
                    __syncwarp();
                    if (++stage == C::kStages) stage = 0;
                    if (++small == C::kSmall) { small = 0; small_phase ^= 1u; }
                    if (end_seg) {
                        in_seg = 0;
                        acc ^= 1;
                        if (acc == 0) acc_phase ^= 1u;
                    }
                }
            }
            if (leader) {
                if (!ok) raise_grouped(p, abort_flag, kErrMma);
                mma_commit_pair(drain_bar, 0x1);
                if (!mbar_wait_cluster(drain_bar, 0, p.timeout_ns)) raise_grouped(p, abort_flag, kErrMma);
            }
            __syncwarp();
        }
    } else if (warp >= kConvWarp) {
        // ------------------------------------------------------------ converter (each CTA its own half)
        fewer_registers<C::kConvRegs>();
        const int t0 = threadIdx.x - 32 * kConvWarp;
        const uint32_t conv_leader = mapa_shared(conv_bar(0), 0);
        int stage = 0, small = 0, sum_buf = 0;
        uint32_t phase = 0, small_phase = 0, sum_phase = 0;
        bool failed = false;
        for (int round = 0; !failed; ++round) {
            const int t = grouped_turn(round, pair, num_pairs, total_tiles);
            if (t == -2) break;
            if (t < 0) continue;
            const GroupedTile g = grouped_tile<MODE, BT, 256>(tab, t, p);
            const bool sums = MODE == kGradB && p.dbias && g.col0 == 0;  // the bias gradient, once for each lane tile
            float sum[MODE == kGradB ? 16 : 1];
#pragma unroll
            for (int e = 0; e < (MODE == kGradB ? 16 : 1); ++e) sum[e] = 0.0f;
            const int col_boxes = (half_cols(g.cols) + 31) / 32;
            const int num_kb = (g.sum + kBK - 1) / kBK;
            for (int kb = 0; kb < num_kb; ++kb) {
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait(full_bar(stage), phase, p.timeout_ns) &&
                                 mbar_wait_cluster(sfree_bar(small), small_phase ^ 1u, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_grouped(p, abort_flag, kErrProducer);
                    failed = true;
                    break;
                }
                convert_tile<MODE, 32 * C::kConvWarps>(smem + stage * C::kStageBytes, smem + C::kSmallOffset + small * C::kStageBytes, t0,
                                        1024 + col_boxes * 256, g.sum - kb * kBK, p.split3);
                if (sums) add_lane_columns(smem + stage * C::kStageBytes, t0, sum);
                fence_proxy_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive_peer(conv_leader + 8u * small);
                if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                if (++small == C::kSmall) { small = 0; small_phase ^= 1u; }
            }
            if (failed || !sums) continue;
            float* out = p.dbias + static_cast<long long>(g.group) * p.lane_dim;
            const int col = g.lane0 + static_cast<int>(rank) * 128 + t0;
            if (num_kb == 0) {
                if (t0 < 128 && col < p.lane_dim) out[col] = 0.0f;
                continue;
            }
            // Each warp leaves its sums; the first four add them up in warp order.  No warp is three tiles ahead of
            // another (the MMA of two k-blocks back needs all of them), so three buffers take turns.
            float* part = reinterpret_cast<float*>(smem + C::kSumsOffset) + sum_buf * C::kConvWarps * 128;
            leave_lane_sums(sum, part + (t0 >> 5) * 128, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(sums_bar(sum_buf));
            if (t0 < 128) {
                const bool got = mbar_wait(sums_bar(sum_buf), sum_phase, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0) raise_grouped(p, abort_flag, kErrProducer);
                    failed = true;
                } else if (col < p.lane_dim) {
                    float v = 0.0f;
#pragma unroll
                    for (int w = 0; w < C::kConvWarps; ++w) v += part[w * 128 + t0];
                    out[col] = v;
                }
            }
            if (++sum_buf == C::kSumBuffers) { sum_buf = 0; sum_phase ^= 1u; }
        }
    } else {
        // ------------------------------------------------------------ epilogue (both CTAs, their own lanes)
        more_registers<C::kEpiRegs>();
        constexpr int W = 16;
        const int quad = warp & 3, first_col = (warp >> 2) * C::kTotals;
        const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + first_col;
        const uint32_t tempty_leader = mapa_shared(tempty_bar(0), 0);
        int acc = 0;
        uint32_t acc_phase = 0;
        bool failed = false;
        for (int round = 0; !failed; ++round) {
            const int t = grouped_turn(round, pair, num_pairs, total_tiles);
            if (t == -2) break;
            if (t < 0) continue;
            const GroupedTile g = grouped_tile<MODE, BT, 256>(tab, t, p);
            const int num_kb = (g.sum + kBK - 1) / kBK;
            float total[C::kTotals];
#pragma unroll
            for (int i = 0; i < C::kTotals; ++i) total[i] = 0.0f;
            for (int k_begin = 0; k_begin < num_kb; k_begin += kGroupedSegKb) {
                const bool stop = __any_sync(0xffffffffu, *abort_flag != 0);
                const bool got = !stop && mbar_wait_cluster(tfull_bar(acc), acc_phase, p.timeout_ns);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0 && !stop) raise_grouped(p, abort_flag, kErrEpilogue);
                    failed = true;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < C::kTotals; c += W) {
                    if (first_col + c < g.cols) {
                        uint32_t r[W];
                        tmem_ld_32x32b_x16(lane_base + static_cast<uint32_t>(acc * BT + c), r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < W; ++i) total[c + i] += __uint_as_float(r[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(tempty_leader + 8u * acc);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
            if (failed) break;
            const int col = g.lane0 + static_cast<int>(rank) * 128 + quad * 32 + lane;
            if (col < p.lane_dim) {
#pragma unroll
                for (int c = 0; c < C::kTotals; c += W) {
                    const int n = min(W, g.cols - first_col - c);
                    if (n <= 0) continue;
                    float v[W];
#pragma unroll
                    for (int i = 0; i < W; ++i) v[i] = total[c + i];
                    const long long row = g.col0 + first_col + c + (MODE == kGradB ? 0 : g.row0);
                    if (MODE != kGradB) apply_column<W>(v, row, n, col, g.group, p.epi);
                    float* dst = p.out + row * p.ldo + col + (MODE == kGradB ? g.group * p.out_stride : 0);
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (i < n) __stcs(dst + i * p.ldo, v[i]);
                }
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync();  // no CTA leaves while its peer may still signal its barriers
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, C::kTmemCols);
    }
}

// dbias[e, n] = the sum of dY[r, n] over group e's rows: 32 columns of one group to a block.
__global__ void __launch_bounds__(1024) grouped_column_sums(const float* dy, long long ld, const int* offsets, int rows,
                                                            int N, float* dbias) {
    __shared__ float part[32][33];
    const int e = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
    const int r0 = min(max(__ldg(offsets + e), 0), rows);
    const int r1 = min(max(__ldg(offsets + e + 1), r0), rows);
    float s = 0.0f;
    if (c < N)
        for (int r = r0 + threadIdx.y; r < r1; r += 32) s += __ldg(dy + r * ld + c);
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = part[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int cc = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && cc < N) dbias[static_cast<long long>(e) * N + cc] = s;
}

// Row-major [groups][rows][cols] (groups 0: a plain [rows][cols]) read in boxes of box_rows x 32 floats,
// rounded to TF32 by the copy or (3xTF32) as it is.
bool grouped_map(CUtensorMap* map, const float* base, int groups, long long rows, long long cols, long long ld,
                 long long stride, int box_rows, bool mn_major, bool round) {
    const unsigned long long dims[3] = {static_cast<unsigned long long>(cols), static_cast<unsigned long long>(rows),
                                        static_cast<unsigned long long>(groups)};
    const unsigned long long strides[2] = {static_cast<unsigned long long>(ld) * 4,
                                           static_cast<unsigned long long>(groups > 1 ? stride : rows * ld) * 4};
    const unsigned box[3] = {32, static_cast<unsigned>(box_rows), 1};
    return encode_tensor_map(map, round ? CU_TENSOR_MAP_DATA_TYPE_TFLOAT32 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32,
                             groups ? 3 : 2, base, dims, strides, box,
                             mn_major ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

// The two tensor maps of a call; the lane side's box is 32 x 32 floats, or 128 rows of 32 in grad_a.
template <int MODE>
bool grouped_maps(const GroupedCall& g, bool round, CUtensorMap* lane, CUtensorMap* col) {
    if (MODE == kGradB)
        return grouped_map(lane, g.w, 0, g.rows, g.N, g.ldw, 0, kBK, true, round) &&
               grouped_map(col, g.x, 0, g.rows, g.K, g.ldx, 0, kBK, true, round);
    return grouped_map(lane, g.w, g.groups, g.K, g.N, g.ldw, g.w_stride, MODE == kForward ? kBK : 128, MODE == kForward,
                       round) &&
           grouped_map(col, g.x, 0, g.rows, MODE == kForward ? g.K : g.N, g.ldx, 0, 32, false, round);
}

// Which kernel runs a product, its tile and the CTAs that share one.
struct GroupedPlan {
    bool pair;
    int lanes, cols;   // of a tile: result columns, and rows of a group (grad_b: columns of A)
    long long tiles;   // at most, for non-decreasing offsets
    int cluster;       // CTAs that share a tile's sum
};

constexpr int kMaxSplits = 8;

GroupedPlan plan_grouped(int mode, int rows, int groups, int N, int K, int num_sms) {
    const int lane_dim = mode == kGradA ? K : N;
    // At most so many tiles for non-decreasing offsets: a part of a column tile more for each group that has a row.
    auto most_tiles = [&](int lanes, int cols) {
        const long long col_tiles =
            mode == kGradB ? static_cast<long long>((K + cols - 1) / cols) * groups : rows / cols + std::min(groups, rows);
        return col_tiles * ((lane_dim + lanes - 1) / lanes);
    };
    // By the rows that a group has on average.  8 groups of uneven sizes, 2048 x 4096, cold L2, a CTA with 64 rows to a
    // tile / a pair with 256, in us: 80 rows 131 / -, 88 rows 131 / 127, 96 rows 133 / 129, 128 rows 166 / 135, 192 rows 228 / 191.
    // A pair's tile is eight times the other's, so there also have to be enough of them for the pairs: 459 rows of 12
    // groups, 811 x 1022, 32 us against the pairs' 42.  grad_b has its columns from K instead, and a CTA takes 128.
    const int cols = mode == kGradB ? K : (rows + groups - 1) / groups;
    const long long pair_tiles = most_tiles(256, GroupedPairCfg::kCols);
    if (cols > 84 && lane_dim > 128 && pair_tiles >= num_sms * 3 / 8)
        return {true, 256, GroupedPairCfg::kCols, pair_tiles, 2};
    GroupedPlan plan{false, 128, mode == kGradB ? GroupedGradBCfg::kCols : GroupedFewCfg::kCols, 0, 1};
    plan.tiles = most_tiles(plan.lanes, plan.cols);
    // Clusters while each still has SMs of its own and every CTA two k-blocks (of grad_b's rows, if they are spread
    // evenly, which is only a guess).
    const int sum = mode == kForward ? K : mode == kGradA ? N : rows / groups;
    const int all_kb = (sum + kBK - 1) / kBK;
    while (plan.cluster < kMaxSplits && 2 * plan.cluster * plan.tiles <= num_sms && all_kb >= 4 * plan.cluster) plan.cluster *= 2;
    return plan;
}

// Launches `kernel` as persistent CTAs, or as clusters that share a tile each.
template <typename Kernel>
cudaError_t launch_clusters(Kernel kernel, int threads, int smem, const GroupedPlan& plan, int num_sms, cudaStream_t stream,
                            const CUtensorMap& lane, const CUtensorMap& col, const GroupedParams& p) {
    const dim3 grid(static_cast<unsigned>(plan.cluster > 1 ? plan.tiles * plan.cluster : std::min<long long>(plan.tiles, num_sms)));
    return launch_early(kernel, grid, dim3(threads), smem, stream, plan.cluster, lane, col, p, plan.cluster);
}

cudaError_t run_grouped_grad_b(const GroupedCall& g, GroupedParams& p, bool split3, const GroupedPlan& plan, int num_sms,
                               cudaStream_t stream) {
    using C = GroupedGradBCfg;
    const cudaError_t e = allow_shared<grouped_grad_b_kernel>(C::kSmemBytes);
    if (e != cudaSuccess) return e;
    CUtensorMap lane, col;
    if (!grouped_maps<kGradB>(g, !split3, &lane, &col)) return cudaErrorInvalidValue;
    return launch_clusters(grouped_grad_b_kernel, C::kThreads, C::kSmemBytes, plan, num_sms, stream, lane, col, p);
}

template <int MODE>
cudaError_t run_grouped_few(const GroupedCall& g, GroupedParams& p, bool split3, const GroupedPlan& plan, int num_sms,
                            cudaStream_t stream) {
    using C = GroupedFewCfg;
    const cudaError_t e = allow_shared<grouped_few_kernel<MODE>>(C::kSmemBytes);
    if (e != cudaSuccess) return e;
    CUtensorMap lane, col;
    if (!grouped_maps<MODE>(g, !split3, &lane, &col)) return cudaErrorInvalidValue;
    return launch_clusters(grouped_few_kernel<MODE>, C::kThreads, C::kSmemBytes, plan, num_sms, stream, lane, col, p);
}

template <int MODE>
cudaError_t run_grouped_pair(const GroupedCall& g, GroupedParams& p, bool split3, const GroupedPlan& plan, int num_sms,
                             cudaStream_t stream) {
    using C = GroupedPairCfg;
    auto kernel = grouped_pair_kernel<MODE>;
    cudaError_t e = allow_shared<grouped_pair_kernel<MODE>>(C::kSmemBytes);
    int dev = 0;
    if (e == cudaSuccess) e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<int> max_clusters[64];  // by device; 0: not asked yet
    int clusters = dev < 64 ? max_clusters[dev].load() : 0;
    if (!clusters) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.gridDim = dim3(num_sms / 2 * 2, 1, 1);
        cfg.blockDim = dim3(C::kThreads, 1, 1);
        cfg.dynamicSmemBytes = C::kSmemBytes;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
            cudaGetLastError();
            clusters = num_sms / 2;
        }
        if (dev < 64) max_clusters[dev].store(clusters);
    }
    CUtensorMap lane, col;
    if (!grouped_maps<MODE>(g, !split3, &lane, &col)) return cudaErrorInvalidValue;
    const int pairs = static_cast<int>(std::min<long long>(plan.tiles, clusters));
    return launch_early(kernel, dim3(2 * pairs), dim3(C::kThreads), C::kSmemBytes, stream, 1, lane, col, p);
}

template <int MODE>
cudaError_t run_grouped_mode(const GroupedCall& g, GroupedParams& p, bool split3, int num_sms, cudaStream_t stream) {
    const GroupedPlan plan = plan_grouped(MODE, g.rows, g.groups, g.N, g.K, num_sms);
    p.lane_tiles = (p.lane_dim + plan.lanes - 1) / plan.lanes;
    if (plan.pair) {
        // (TF32 mode: the staged dY is rounded; the bias gradient is summed from memory.)
        p.dbias = split3 ? g.dbias : nullptr;
        return run_grouped_pair<MODE>(g, p, split3, plan, num_sms, stream);
    }
    if constexpr (MODE == kGradB) {
        return run_grouped_grad_b(g, p, split3, plan, num_sms, stream);
    } else {
        return run_grouped_few<MODE>(g, p, split3, plan, num_sms, stream);
    }
}

int grouped_gemm(const char* fn, GpuCtx* ctx, const GroupedCall& g, const mxb_ep_step* steps, int n_steps,
                 int precision, void* stream) {
    const bool grad_b = g.mode == kGradB;
    const int x_cols = g.mode == kGradA ? g.N : g.K, out_cols = g.mode == kGradA ? g.K : g.N;
    if (!ctx || !g.offsets || g.groups < 1 || g.groups > MXB_MAX_GROUPS || g.rows < 0 || g.N < 1 || g.K < 1 ||
        g.ldx < x_cols || g.ldw < g.N || g.ldo < out_cols || n_steps < 0 || n_steps > MXB_MAX_EPILOGUE ||
        (n_steps > 0 && !steps) || (precision != GPU_PRECISION_TF32 && precision != GPU_PRECISION_3XTF32) ||
        ((g.rows > 0 || grad_b) && !g.out) || (g.rows > 0 && (!g.x || !g.w))) {
        set_error("%s: invalid arguments", fn);
        return MXB_E_ARG;
    }
    if (g.groups > 1 && ((!grad_b && g.w_stride < (g.K - 1) * g.ldw + g.N) ||
                         (grad_b && g.out_stride < (g.K - 1) * g.ldo + g.N))) {
        set_error("%s: the groups' matrices overlap", fn);
        return MXB_E_ARG;
    }
    if (g.ldx % 4 || g.ldw % 4 || (!grad_b && g.groups > 1 && g.w_stride % 4) || !aligned16(g.x) || !aligned16(g.w)) {
        set_error("%s: the operands need 16-byte aligned bases, pitches and group strides (multiples of 4)", fn);
        return MXB_E_ARG;
    }
    if (g.rows > kMaxExtent || g.N > kMaxExtent || g.K > kMaxExtent) {
        set_error("%s: rows, N and K are limited to 2^30", fn);
        return MXB_E_UNSUPPORTED;
    }
    GroupedParams p{};
    if (!take_cell_steps(fn, steps, n_steps, out_cols, true, p.epi)) return MXB_E_ARG;
    if (g.rows == 0 && !grad_b) return MXB_OK;
    p.offsets = g.offsets;
    p.groups = g.groups;
    p.rows = g.rows;
    p.out = g.out;
    p.ldo = g.ldo;
    p.out_stride = g.out_stride;
    p.lane_dim = out_cols;
    p.col_dim = g.K;
    p.sum_dim = x_cols;
    p.split3 = precision == GPU_PRECISION_3XTF32;
    p.timeout_ns = ctx->timeout_ns;
    p.err = ctx->d_err;
    DeviceScope scope(ctx->device);
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    if (g.rows == 0) {  // grad_b without a row: every gradient is zero
        for (int e = 0; e < g.groups; ++e)
            if (!cuda_ok(cudaMemset2DAsync(g.out + e * g.out_stride, g.ldo * 4, 0, static_cast<size_t>(g.N) * 4, g.K, st),
                         "gradient clear"))
                return MXB_E_CUDA;
        if (g.dbias && !cuda_ok(cudaMemsetAsync(g.dbias, 0, static_cast<size_t>(g.groups) * g.N * 4, st), "gradient clear"))
            return MXB_E_CUDA;
        return MXB_OK;
    }
    const cudaError_t e = g.mode == kForward ? run_grouped_mode<kForward>(g, p, p.split3, ctx->num_sms, st)
                          : g.mode == kGradA ? run_grouped_mode<kGradA>(g, p, p.split3, ctx->num_sms, st)
                                             : run_grouped_mode<kGradB>(g, p, p.split3, ctx->num_sms, st);
    if (!cuda_ok(e, "grouped product launch")) return MXB_E_CUDA;
    if (g.dbias && !p.dbias) {
        grouped_column_sums<<<dim3((g.N + 31) / 32, g.groups), dim3(32, 32), 0, st>>>(g.w, g.ldw, g.offsets, g.rows, g.N,
                                                                                     g.dbias);
        note_launch();
        if (!cuda_ok(cudaGetLastError(), "bias gradient launch")) return MXB_E_CUDA;
    }
    return MXB_OK;
}

}  // namespace
}  // namespace mxb

extern "C" {

int mxb_grouped_plan_for(int product, int rows, int groups, int N, int K, int num_sms, mxb_gemm_plan* plan) {
    if (!plan || product < MXB_GROUPED_FORWARD || product > MXB_GROUPED_GRAD_B || rows < 1 || groups < 1 ||
        groups > MXB_MAX_GROUPS || N < 1 || K < 1 || rows > mxb::kMaxExtent || N > mxb::kMaxExtent || K > mxb::kMaxExtent ||
        num_sms < 2) {
        mxb::set_error("mxb_grouped_plan_for: invalid arguments");
        return MXB_E_ARG;
    }
    const mxb::GroupedPlan p = mxb::plan_grouped(product, rows, groups, N, K, num_sms);
    memset(plan, 0, sizeof(*plan));
    plan->kernel = p.pair ? MXB_KERNEL_CTA_PAIR : MXB_KERNEL_SINGLE_CTA;
    plan->tile_rows = p.cols;
    plan->tile_cols = p.lanes;
    plan->k_splits = p.pair ? 1 : p.cluster;
    plan->products = groups;
    return MXB_OK;
}

int mxb_grouped_gemm(GpuCtx* ctx, const float* A, long long lda, const float* B, long long ldb, long long b_stride,
                     const int* offsets, int groups, float* out, long long ldo, int rows, int N, int K,
                     const mxb_ep_step* steps, int n_steps, int precision, void* stream) {
    try {
        const mxb::GroupedCall g{mxb::kForward, A, lda, B, ldb, b_stride, offsets, groups, rows, out, ldo, 0, nullptr, N, K};
        return mxb::grouped_gemm("mxb_grouped_gemm", ctx, g, steps, n_steps, precision, stream);
    } catch (const std::exception& e) {  // host allocations of the tensor-map cache
        mxb::set_error("mxb_grouped_gemm: %s", e.what());
        return MXB_E_NOMEM;
    }
}

int mxb_grouped_gemm_grad_a(GpuCtx* ctx, const float* dY, long long lddy, const float* B, long long ldb,
                            long long b_stride, const int* offsets, int groups, float* dA, long long ldda, int rows,
                            int N, int K, const mxb_ep_step* steps, int n_steps, int precision, void* stream) {
    try {
        const mxb::GroupedCall g{mxb::kGradA, dY, lddy, B, ldb, b_stride, offsets, groups, rows, dA, ldda, 0, nullptr, N, K};
        return mxb::grouped_gemm("mxb_grouped_gemm_grad_a", ctx, g, steps, n_steps, precision, stream);
    } catch (const std::exception& e) {
        mxb::set_error("mxb_grouped_gemm_grad_a: %s", e.what());
        return MXB_E_NOMEM;
    }
}

int mxb_grouped_gemm_grad_b(GpuCtx* ctx, const float* A, long long lda, const float* dY, long long lddy,
                            const int* offsets, int groups, float* dB, long long lddb, long long db_stride,
                            float* dbias, int rows, int N, int K, int precision, void* stream) {
    try {
        const mxb::GroupedCall g{mxb::kGradB, A, lda, dY, lddy, 0, offsets, groups, rows, dB, lddb, db_stride, dbias, N, K};
        return mxb::grouped_gemm("mxb_grouped_gemm_grad_b", ctx, g, nullptr, 0, precision, stream);
    } catch (const std::exception& e) {
        mxb::set_error("mxb_grouped_gemm_grad_b: %s", e.what());
        return MXB_E_NOMEM;
    }
}

}  // extern "C"
