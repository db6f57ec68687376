// fz_int8_linear.cu -- the linear layer on int8 rows (zf_int8_linear): output = scales x weight_scales x (codes
// weight_codes^T) + bias, the integer products summed exactly on the tcgen05 tensor cores (kind::i8, 32-bit
// accumulators in tensor memory).
//
// A persistent kernel walks over tiles of 128 rows x bn outputs (bn <= 256), one CTA per SM, or (kPair) of 256 rows, a
// cluster of two CTAs per tile whose MMAs (cta_group::2) read both CTAs' shared memory: each CTA holds 128 rows and half
// of the outputs' weights, so a tile's weights are fetched once for 256 rows. Warp 0 (one lane) brings 128-byte K-blocks
// of both operands into a ring by TMA tensor copies (128-byte swizzle, K-major, no multicast; columns past `in` and rows
// past the operands arrive as zeros), warp 1 (one lane, of the pair's first CTA) issues the MMAs, warps 2-17 run the
// epilogue of the CTA's own 128 rows. Tensor memory holds two accumulators, so the epilogue of a tile runs under the MMAs
// of the next.
//
// The epilogue reads accumulators in the 16x256b shape, in which a lane holds two neighbouring columns of every eight: the
// weight scales and biases of its 16 columns stay in registers over the tiles of a column block. (With a row per lane
// every column's scale and bias came from shared memory, and those reads were what bound the kernel.) bf16 rows go
// through a staging tile per warp (stmatrix, 128-byte swizzle) and leave by TMA store when the output lies on the 16-byte
// grid; fp32 pairs are stored as they are, 32-byte sectors at a time. Outputs off the grid whose rows lie back to back
// (kFlat: an odd width, all outputs in one tile) form one sequence: the four warps of 32 rows stage them together, and one
// bulk copy writes them, whose start is on the grid again (32 rows). Any other layout is written 32 columns at a time.
//
// Measured on one B200: 2,097,152 x 256 -> 256 bf16 with bias and ReLU 0.27 ms, 6.0 TB/s of the 6.5 that a copy moves
// (floor 0.25 ms); 8,192 x 4,096 -> 4,096 0.099 ms, 2.8 PFLOP/s, or 0.120 ms sustained under the power cap; the tensor pipe
// is busy 64 % of the time there, and longer ring stages (two K-blocks per commit) measured the same. Up to 16 rows take
// fz_int8_linear_few_kernel, whose bound is the weights' bytes and the launch: 1 row 1,024 -> 1,024 2.0 us against 7.5 in
// tiles, 16 rows 4,096 -> 4,096 11.1 against 17.1.
//
// Every wait is bounded: a wait that runs out raises the CTA's abort flag, which ends every role's loop (the other CTA of
// a pair runs out on its own); the CTA then waits (bounded) for its own copies and MMAs in flight, frees its tensor
// memory and sets *status.
#include "zf_int8.h"
#include "fz_status.h"
#include "fz_launch.h"
#include "fz_pair.cuh"
#include "fz_tcgen05.cuh"
#include "fz_tma.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <cstdint>

namespace zf::int8_linear {

using namespace zf::nerf_mlp;  // the tcgen05 building blocks

constexpr int kBlockK = 128;                 // bytes of K per ring stage: the swizzle's width
constexpr int kMaxN = 256;                   // outputs of a tile at the most
constexpr int kEpilogueWarps = 16;           // four groups of four warps; a group covers the 128 accumulator lanes
constexpr int kGroups = kEpilogueWarps / 4;
constexpr int kFirstEpilogueWarp = 2;
constexpr int kThreads = 32 * (kFirstEpilogueWarp + kEpilogueWarps);
constexpr int kMaxStages = 8;
constexpr int kOperandABytes = kTileRows * kBlockK;
constexpr int kStagingBytes = 32 * 128;      // a warp's 32 rows x 64 bf16 columns
constexpr int kStagingOffset = 1024;         // behind the barriers
constexpr int kRingOffset = kStagingOffset + kEpilogueWarps * kStagingBytes;
constexpr int kMaxSmem = 227 * 1024;
constexpr uint32_t kTmemColumns = 512;       // two accumulators of 256 columns
static_assert(kRingOffset % 1024 == 0, "the swizzled ring starts on a 1024-byte boundary");

struct Args {
    CUtensorMap x_map;       // codes [n, in], boxes of x_rows x 128
    CUtensorMap w_map;       // weight codes [out, in], boxes of w_rows x 128
    CUtensorMap out_map;     // bf16 output [n, out], boxes of 32 x 64 (vector)
    const float* scales;
    const float* weight_scales;
    const float* bias;
    int n, in, out;
    int bn, x_rows, w_rows;  // outputs of a tile; operand rows that one CTA loads
    int tiles_n;
    int tiles;
    int stages, stage_bytes, ring_offset;
    int flat_bytes;          // kFlat: staging of 32 rows
    bool vector;             // output rows on the 16-byte grid
    void* output;
    int64_t output_stride;
    int* status;
};

// instruction descriptor of kind::i8: 32-bit integer accumulator (bits 4-5 = 2), signed 8-bit A and B (bits 7-9, 10-12 =
// 1), both K-major, N / 8 in bits 17-22, M / 16 in bits 24-28
__device__ __forceinline__ uint32_t int8_descriptor(const int m, const int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <bool kPair>
__device__ __forceinline__ void mma_int8(const uint32_t d_tmem, const uint64_t a, const uint64_t b, const uint32_t idesc, const uint32_t accumulate) {
    if constexpr (kPair) {
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    }
    else {
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    }
}

// the MMAs issued so far arrive on the barrier when they are done; of a pair, on both CTAs' barriers at this offset
template <bool kPair>
__device__ __forceinline__ void commit_to(const uint32_t bar) {
    if constexpr (kPair) commit_pair(bar);
    else commit(bar);
}

// a copy of a pair: into this CTA's shared memory, counted on the first CTA's barrier
__device__ __forceinline__ void tma_load_2d_pair(const uint32_t dst, const CUtensorMap* map, const int x, const int y, const uint32_t first_cta_bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(first_cta_bar)
                 : "memory");
}

// 16 accumulator lanes x 32 columns: of block i of 8 columns, words 4 i, 4 i + 1 are columns 2 (lane % 4), + 1 of row
// lane / 4, words 4 i + 2, 4 i + 3 the same columns of row lane / 4 + 8 (no wait)
__device__ __forceinline__ void load_16x256(const uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// four 8 x 8 matrices of 16-bit elements; lane l gives the address of row l % 8 of matrix l / 8 and holds columns
// 2 (l % 4), + 1 of row l / 4 of each
__device__ __forceinline__ void store_matrices(const uint32_t address, const uint32_t m0, const uint32_t m1, const uint32_t m2, const uint32_t m3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(m0), "r"(m1), "r"(m2), "r"(m3) : "memory");
}

// the larger of v and 0; a NaN stays one
__device__ __forceinline__ float relu(const float v) {
    float out;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(out) : "f"(v));
    return out;
}

// the tiles of one CTA (or pair): every step-th one, outputs fastest, as tile rows m and tile columns c
struct Walk {
    int tile, m, c;
    int step, step_m, step_c;

    __device__ __forceinline__ Walk(const int first, const int step_, const int tiles_n)
        : tile(first), m(first / tiles_n), c(first % tiles_n), step(step_), step_m(step_ / tiles_n), step_c(step_ % tiles_n) {}
    __device__ __forceinline__ void next(const int tiles_n) {
        tile += step;
        m += step_m;
        c += step_c;
        if (c >= tiles_n) c -= tiles_n, m++;
    }
};

// kRelu: each output's ReLU, in the conversion for bf16
template <typename Out, bool kRelu, bool kPair, bool kFlat>
__global__ void __launch_bounds__(kThreads, 1) fz_int8_linear_kernel(const __grid_constant__ Args a) {
    constexpr int kChunk = 128 / static_cast<int>(sizeof(Out));  // neighbouring columns of one warp
    constexpr int kCtas = kPair ? 2 : 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + 516);
    const uint32_t bar0 = smem_address(bars);
    auto full_bar = [&](const uint32_t i) { return bar0 + 8u * i; };
    auto empty_bar = [&](const uint32_t i) { return bar0 + 8u * (kMaxStages + i); };
    auto acc_full = [&](const uint32_t i) { return bar0 + 8u * (2 * kMaxStages + i); };
    auto acc_empty = [&](const uint32_t i) { return bar0 + 8u * (2 * kMaxStages + 2 + i); };
    const uint32_t drain_bar = bar0 + 8u * (2 * kMaxStages + 4);
    auto staged_bar = [&](const uint32_t i) { return bar0 + 8u * (2 * kMaxStages + 5 + i); };    // kFlat, per 32 rows: staged by four warps
    auto reusable_bar = [&](const uint32_t i) { return bar0 + 8u * (2 * kMaxStages + 9 + i); };  // and read by the copy
    const uint32_t ring = smem_address(smem) + a.ring_offset;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = kPair ? blockIdx.x % 2 : 0;
    const int first_tile = blockIdx.x / kCtas, tile_step = gridDim.x / kCtas;
    const int k_blocks = (a.in + kBlockK - 1) / kBlockK;
    const uint32_t stages = static_cast<uint32_t>(a.stages);

    if (warp == 1) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(kTmemColumns));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        }
        else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(kTmemColumns));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxStages; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full_bar(i)), "r"(1));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty_bar(i)), "r"(1));
        }
        for (int i = 0; i < 2; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(acc_full(i)), "r"(1));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(acc_empty(i)), "r"(kCtas * kEpilogueWarps));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(drain_bar), "r"(1));
        for (int i = 0; i < 4; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(staged_bar(i)), "r"(kGroups));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(reusable_bar(i)), "r"(1));
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort = 0;
    }
    fence_before_sync();
    __syncthreads();
    if constexpr (kPair) sync_cluster();  // the other CTA's barriers are ready for remote arrivals
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.x_map)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.w_map)) : "memory");
            const uint32_t bytes = static_cast<uint32_t>(kCtas * (a.x_rows + a.w_rows) * kBlockK);
            uint32_t stage = 0, round = 0;
            bool ok = true;
            for (Walk walk(first_tile, tile_step, a.tiles_n); walk.tile < a.tiles && ok; walk.next(a.tiles_n)) {
                const int row = walk.m * (kCtas * kTileRows) + rank * kTileRows, column = walk.c * a.bn + rank * a.w_rows;
                for (int k = 0; k < k_blocks; k++) {
                    // of a pair, the first CTA's MMAs have read the slot in both CTAs, so its barrier's last phase is over
                    if (round > 0 && !(ok = wait_phase(empty_bar(stage), (round - 1) & 1u, abort))) break;
                    const uint32_t at = ring + stage * a.stage_bytes;
                    if (rank == 0) expect_bytes(full_bar(stage), bytes);
                    if constexpr (kPair) {
                        const uint32_t bar = of_first_cta(full_bar(stage));
                        tma_load_2d_pair(at, &a.x_map, k * kBlockK, row, bar);
                        tma_load_2d_pair(at + kOperandABytes, &a.w_map, k * kBlockK, column, bar);
                    }
                    else {
                        tma_load_2d(at, &a.x_map, k * kBlockK, row, full_bar(stage));
                        tma_load_2d(at + kOperandABytes, &a.w_map, k * kBlockK, column, full_bar(stage));
                    }
                    if (++stage == stages) stage = 0, round++;
                }
            }
            // every copy issued has landed before the CTA's shared memory can go to another CTA
            if (rank == 0) {
                for (uint32_t i = 0; i < stages; i++) {
                    const uint32_t issued = round + (i < stage ? 1 : 0);
                    if (issued > 0) drain_phase(full_bar(i), (issued - 1) & 1u);
                }
            }
            else if (!ok) {
                // the first CTA may not have expected this CTA's last copies: they depend on nothing and land within
                // microseconds (without an abort its drain above covers them)
                const uint64_t start = global_ns();
                while (global_ns() - start < 1000000) {
                }
            }
        }
    }
    else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = int8_descriptor(kCtas * kTileRows, a.bn);
            uint32_t stage = 0, round = 0, count = 0;
            bool ok = true;
            for (int tile = first_tile; tile < a.tiles && ok; tile += tile_step, count++) {
                const uint32_t buffer = count & 1u, use = count >> 1;
                if (use > 0 && !wait_phase(acc_empty(buffer), (use - 1) & 1u, abort)) break;
                fence_after_sync();
                const uint32_t d = tmem + buffer * kMaxN;
                for (int k = 0; k < k_blocks; k++) {
                    if (!(ok = wait_phase(full_bar(stage), round & 1u, abort))) break;
                    fence_after_sync();
                    const uint32_t at = ring + stage * a.stage_bytes;
                    const int steps = min(kBlockK, a.in - k * kBlockK);
                    for (int s = 0; s < steps; s += 32) {
                        // 8-row groups 1024 bytes apart; a K step is 32 bytes further along the swizzled rows
                        mma_int8<kPair>(d, smem_descriptor(at + s, 16, 1024, 2), smem_descriptor(at + kOperandABytes + s, 16, 1024, 2), idesc, k > 0 || s > 0);
                    }
                    commit_to<kPair>(empty_bar(stage));
                    if (++stage == stages) stage = 0, round++;
                }
                if (ok) commit_to<kPair>(acc_full(buffer));
            }
        }
    }
    else {
        const int group = (warp - kFirstEpilogueWarp) / 4, quadrant = warp % 4;
        uint8_t* staging = smem + kStagingOffset + (kFlat ? quadrant * a.flat_bytes : (warp - kFirstEpilogueWarp) * kStagingBytes);
        uint32_t flat_count = 0;
        const int pair_column = 2 * (lane % 4), lane_row = lane / 4;  // of every 8 columns; of every 8 rows
        // weight scales and biases of this lane's columns: of block b of 8 columns, the chunk's for bf16 (8 blocks), the
        // two chunks' for fp32 (4 blocks each)
        float2 column_scale[8], column_bias[8];
        auto block_column = [&](const int b) { return (b / (kChunk / 8) * kGroups + group) * kChunk + b % (kChunk / 8) * 8 + pair_column; };
        int columns_of = -1;  // the first output of the tile whose scales and biases are held
        // this lane's four rows of a tile row: 8 i + lane_row; the scales of the next tile's are fetched a tile ahead
        auto row_of = [&](const int m) { return m * (kCtas * kTileRows) + rank * kTileRows + 32 * quadrant; };
        auto fetch_scales = [&](const int m, float (&out)[4]) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = row_of(m) + 8 * i + lane_row;
                out[i] = row < a.n ? __ldg(a.scales + row) : 0.0f;
            }
        };
        uint32_t count = 0;
        float next_scales[4] = {};
        Walk walk(first_tile, tile_step, a.tiles_n);
        if (walk.tile < a.tiles) fetch_scales(walk.m, next_scales);
        for (; walk.tile < a.tiles; count++) {
            const uint32_t buffer = count & 1u, use = count >> 1;
            const int row0 = row_of(walk.m), column0 = walk.c * a.bn;
            const int columns = min(a.bn, a.out - column0), rows = min(32, a.n - row0);
            float scales[4];
            #pragma unroll
            for (int i = 0; i < 4; i++) scales[i] = next_scales[i];
            walk.next(a.tiles_n);
            if (walk.tile < a.tiles) fetch_scales(walk.m, next_scales);
            if (column0 != columns_of) {
                #pragma unroll
                for (int b = 0; b < 8; b++) {
                    const int c = block_column(b);
                    column_scale[b].x = c < columns ? __ldg(a.weight_scales + column0 + c) : 0.0f;
                    column_scale[b].y = c + 1 < columns ? __ldg(a.weight_scales + column0 + c + 1) : 0.0f;
                    column_bias[b].x = a.bias != nullptr && c < columns ? __ldg(a.bias + column0 + c) : 0.0f;
                    column_bias[b].y = a.bias != nullptr && c + 1 < columns ? __ldg(a.bias + column0 + c + 1) : 0.0f;
                }
                columns_of = column0;
            }
            // warp-uniform: the tensor-memory loads below are collective
            if (!__all_sync(0xFFFFFFFFu, wait_phase(acc_full(buffer), use & 1u, abort))) break;
            fence_after_sync();
            const uint32_t acc = tmem + (static_cast<uint32_t>(32 * quadrant) << 16) + buffer * kMaxN;
            auto release = [&]() {  // the accumulator is read: the next MMAs may overwrite it
                fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (kPair) arrive_first_cta(acc_empty(buffer));
                    else arrive(acc_empty(buffer));
                }
            };
            const bool any = group * kChunk < columns && rows > 0;
            if (!any) release();
            if (kFlat && rows > 0 && flat_count > 0) {
                // the last sequence's copy has read the staging
                if (group == kGroups - 1 && lane == 0) {
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    arrive(reusable_bar(quadrant));
                }
                if (!__all_sync(0xFFFFFFFFu, wait_phase(reusable_bar(quadrant), (flat_count - 1) & 1u, abort))) break;
            }
            if (!kFlat && sizeof(Out) == 2 && any) {
                // the staging tile's last store has been read
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
            }
            #pragma unroll
            for (int i = 0; i < 64 / kChunk; i++) {
                const int c = (i * kGroups + group) * kChunk;
                if (c >= columns || rows <= 0) break;
                const bool last = c + kGroups * kChunk >= columns;
                #pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t words[kChunk / 8][4];
                    #pragma unroll
                    for (int b = 0; b < kChunk / 8; b += 4) load_16x256(acc + (static_cast<uint32_t>(16 * half) << 16) + c + 8 * b, &words[b][0]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (last && half == 1) release();
                    #pragma unroll
                    for (int b = 0; b < kChunk / 8; b++) {
                        #pragma unroll
                        for (int e = 0; e < 4; e += 2) {  // rows 16 half + 8 (e / 2) + lane_row
                            const float s = scales[2 * half + e / 2];
                            const float2 w = column_scale[i * (kChunk / 8) + b], bias = column_bias[i * (kChunk / 8) + b];
                            const float x = fmaf(static_cast<float>(static_cast<int>(words[b][e])) * s, w.x, bias.x);
                            const float y = fmaf(static_cast<float>(static_cast<int>(words[b][e + 1])) * s, w.y, bias.y);
                            if constexpr (kFlat) {
                                const int r = 16 * half + 4 * e + lane_row, at = c + 8 * b + pair_column;
                                Out* to = reinterpret_cast<Out*>(staging) + r * a.out + at;
                                if constexpr (sizeof(Out) == 4) {
                                    if (at < columns) to[0] = kRelu ? relu(x) : x;
                                    if (at + 1 < columns) to[1] = kRelu ? relu(y) : y;
                                }
                                else {
                                    const uint32_t pair = kRelu ? pack_bf16x2_relu(x, y) : pack_bf16x2(x, y);
                                    if (at < columns) to[0] = __ushort_as_bfloat16(static_cast<uint16_t>(pair));
                                    if (at + 1 < columns) to[1] = __ushort_as_bfloat16(static_cast<uint16_t>(pair >> 16));
                                }
                            }
                            else if constexpr (sizeof(Out) == 2) words[b][e / 2] = kRelu ? pack_bf16x2_relu(x, y) : pack_bf16x2(x, y);
                            else {
                                const float u = kRelu ? relu(x) : x, v = kRelu ? relu(y) : y;
                                const int r = 16 * half + 4 * e + lane_row, at = 8 * b + pair_column;
                                if (a.vector && c + at + 1 < columns) {
                                    float* out = static_cast<float*>(a.output) + (row0 + r) * a.output_stride + column0 + c + at;
                                    if (r < rows) *reinterpret_cast<float2*>(out) = make_float2(u, v);
                                }
                                else {
                                    // 16-byte piece p of row r at place p ^ (r & 7), as the bf16 rows
                                    *reinterpret_cast<float2*>(staging + r * 128 + (((at / 4) ^ (r & 7)) << 4) + at % 4 * 4) = make_float2(u, v);
                                }
                            }
                        }
                    }
                    if (!kFlat && sizeof(Out) == 4 && half == 1 && !(a.vector && c + kChunk <= columns)) {
                        // rows off the 16-byte grid, or their last columns: 32 neighbouring columns of a row per store
                        __syncwarp();
                        const int first = a.vector ? (columns - c) & ~1 : 0;  // whole pairs are stored already
                        float* out = static_cast<float*>(a.output) + row0 * a.output_stride + column0 + c;
                        #pragma unroll
                        for (int r = 0; r < 32; r += 8) {  // eight reads, then eight stores
                            float held[8];
                            #pragma unroll
                            for (int e = 0; e < 8; e++) held[e] = *reinterpret_cast<const float*>(staging + (r + e) * 128 + (((lane / 4) ^ e) << 4) + lane % 4 * 4);
                            #pragma unroll
                            for (int e = 0; e < 8; e++) {
                                if (r + e < rows && lane >= first && c + lane < columns) out[(r + e) * a.output_stride + lane] = held[e];
                            }
                        }
                        __syncwarp();
                    }
                    if constexpr (!kFlat && sizeof(Out) == 2) {
                        // 8 x 8 matrices (block b, rows 0-7), (b, rows 8-15), (b + 1, ...): lane l holds the address of row
                        // l % 8 of matrix l / 8; 16-byte piece p of row r lies at place p ^ (r & 7) of its 128 bytes
                        const int r = 16 * half + lane % 16;
                        #pragma unroll
                        for (int b = 0; b < kChunk / 8; b += 2) {
                            store_matrices(smem_address(staging) + r * 128 + (((b + lane / 16) ^ (r & 7)) << 4), words[b][0], words[b][1], words[b + 1][0],
                                           words[b + 1][1]);
                        }
                    }
                }
            }
            if (kFlat && rows > 0) {
                fence_async_shared();
                __syncwarp();
                if (lane == 0) arrive(staged_bar(quadrant));
                if (group == kGroups - 1) {
                    if (!__all_sync(0xFFFFFFFFu, wait_phase(staged_bar(quadrant), flat_count & 1u, abort))) break;
                    if (lane == 0) {
                        const uint32_t bytes = static_cast<uint32_t>(rows * a.out) * sizeof(Out), whole = bytes & ~15u;
                        uint8_t* to = static_cast<uint8_t*>(a.output) + static_cast<int64_t>(row0) * a.out * sizeof(Out);
                        if (whole > 0) {  // a few rows of a narrow output may be less than the copy's 16 bytes
                            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(smem_address(staging)), "r"(whole) : "memory");
                        }
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        // the last rows' last elements
                        for (uint32_t e = whole; e < bytes; e += sizeof(Out)) *reinterpret_cast<Out*>(to + e) = *reinterpret_cast<const Out*>(staging + e);
                    }
                    __syncwarp();
                }
                flat_count++;
            }
            if (!kFlat && sizeof(Out) == 2 && any) {
                const int c = group * kChunk;
                if (a.vector) {
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        // rows past n and columns past out are not written; bn is a multiple of 64 where a tile borders on another
                        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                                         reinterpret_cast<uint64_t>(&a.out_map)),
                                     "r"(column0 + c), "r"(row0), "r"(smem_address(staging))
                                     : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
                else {
                    __syncwarp();
                    const int width = min(kChunk, columns - c);
                    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.output) + row0 * a.output_stride + column0 + c;
                    #pragma unroll
                    for (int r = 0; r < 32; r += 8) {  // 32 neighbouring columns of a row per store; eight rows' reads, then their stores
                        #pragma unroll
                        for (int h = 0; h < kChunk; h += 32) {
                            __nv_bfloat16 held[8];
                            #pragma unroll
                            for (int e = 0; e < 8; e++) {
                                held[e] = *reinterpret_cast<const __nv_bfloat16*>(staging + (r + e) * 128 + ((((h + lane) / 8) ^ e) << 4) + lane % 8 * 2);
                            }
                            #pragma unroll
                            for (int e = 0; e < 8; e++) {
                                if (r + e < rows && h + lane < width) out[(r + e) * a.output_stride + h + lane] = held[e];
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if ((kFlat || sizeof(Out) == 2) && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    // teardown: every role has left its loop; the MMAs already issued finish before the tensor memory is freed
    fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 32 && rank == 0) {
        if constexpr (kPair) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_bar) : "memory");
        else commit(drain_bar);
        drain_phase(drain_bar, 0);
    }
    if (threadIdx.x == 0 && *abort) atomicExch(a.status, kWaitTimeout);
    fence_before_sync();
    __syncthreads();
    if constexpr (kPair) sync_cluster();  // no MMA, copy or arrival reaches this CTA any more
    fence_after_sync();
    if (warp == 1) {
        if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
    }
}

// A few rows (kRows at the most): bound by the weights' bytes and by latency, so no tiles: a warp takes kOutputs outputs,
// its lanes 16 codes of each at a time, and multiplies them with the same codes of every row (dp4a, exact); one
// integer reduction over the warp per output and row.
constexpr int kFewBlock = 128;
constexpr int kFewRows = 16;

struct FewArgs {
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    const int8_t* weight;
    int64_t weight_stride;
    const float* weight_scales;
    const float* bias;
    int n, in, out;
    bool relu;
    void* output;
    int64_t output_stride;
};

template <typename Out, int kRows, int kOutputs>
__global__ void __launch_bounds__(kFewBlock) fz_int8_linear_few_kernel(const FewArgs a) {
    const int lane = threadIdx.x % 32;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * (kFewBlock / 32) + threadIdx.x / 32) * kOutputs;
    if (first >= a.out) return;
    const int outputs = static_cast<int>(min(static_cast<int64_t>(kOutputs), a.out - first));
    int sums[kOutputs][kRows] = {};
    // outputs and rows past the last repeat it: their sums are not used
    const int8_t* w[kOutputs];
    #pragma unroll
    for (int o = 0; o < kOutputs; o++) w[o] = a.weight + (first + min(o, outputs - 1)) * a.weight_stride;
    const int whole = a.in & ~15;
    #pragma unroll 2
    for (int k = 16 * lane; k < whole; k += 512) {
        uint4 wv[kOutputs];
        #pragma unroll
        for (int o = 0; o < kOutputs; o++) wv[o] = __ldg(reinterpret_cast<const uint4*>(w[o] + k));
        #pragma unroll
        for (int r = 0; r < kRows; r++) {
            const uint4 xv = __ldg(reinterpret_cast<const uint4*>(a.codes + min(r, a.n - 1) * a.codes_stride + k));
            #pragma unroll
            for (int o = 0; o < kOutputs; o++) {
                int sum = __dp4a(static_cast<int>(xv.x), static_cast<int>(wv[o].x), sums[o][r]);
                sum = __dp4a(static_cast<int>(xv.y), static_cast<int>(wv[o].y), sum);
                sum = __dp4a(static_cast<int>(xv.z), static_cast<int>(wv[o].z), sum);
                sums[o][r] = __dp4a(static_cast<int>(xv.w), static_cast<int>(wv[o].w), sum);
            }
        }
    }
    if (whole + lane < a.in) {  // the last codes, one per lane
        #pragma unroll
        for (int r = 0; r < kRows; r++) {
            const int x = a.codes[min(r, a.n - 1) * a.codes_stride + whole + lane];
            #pragma unroll
            for (int o = 0; o < kOutputs; o++) sums[o][r] += x * w[o][whole + lane];
        }
    }
    // lane l finishes sums l, l + 32, ... (row-major over rows and outputs)
    constexpr int kSums = kOutputs * kRows;
    #pragma unroll
    for (int i = 0; i < kSums; i += 32) {
        int mine = 0;
        #pragma unroll
        for (int j = i; j < kSums && j < i + 32; j++) {
            const int sum = __reduce_add_sync(0xFFFFFFFFu, sums[j % kOutputs][j / kOutputs]);
            if (lane == j - i) mine = sum;
        }
        const int r = (i + lane) / kOutputs, o = (i + lane) % kOutputs;
        if (i + lane < kSums && r < a.n && o < outputs) {
            const float s = __ldg(a.scales + r), ws = __ldg(a.weight_scales + first + o);
            float v = fmaf(static_cast<float>(mine) * s, ws, a.bias != nullptr ? __ldg(a.bias + first + o) : 0.0f);
            if (a.relu) v = relu(v);
            static_cast<Out*>(a.output)[r * a.output_stride + first + o] = static_cast<Out>(v);
        }
    }
}

template <typename Out>
cudaError_t launch_few(const FewArgs& a, cudaStream_t stream) {
    auto run = [&](auto rows, auto outputs) {
        constexpr int kRows = decltype(rows)::value, kOutputs = decltype(outputs)::value;
        constexpr int kPerBlock = kFewBlock / 32 * kOutputs;
        const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(a.out) + kPerBlock - 1) / kPerBlock);
        fz_int8_linear_few_kernel<Out, kRows, kOutputs><<<blocks, kFewBlock, 0, stream>>>(a);
    };
    using std::integral_constant;
    if (a.n == 1) run(integral_constant<int, 1>{}, integral_constant<int, 2>{});
    else if (a.n == 2) run(integral_constant<int, 2>{}, integral_constant<int, 2>{});
    else if (a.n <= 4) run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else if (a.n <= 8) run(integral_constant<int, 8>{}, integral_constant<int, 2>{});
    else run(integral_constant<int, 16>{}, integral_constant<int, 2>{});
    return cudaGetLastError();
}

// the tensor map of code rows [rows, columns], boxes of box_rows rows x 128 bytes with the 128-byte swizzle
bool encode_codes(CUtensorMap* map, const int8_t* codes, const int64_t columns, const int64_t stride, const int64_t rows, const int box_rows) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = zf::tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
    const cuuint32_t box[2] = {kBlockK, static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(codes), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// the tensor map of the bf16 output [n, out], boxes of 32 rows x 64 columns with the 128-byte swizzle
bool encode_output(CUtensorMap* map, void* output, const int64_t out, const int64_t stride, const int64_t n) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = zf::tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(out), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
    const cuuint32_t box[2] = {64, 32};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, output, dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int round_up(const int v, const int to) { return (v + to - 1) / to * to; }

template <typename Out, bool kRelu, bool kPair, bool kFlat>
cudaError_t launch_kernel(const Args& a, const int n_sms, cudaStream_t stream) {
    const auto kernel = fz_int8_linear_kernel<Out, kRelu, kPair, kFlat>;
    const cudaError_t error = zf::allow_shared_memory<fz_int8_linear_kernel<Out, kRelu, kPair, kFlat>>(kMaxSmem);
    if (error != cudaSuccess) return error;
    constexpr int kCtas = kPair ? 2 : 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(kCtas * static_cast<unsigned>(std::min(a.tiles, n_sms / kCtas)));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = a.ring_offset + a.stages * a.stage_bytes;
    config.stream = stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = kCtas;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = kPair ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, a);
}

template <typename Out, bool kRelu>
cudaError_t launch(const Args& a, const bool pair, const int n_sms, cudaStream_t stream) {
    if (a.flat_bytes > 0) return pair ? launch_kernel<Out, kRelu, true, true>(a, n_sms, stream) : launch_kernel<Out, kRelu, false, true>(a, n_sms, stream);
    return pair ? launch_kernel<Out, kRelu, true, false>(a, n_sms, stream) : launch_kernel<Out, kRelu, false, false>(a, n_sms, stream);
}

int invalid(const char* message) { return zf::set_error(ZF_ERROR_INVALID_ARGUMENT, message); }

bool valid_codes(const void* codes, const int64_t stride, const int64_t d) {
    return codes != nullptr && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && stride % 16 == 0 && stride >= d;
}

}  // namespace zf::int8_linear

int zf_int8_linear(const zf_int8_linear_args* args, cudaStream_t stream) {
    using namespace zf::int8_linear;
    constexpr int64_t kMost = (int64_t{1} << 31) - 256;
    if (args == nullptr || args->n < 0 || args->in <= 0 || args->out <= 0 || args->n >= kMost || args->out >= kMost) return invalid("int8_linear: invalid sizes");
    if (args->in > 131071) return invalid("int8_linear: more than 131071 inputs could overflow the 32-bit sums");
    if (args->n == 0) return ZF_OK;
    if (!valid_codes(args->codes, args->codes_stride, args->in) || !valid_codes(args->weight_codes, args->weight_stride, args->in)) {
        return invalid("int8_linear: codes must be 16-byte aligned with a row stride that is a multiple of 16");
    }
    if (args->scales == nullptr || args->weight_scales == nullptr || args->status == nullptr) return invalid("int8_linear: scales and status must be given");
    if (!zf::aligned_as<float>(args->scales, args->weight_scales, args->bias, args->status)) return invalid("int8_linear: misaligned scales, bias or status");
    const int size = args->output_dtype == ZF_FLOAT32 ? 4 : 2;
    if ((args->output_dtype != ZF_FLOAT32 && args->output_dtype != ZF_BFLOAT16) || args->output == nullptr || args->output_stride < args->out
        || reinterpret_cast<uintptr_t>(args->output) % size != 0) {
        return invalid("int8_linear: invalid output");
    }
    cudaError_t error;
    if (args->n <= kFewRows) {
        const FewArgs f{args->codes, args->codes_stride, args->scales, args->weight_codes, args->weight_stride, args->weight_scales, args->bias,
                        static_cast<int>(args->n), static_cast<int>(args->in), static_cast<int>(args->out), args->relu != 0, args->output, args->output_stride};
        error = args->output_dtype == ZF_FLOAT32 ? launch_few<float>(f, stream) : launch_few<__nv_bfloat16>(f, stream);
        return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, "int8_linear");
    }
    int n_sms = 0;
    error = zf::current_multiprocessors(&n_sms);
    if (error != cudaSuccess) return zf::set_cuda_error(error, "device query");
    Args a{};
    a.scales = args->scales;
    a.weight_scales = args->weight_scales;
    a.bias = args->bias;
    a.n = static_cast<int>(args->n);
    a.in = static_cast<int>(args->in);
    a.out = static_cast<int>(args->out);
    // more than one tile's rows: pairs of CTAs
    const bool pair = a.n > kTileRows;
    const int tile_rows = pair ? 2 * kTileRows : kTileRows;
    // the outputs in equal shares of at most 256: multiples of 32 for the MMAs, of 64 where a tile borders on another (the
    // width of a bf16 store); halved while twice the tiles still find a multiprocessor each
    const int64_t tiles_m = (a.n + tile_rows - 1) / tile_rows;
    int shares = (a.out + kMaxN - 1) / kMaxN;
    while (tiles_m * shares * 2 <= (pair ? n_sms / 2 : n_sms) && a.out > 64 * shares) shares *= 2;
    a.bn = round_up((a.out + shares - 1) / shares, shares > 1 ? 64 : 32);
    a.x_rows = std::min(a.n, kTileRows);
    a.w_rows = pair ? a.bn / 2 : a.bn;
    a.tiles_n = (a.out + a.bn - 1) / a.bn;
    const int64_t tiles = tiles_m * a.tiles_n;
    if (tiles > (1 << 30)) return invalid("int8_linear: invalid sizes");
    a.tiles = static_cast<int>(tiles);
    a.stage_bytes = round_up(kOperandABytes + a.w_rows * kBlockK, 1024);
    const bool aligned = reinterpret_cast<uintptr_t>(args->output) % 16 == 0;
    a.vector = aligned && args->output_stride * size % 16 == 0;
    a.flat_bytes = !a.vector && aligned && args->output_stride == args->out && a.tiles_n == 1 ? round_up(32 * a.out * size, 1024) : 0;
    a.ring_offset = a.flat_bytes > 0 ? kStagingOffset + 4 * a.flat_bytes : kRingOffset;
    a.stages = std::min(kMaxStages, (kMaxSmem - a.ring_offset) / a.stage_bytes);
    a.output = args->output;
    a.output_stride = args->output_stride;
    a.status = args->status;
    if (!encode_codes(&a.x_map, args->codes, args->in, args->codes_stride, args->n, a.x_rows)
        || !encode_codes(&a.w_map, args->weight_codes, args->in, args->weight_stride, args->out, a.w_rows)) {
        return zf::set_error(ZF_ERROR_CUDA, "int8_linear: no tensor map");
    }
    if (args->output_dtype == ZF_BFLOAT16 && a.vector && !encode_output(&a.out_map, args->output, args->out, args->output_stride, args->n)) {
        return zf::set_error(ZF_ERROR_CUDA, "int8_linear: no tensor map");
    }
    const bool relu = args->relu != 0;
    if (args->output_dtype == ZF_FLOAT32) error = relu ? launch<float, true>(a, pair, n_sms, stream) : launch<float, false>(a, pair, n_sms, stream);
    else error = relu ? launch<__nv_bfloat16, true>(a, pair, n_sms, stream) : launch<__nv_bfloat16, false>(a, pair, n_sms, stream);
    return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, "int8_linear");
}
