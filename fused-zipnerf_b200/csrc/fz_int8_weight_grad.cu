// fz_int8_weight_grad.cu -- the weight and bias gradient of a linear layer from the 8-bit checkpoint of its input
// (zf_int8_weight_grad): grad_weight += grad^T (codes x scales), grad_bias += column sums of grad, on the tcgen05 tensor
// cores (kind::f16 on bf16, fp32 accumulators in tensor memory).
//
// The samples are the K dimension of this product, so both operands are MN-major. A pair of CTAs (a cluster, cta_group::2)
// takes one tile of grad_weight, up to 256 outputs x 256 inputs, and a share of the samples, 64 at a time through a ring
// of stages. Each CTA holds 128 of the outputs' gradients and half of the inputs, so that no code is read or turned into
// bf16 twice:
//   warp 0 (one lane)  brings the stage's codes and gradients by TMA tensor copies (128-byte swizzle, no multicast; rows
//                      and columns past the tensors arrive as zeros);
//   warps 2-17         turn the codes into bf16 values codes x scale, the MMAs' second operand; gradients whose rows do
//                      not lie on the 16-byte grid they bring too; they sum the bias;
//   warp 1 (one lane)  of the first CTA issues the MMAs for both;
//   warps 18-25        add the accumulators to a running sum, every kPeriod stages.
// With power-of-two scales codes x scale is a bf16 number, so both operands are exact and only the sums round. The
// accumulation in the tensor cores truncates: over one share of 14,000 samples the sums came out 1.5e-5 too small in
// magnitude (relative; 885 MMA steps). So the accumulator holds 48 MMA steps at a time (an error below 1e-6, what a plain
// fp32 product has; every 128 steps: 2.0e-6, and 4 % faster); the running sum, rounded to nearest, lies beside it in tensor
// memory (256 + 256 columns), where it needs neither registers nor shared memory.
//
// Each CTA leaves its sums in the workspace, in the order of its tensor-memory reads; the join kernel adds the shares of a
// tile in their order, so that results do not depend on timing. It is launched while the first kernel runs and waits for
// it.
//
// Measured on one B200 (2,097,152 samples, 256 -> 256, with bias): 0.33 ms, 4.9 TB/s of the 6.5 that a copy moves (0.38 to
// 0.40 ms sustained, when the power cap holds the clock at about 1.5 GHz), against a floor of 0.25 ms for the bytes. The join
// takes 0.01 ms of it. A pair's 443 stages take 1,180 cycles each (the difference of two row counts) and the launch, the first
// stages and the sums' way out another 23,000: 546,000 cycles, 0.32 ms at the 1.7 GHz that the kernel runs at. Of a stage's
// cycles 850 are the MMA thread's (four MMAs run 512) and 220 its share of the additions to the running sum; the other 110
// are not accounted for. Ring stages hold gradients and codes until the MMAs are done and values only from the workers to the
// MMAs: with all three in one slot the copies' latency showed.
//
// Bounded waits, pairs and the status as in fz_int8_linear.cu.
#include "zf_int8.h"
#include "fz_status.h"
#include "fz_grad_words.h"
#include "fz_launch.h"
#include "fz_pair.cuh"
#include "fz_tcgen05.cuh"
#include "fz_tma.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <cstdint>

namespace zf::int8_weight_grad {

using namespace zf::nerf_mlp;  // the tcgen05 building blocks

constexpr int kRows = 64;                    // samples of a stage
constexpr int kPeriod = 12;                  // stages between two additions to the running sum: 48 MMA steps
constexpr int kAtom = 64;                    // columns of a 128-byte-swizzled atom
constexpr int kAtomBytes = kRows * 128;
constexpr int kTileOut = 256;                // outputs of a tile: 128 per CTA
constexpr int kMaxTileIn = 256;              // inputs of a tile: half per CTA, whole atoms
constexpr int kGradBytes = 2 * kAtomBytes;   // a stage of one CTA: 128 columns of gradients,
constexpr int kValueBytes = 2 * kAtomBytes;  // up to 128 columns of values
constexpr int kCodeBytes = kAtomBytes;       // and their codes
constexpr int kStageBytes = kGradBytes + kCodeBytes;  // what arrives by copies
constexpr int kStages = 6;                   // enough bytes in flight for the memory's latency
constexpr int kValueSlots = 4;               // values exist only between the workers and the MMAs
constexpr int kTeam = 8;                     // warps that convert a stage
constexpr int kWorkers = 2 * kTeam;          // two teams take alternate stages: a stage's waits are longer than its work
constexpr int kFirstWorker = 2;
constexpr int kSummers = 8;                  // warps that read the accumulators
constexpr int kThreads = 32 * (kFirstWorker + kWorkers + kSummers);
constexpr int kBiasOffset = 1024;            // behind the barriers: 16 x 128 partial bias sums
constexpr int kRingOffset = kBiasOffset + kWorkers * 128 * 4;
constexpr int kValueOffset = kRingOffset + kStages * kStageBytes;
constexpr int kSmemBytes = kValueOffset + kValueSlots * kValueBytes;
constexpr uint32_t kTmemColumns = 512;       // accumulator, running sum
constexpr uint32_t kSumColumn = 256;
static_assert(kRingOffset % 1024 == 0 && kStageBytes % 1024 == 0, "the swizzled tiles start on 1024-byte boundaries");
static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM");

struct Args {
    CUtensorMap grad_map;    // grad [n, out] bf16, boxes of 64 samples x 64 columns (on the 16-byte grid)
    CUtensorMap code_map;    // codes [n, in], boxes of 64 samples x half a tile's columns
    const uint16_t* grad;
    int64_t grad_stride;
    const float* scales;
    int n, in, out;
    int tile_in;             // a multiple of 128, at most 256
    int tiles_out, tiles_in;
    int splits;
    int stages_total;        // stages over all samples
    float* partial;          // [splits][tiles][tile_in / 4][256] float4
    float* bias_partial;     // [splits][out], or null
    int* status;
};

// D (+)= A B of a pair of CTAs, both operands MN-major bf16
__device__ __forceinline__ void mma_pair(const uint32_t d_tmem, const uint64_t a, const uint64_t b, const uint32_t idesc, const uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// four codes (one word) as bf16 values code x scale, rounded once, two to a word
__device__ __forceinline__ uint2 values_of(const uint32_t word, const uint64_t scales) {
    const uint32_t biased = word ^ 0x80808080u;  // code + 128
    uint32_t out[2];
    #pragma unroll
    for (int e = 0; e < 2; e++) {
        // 2^23 + (code + 128) as floats without a conversion, then both at once: - (2^23 + 128), which is exact, x scale
        const uint32_t lo = __byte_perm(biased, 0x4B000000u, 0x7440u + 2 * e), hi = __byte_perm(biased, 0x4B000000u, 0x7441u + 2 * e);
        asm("{\n.reg .b64 v, c;\n.reg .f32 l, h;\n"
            "mov.b64 v, {%1, %2};\nmov.b64 c, {0fCB000080, 0fCB000080};\n"
            "add.rn.f32x2 v, v, c;\nmul.rn.f32x2 v, v, %3;\n"
            "mov.b64 {l, h}, v;\ncvt.rn.bf16x2.f32 %0, h, l;\n}\n"
            : "=r"(out[e])
            : "r"(lo), "r"(hi), "l"(scales));
    }
    return make_uint2(out[0], out[1]);
}

template <bool kOnGrid>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) fz_int8_weight_grad_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + 516);
    const uint32_t bar0 = smem_address(smem);
    auto landed_bar = [&](const uint32_t i) { return bar0 + 8u * i; };               // this CTA's copies of a stage
    auto empty_bar = [&](const uint32_t i) { return bar0 + 8u * (kStages + i); };    // the stage's MMAs are done
    auto full_bar = [&](const uint32_t i) { return bar0 + 8u * (2 * kStages + i); };  // first CTA: both CTAs' operands are ready
    const uint32_t sum_bar = bar0 + 8u * (2 * kStages + kValueSlots);                 // a period's MMAs are done
    const uint32_t read_bar = sum_bar + 8u;                                          // first CTA: both CTAs have read the accumulator
    const uint32_t drain_bar = read_bar + 8u;
    const uint32_t ring = bar0 + kRingOffset;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = blockIdx.x % 2, tiles = a.tiles_out * a.tiles_in;
    const int tile = blockIdx.x / 2 % tiles, split = blockIdx.x / 2 / tiles;
    const int half = a.tile_in / 2;
    const int out0 = tile / a.tiles_in * kTileOut + 128 * rank, tile_in0 = tile % a.tiles_in * a.tile_in, in0 = tile_in0 + half * rank;
    // this share's stages: split, split + splits, ...; neighbouring shares read neighbouring rows at about the same time
    const int stages = split < a.stages_total ? (a.stages_total - split - 1) / a.splits + 1 : 0;
    auto row_of = [&](const int i) { return (static_cast<int64_t>(i) * a.splits + split) * kRows; };
    const int grad_columns = max(0, min(128, a.out - out0)), grad_atoms = (grad_columns + kAtom - 1) / kAtom;
    const bool bias = a.bias_partial != nullptr && tile_in0 == 0;

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(kTmemColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(landed_bar(i)), "r"(1));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty_bar(i)), "r"(1));
        }
        for (int i = 0; i < kValueSlots; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full_bar(i)), "r"(2 * kTeam));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sum_bar), "r"(1));
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(read_bar), "r"(2 * kSummers));
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(drain_bar), "r"(1));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort = 0;
    }
    fence_before_sync();
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join's blocks may be scheduled; they wait for this grid's end
    sync_cluster();  // the other CTA's barriers are ready for remote arrivals
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.code_map)) : "memory");
            if (kOnGrid) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.grad_map)) : "memory");
            const uint32_t bytes = static_cast<uint32_t>(half * kRows + (kOnGrid ? grad_atoms * kAtomBytes : 0));
            int issued = 0;
            for (int i = 0; i < stages; i++) {
                const uint32_t slot = i % kStages;
                if (i >= kStages && !wait_phase(empty_bar(slot), (i / kStages - 1) & 1u, abort)) break;
                const uint32_t at = ring + slot * kStageBytes;
                expect_bytes(landed_bar(slot), bytes);
                if (kOnGrid) {
                    for (int g = 0; g < grad_atoms; g++) tma_load_2d(at + g * kAtomBytes, &a.grad_map, out0 + g * kAtom, static_cast<int>(row_of(i)), landed_bar(slot));
                }
                tma_load_2d(at + kGradBytes, &a.code_map, in0, static_cast<int>(row_of(i)), landed_bar(slot));
                issued = i + 1;
            }
            // every copy issued has landed before the CTA's shared memory can go to another CTA
            for (int i = issued > kStages ? issued - kStages : 0; i < issued; i++) drain_phase(landed_bar(i % kStages), (i / kStages) & 1u);
        }
    }
    else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = instr_descriptor(kTileOut, a.tile_in, true, true);
            // one thread's dependent instructions add up to a stage's time: slots, parities and descriptors are carried along
            // instead of computed from the stage (16 samples, two 8-row groups of 1024 bytes, are 128 further in a descriptor)
            const uint64_t first_grad = mn_sw128_descriptor(ring, kRows), first_values = mn_sw128_descriptor(bar0 + kValueOffset, kRows);
            uint64_t grad = first_grad, values = first_values;
            uint32_t slot = 0, value = 0, parity = 0, in_period = 0, period = 0;
            bool ready = false;
            for (int i = 0; i < stages; i++) {
                if (in_period == kPeriod) {  // a new period overwrites the accumulator
                    if (!wait_phase(read_bar, period & 1u, abort)) break;
                    period++;
                    in_period = 0;
                }
                if (!ready && !wait_phase(full_bar(value), parity, abort)) break;
                fence_after_sync();
                const uint32_t next_value = value + 1 == kValueSlots ? 0 : value + 1, next_parity = next_value == 0 ? parity ^ 1u : parity;
                mma_pair(tmem, grad, values, idesc, in_period > 0 ? 1u : 0u);
                #pragma unroll
                for (int k = 1; k < kRows / kMmaK; k++) {
                    // the next stage is asked for while this one's MMAs run
                    if (k + 1 == kRows / kMmaK) ready = i + 1 < stages && test_phase(full_bar(next_value), next_parity);
                    mma_pair(tmem, grad + 128 * k, values + 128 * k, idesc, 1u);
                }
                commit_pair(empty_bar(slot));
                if (++in_period == kPeriod || i + 1 == stages) commit_pair(sum_bar);
                value = next_value;
                parity = next_parity;
                values = value == 0 ? first_values : values + kValueBytes / 16;
                if (++slot == kStages) slot = 0;
                grad = slot == 0 ? first_grad : grad + kStageBytes / 16;
            }
        }
    }
    else if (warp < kFirstWorker + kWorkers) {
        const int team = (warp - kFirstWorker) / kTeam, w = (warp - kFirstWorker) % kTeam;
        // codes: warp w's rows are 8 w .. 8 w + 7 of a stage; lane l holds row l % 8 and the 16 codes l / 8 of each atom, so
        // that eight lanes of a shared-memory access lie in eight different places of the swizzle
        const int own_row = 8 * w + lane % 8, own_code = 16 * (lane / 8);
        // the scales of four of the team's stages at a time, four of them ahead: lane l holds row 8 w + l % 8 of the
        // (l / 8)-th
        auto scales_of = [&](const int i) {
            const int stage = i + 2 * (lane / 8);
            const int64_t row = row_of(stage) + own_row;
            return stage < stages && row < a.n ? __ldg(a.scales + row) : 0.0f;
        };
        // gradients off the grid: warp w's rows w + 8 r as the aligned 32-bit words that hold them, fetched one of the team's
        // stages ahead: lane l words l and l + 32, lane 31 word 64 too. A row that begins in the middle of a word is shifted
        // by 16 bits when it is stored; a warp's rows lie multiples of 8 rows apart, so all of them do or none.
        constexpr int kFetched = kOnGrid ? 1 : kRows / kTeam;
        uint32_t next[kFetched][3] = {};
        const int odd = static_cast<int>((reinterpret_cast<uintptr_t>(a.grad) / 2 + static_cast<uint64_t>(w) * a.grad_stride + out0) & 1);
        const bool needs[3] = {word_needed(lane, odd, grad_columns), word_needed(lane + 32, odd, grad_columns),
                               lane == 31 && word_needed(64, odd, grad_columns)};
        auto fetch = [&](const int i) {
            if (i >= stages) return;
            const int64_t row0 = row_of(i);
            const uint16_t* from = a.grad + (row0 + w) * a.grad_stride + out0;
            if (whole_words(row0, kRows, a.n)) {
                const uint32_t* words = reinterpret_cast<const uint32_t*>(from - odd) + lane;
                #pragma unroll
                for (int r = 0; r < kFetched; r++) {
                    next[r][0] = needs[0] ? __ldg(words) : 0u;
                    next[r][1] = needs[1] ? __ldg(words + 32) : 0u;
                    next[r][2] = needs[2] ? __ldg(words + 33) : 0u;
                    words += 4 * a.grad_stride;
                }
                return;
            }
            #pragma unroll
            for (int r = 0; r < kFetched; r++) {
                const bool live = row0 + w + kTeam * r < a.n;
                #pragma unroll
                for (int j = 0; j < 3; j++) {
                    const int c = word_column(j == 2 ? 64 : lane + 32 * j, odd);
                    const uint32_t lo = live && needs[j] && c >= 0 ? from[c] : 0u, hi = live && needs[j] && c + 1 < grad_columns ? from[c + 1] : 0u;
                    next[r][j] = lo | hi << 16;
                }
                from += kTeam * a.grad_stride;
            }
        };
        // bias: on the grid the 8 columns of 16-byte word lane % 16, else columns 2 lane + e % 2 + 64 (e / 2); the sum of a stage's rows
        // first, so that the long sum has few steps
        float sums[8] = {};
        float scales = 0.0f, next_scales = scales_of(team);
        if (!kOnGrid) fetch(team);
        for (int i = team; i < stages; i += 2) {
            const uint32_t slot = i % kStages, value = i % kValueSlots;
            const int quarter = i / 2 % 4;
            if (quarter == 0) scales = next_scales;
            const uint32_t scale_bits = __float_as_uint(__shfl_sync(0xFFFFFFFFu, scales, quarter * 8 + lane % 8));
            const uint64_t scale = static_cast<uint64_t>(scale_bits) << 32 | scale_bits;
            uint8_t* stage = smem + kRingOffset + slot * kStageBytes;
            // warp-uniform, for the shuffle
            if (!__all_sync(0xFFFFFFFFu, wait_phase(landed_bar(slot), (i / kStages) & 1u, abort))) break;
            const uint8_t* codes = stage + kGradBytes;
            uint4 held[2];
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                // the box's rows are `half` bytes long, 64 or 128, and so is its swizzle: it follows the address bits from 7 on
                const uint32_t at = own_row * half + j * kAtom + own_code;
                if (j * kAtom < half) held[j] = *reinterpret_cast<const uint4*>(codes + (at ^ (((at >> 7) & (half / 16 - 1)) << 4)));
            }
            if (i >= kValueSlots) {  // the MMAs of the stage that had this slot
                const int last = i - kValueSlots;
                if (!__all_sync(0xFFFFFFFFu, wait_phase(empty_bar(last % kStages), (last / kStages) & 1u, abort))) break;
            }
            uint8_t* values = smem + kValueOffset + value * kValueBytes + own_row * 128;
            #pragma unroll
            for (int j = 0; j < 2; j++) {
                if (j * kAtom >= half) break;
                const uint32_t words[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
                #pragma unroll
                for (int p = 0; p < 2; p++) {
                    const uint2 lo = values_of(words[2 * p], scale), hi = values_of(words[2 * p + 1], scale);
                    *reinterpret_cast<uint4*>(values + j * kAtomBytes + (((own_code / 8 + p) ^ (own_row & 7)) << 4)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
                }
            }
            float stage_sums[8] = {};
            if constexpr (!kOnGrid) {
                #pragma unroll
                for (int r = 0; r < kFetched; r++) {
                    const int own = w + kTeam * r;  // own & 7 == w
                    uint32_t pairs[2] = {next[r][0], next[r][1]};
                    if (odd) {
                        const uint32_t after0 = __shfl_sync(0xFFFFFFFFu, lane == 0 ? next[r][1] : next[r][0], (lane + 1) % 32);
                        const uint32_t after1 = __shfl_down_sync(0xFFFFFFFFu, next[r][1], 1);
                        pairs[0] = __funnelshift_r(next[r][0], after0, 16);
                        pairs[1] = __funnelshift_r(next[r][1], lane == 31 ? next[r][2] : after1, 16);
                    }
                    #pragma unroll
                    for (int j = 0; j < 2; j++) {
                        *reinterpret_cast<uint32_t*>(stage + j * kAtomBytes + own * 128 + (((lane / 4) ^ w) << 4) + lane % 4 * 4) = pairs[j];
                        stage_sums[2 * j] += __uint_as_float(pairs[j] << 16);
                        stage_sums[2 * j + 1] += __uint_as_float(pairs[j] & 0xFFFF0000u);
                    }
                }
            }
            else if (bias && lane % 16 < 8 * grad_atoms) {
                #pragma unroll
                for (int r = 0; r < kRows / 16; r++) {
                    const int row = 2 * w + lane / 16 + 16 * r, word = lane % 16;
                    const uint4 v = *reinterpret_cast<const uint4*>(stage + word / 8 * kAtomBytes + row * 128 + (((word % 8) ^ (row & 7)) << 4));
                    const uint32_t words[4] = {v.x, v.y, v.z, v.w};
                    #pragma unroll
                    for (int q = 0; q < 4; q++) {
                        stage_sums[2 * q] += __uint_as_float(words[q] << 16);
                        stage_sums[2 * q + 1] += __uint_as_float(words[q] & 0xFFFF0000u);
                    }
                }
            }
            #pragma unroll
            for (int e = 0; e < 8; e++) sums[e] += stage_sums[e];
            fence_async_shared();
            __syncwarp();
            if (lane == 0) arrive_first_cta(full_bar(value));
            // behind the fence, which waits for the loads in flight
            if (quarter == 0) next_scales = scales_of(i + 8);
            if (!kOnGrid) fetch(i + 2);
        }
        if (bias) {
            float* partial = reinterpret_cast<float*>(smem + kBiasOffset) + (warp - kFirstWorker) * 128;
            if (kOnGrid) {
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    sums[e] += __shfl_xor_sync(0xFFFFFFFFu, sums[e], 16);
                    if (lane < 16) partial[8 * lane + e] = sums[e];
                }
            }
            else {
                #pragma unroll
                for (int e = 0; e < 4; e++) partial[2 * lane + e % 2 + e / 2 * 64] = sums[e];
            }
        }
    }
    else {
        // the accumulator's rows 32 quadrant .. + 31, every second 16 columns: added to the running sum, the last time on their way to the workspace,
        // 4 columns of a row per 16-byte word, neighbouring rows next to one another
        const int quadrant = warp % 4, group = (warp - kFirstWorker - kWorkers) / 4, periods = (stages + kPeriod - 1) / kPeriod;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quadrant) << 16);
        float4* to = reinterpret_cast<float4*>(a.partial) + (static_cast<int64_t>(split) * tiles + tile) * (a.tile_in / 4) * kTileOut + 128 * rank +
                     32 * quadrant + lane;
        for (int p = 0; p < periods; p++) {
            // warp-uniform: the tensor-memory accesses are collective
            if (!__all_sync(0xFFFFFFFFu, wait_phase(sum_bar, p & 1u, abort))) break;
            fence_after_sync();
            for (int c = 16 * group; c < a.tile_in; c += 32) {
                uint32_t r[16], sum[16];
                issue_load<16>(lanes + c, r);
                if (p > 0) issue_load<16>(lanes + kSumColumn + c, sum);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (p > 0) {
                    #pragma unroll
                    for (int e = 0; e < 16; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(sum[e]));
                }
                if (p + 1 < periods) store_columns(lanes + kSumColumn + c, r);
                else if (32 * quadrant < grad_columns) {
                    #pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        to[static_cast<int64_t>((c + e) / 4) * kTileOut] =
                            make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]), __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
                    }
                }
            }
            if (p + 1 < periods) {
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_first_cta(read_bar);
            }
        }
    }

    fence_before_sync();
    __syncthreads();
    if (bias && threadIdx.x < grad_columns) {
        const float* partial = reinterpret_cast<const float*>(smem + kBiasOffset) + threadIdx.x;
        float sum = 0.0f;
        #pragma unroll
        for (int w = 0; w < kWorkers; w++) sum += partial[w * 128];
        a.bias_partial[static_cast<int64_t>(split) * a.out + out0 + threadIdx.x] = sum;
    }
    if (threadIdx.x == 32 && rank == 0) {
        // no MMA still writes the tensor memory freed below
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_bar) : "memory");
        drain_phase(drain_bar, 0);
    }
    if (threadIdx.x == 0 && *abort) atomicExch(a.status, kWaitTimeout);
    fence_before_sync();
    __syncthreads();
    sync_cluster();  // no MMA or arrival reaches this CTA any more
    fence_after_sync();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
}

// grad_weight += the shares' sums in their order. A warp takes 4 rows x 32 columns of a tile (32 words of 4 columns): 64-byte
// pieces of the workspace, 128-byte pieces of grad_weight. With many shares (kSpread) the block's 8 warps take every
// eighth share of the same words and their sums are added in order, else each warp has words of its own. The blocks past
// the tiles do the bias, 32 outputs each.
constexpr int kJoinWarps = 8;

struct JoinArgs {
    const float* partial;
    const float* bias_partial;
    int in, out, tile_in, tiles_in, splits;
    int64_t words;           // of one share
    int64_t word_blocks;
    float* grad_weight;
    float* grad_bias;
};

template <bool kSpread>
__global__ void __launch_bounds__(32 * kJoinWarps) fz_int8_weight_grad_join_kernel(const JoinArgs a) {
    __shared__ float4 parts[kJoinWarps][32];
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the shares are complete and visible
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (blockIdx.x >= a.word_blocks) {
        const int64_t o = (blockIdx.x - a.word_blocks) * 32 + lane;
        float sum = 0.0f;
        if (o < a.out) {
            for (int s = warp; s < a.splits; s += kJoinWarps) sum += __ldg(a.bias_partial + s * static_cast<int64_t>(a.out) + o);
        }
        parts[warp][lane].x = sum;
        __syncthreads();
        if (warp == 0 && o < a.out) {
            for (int w = 1; w < kJoinWarps; w++) sum += parts[w][lane].x;
            a.grad_bias[o] += sum;
        }
        return;
    }
    // piece: 8 words along the columns x 4 rows; pieces of a tile row by row of 4, then 32 columns further
    const int64_t piece = kSpread ? blockIdx.x : blockIdx.x * int64_t{kJoinWarps} + warp;
    const int per_tile = a.tile_in / 32 * (kTileOut / 4);
    const int64_t tile = piece / per_tile;
    const int within = static_cast<int>(piece - tile * per_tile);
    const int row = within % (kTileOut / 4) * 4 + lane % 4, column_word = within / (kTileOut / 4) * 8 + lane / 4;
    const int64_t o = tile / a.tiles_in * kTileOut + row, k = tile % a.tiles_in * a.tile_in + column_word * 4;
    const bool live = piece * 32 < a.words && o < a.out && k < a.in;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (live) {
        const float4* from = reinterpret_cast<const float4*>(a.partial) + tile * (a.tile_in / 4) * kTileOut + static_cast<int64_t>(column_word) * kTileOut + row;
        #pragma unroll 8
        for (int s = kSpread ? warp : 0; s < a.splits; s += kSpread ? kJoinWarps : 1) {
            const float4 v = __ldcs(from + s * a.words);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
    }
    if constexpr (kSpread) {
        parts[warp][lane] = sum;
        __syncthreads();
        if (warp > 0) return;
        #pragma unroll
        for (int w = 1; w < kJoinWarps; w++) {
            const float4 v = parts[w][lane];
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
    }
    if (!live) return;
    float* to = a.grad_weight + o * a.in + k;
    if (k + 4 <= a.in && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
        float4 v = *reinterpret_cast<const float4*>(to);
        v.x += sum.x, v.y += sum.y, v.z += sum.z, v.w += sum.w;
        *reinterpret_cast<float4*>(to) = v;
    }
    else {
        const float part[4] = {sum.x, sum.y, sum.z, sum.w};
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            if (k + e < a.in) to[e] += part[e];
        }
    }
}

struct Plan {
    int tile_in, tiles_out, tiles_in, splits, stages_total;
    int64_t words() const { return static_cast<int64_t>(tiles_out) * tiles_in * (tile_in / 4) * kTileOut; }
};

constexpr int kPlanPairs = 74;    // pairs of multiprocessors the plan counts on (the workspace's size does not depend on the device)
constexpr int kMinStages = 4;     // stages of a share: enough that its sums' way through the workspace stays small

Plan plan_of(const int64_t n, const int64_t in, const int64_t out) {
    Plan p{};
    p.tile_in = in <= 128 ? 128 : kMaxTileIn;
    p.tiles_out = static_cast<int>((out + kTileOut - 1) / kTileOut);
    p.tiles_in = static_cast<int>((in + p.tile_in - 1) / p.tile_in);
    p.stages_total = static_cast<int>((n + kRows - 1) / kRows);
    const int64_t tiles = static_cast<int64_t>(p.tiles_out) * p.tiles_in;
    const int64_t most = std::max<int64_t>(1, p.stages_total / kMinStages);
    if (tiles < kPlanPairs) p.splits = static_cast<int>(std::min<int64_t>(most, kPlanPairs / tiles));
    else {
        // more tiles than pairs: up to four shares where the last wave is fuller for it
        auto waves = [&](const int64_t s) { return static_cast<double>((tiles * s + kPlanPairs - 1) / kPlanPairs) / static_cast<double>(s); };
        p.splits = 1;
        for (int s = 2; s <= 4 && s <= most; s++) {
            if (waves(s) < 0.93 * waves(p.splits)) p.splits = s;
        }
    }
    return p;
}

bool encode_grad(CUtensorMap* map, const uint16_t* grad, const int64_t out, const int64_t stride, const int64_t n) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = zf::tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(out), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
    const cuuint32_t box[2] = {kAtom, kRows};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<uint16_t*>(grad), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_codes(CUtensorMap* map, const int8_t* codes, const int64_t in, const int64_t stride, const int64_t n, const int columns) {
    const PFN_cuTensorMapEncodeTiled_v12000 encode = zf::tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(in), static_cast<cuuint64_t>(n)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(columns), kRows};
    const cuuint32_t element_strides[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(codes), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  columns == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kOnGrid>
cudaError_t launch(const Args& a, const unsigned blocks, cudaStream_t stream) {
    const cudaError_t error = zf::allow_shared_memory<fz_int8_weight_grad_kernel<kOnGrid>>(kSmemBytes);
    if (error != cudaSuccess) return error;
    fz_int8_weight_grad_kernel<kOnGrid><<<blocks, kThreads, kSmemBytes, stream>>>(a);
    return cudaGetLastError();
}

int invalid(const char* message) { return zf::set_error(ZF_ERROR_INVALID_ARGUMENT, message); }

}  // namespace zf::int8_weight_grad

int64_t zf_int8_weight_grad_workspace_size(const int64_t n, const int64_t in, const int64_t out) {
    using namespace zf::int8_weight_grad;
    if (n <= 0 || in <= 0 || out <= 0) return 0;
    const Plan p = plan_of(n, in, out);
    return p.splits * (p.words() * 16 + out * 4);
}

int zf_int8_weight_grad(const zf_int8_weight_grad_args* args, cudaStream_t stream) {
    using namespace zf::int8_weight_grad;
    constexpr int64_t kMost = (int64_t{1} << 31) - 256, kMostColumns = 1 << 20;
    if (args == nullptr || args->n < 0 || args->in <= 0 || args->out <= 0 || args->n >= kMost || args->in > kMostColumns || args->out > kMostColumns) {
        return invalid("int8_weight_grad: invalid sizes");
    }
    if (args->n == 0) return ZF_OK;
    if (args->codes == nullptr || reinterpret_cast<uintptr_t>(args->codes) % 16 != 0 || args->codes_stride % 16 != 0 || args->codes_stride < args->in) {
        return invalid("int8_weight_grad: codes must be 16-byte aligned with a row stride that is a multiple of 16");
    }
    if (args->grad == nullptr || args->grad_stride < args->out || args->scales == nullptr || args->grad_weight == nullptr || args->status == nullptr) {
        return invalid("int8_weight_grad: invalid grad, scales, grad_weight or status");
    }
    if (!zf::aligned_as<uint16_t>(args->grad) || !zf::aligned_as<float>(args->scales, args->grad_weight, args->grad_bias, args->status)) {
        return invalid("int8_weight_grad: misaligned grad, scales, grad_weight, grad_bias or status");
    }
    if (args->workspace == nullptr || reinterpret_cast<uintptr_t>(args->workspace) % 16 != 0
        || args->workspace_bytes < zf_int8_weight_grad_workspace_size(args->n, args->in, args->out)) {
        return invalid("int8_weight_grad: workspace too small");
    }
    const Plan p = plan_of(args->n, args->in, args->out);
    Args a{};
    a.grad = args->grad;
    a.grad_stride = args->grad_stride;
    a.scales = args->scales;
    a.n = static_cast<int>(args->n);
    a.in = static_cast<int>(args->in);
    a.out = static_cast<int>(args->out);
    a.tile_in = p.tile_in;
    a.tiles_out = p.tiles_out;
    a.tiles_in = p.tiles_in;
    a.splits = p.splits;
    a.stages_total = p.stages_total;
    a.partial = static_cast<float*>(args->workspace);
    a.bias_partial = args->grad_bias != nullptr ? a.partial + p.splits * p.words() * 4 : nullptr;
    a.status = args->status;
    const bool on_grid = reinterpret_cast<uintptr_t>(args->grad) % 16 == 0 && args->grad_stride % 8 == 0;
    if (!encode_codes(&a.code_map, args->codes, args->in, args->codes_stride, args->n, p.tile_in / 2)
        || (on_grid && !encode_grad(&a.grad_map, args->grad, args->out, args->grad_stride, args->n))) {
        return zf::set_error(ZF_ERROR_CUDA, "int8_weight_grad: no tensor map");
    }
    const unsigned blocks = 2u * static_cast<unsigned>(p.splits * p.tiles_out * p.tiles_in);
    cudaError_t error = on_grid ? launch<true>(a, blocks, stream) : launch<false>(a, blocks, stream);
    if (error == cudaSuccess) {
        const bool spread = p.splits >= kJoinWarps;
        const int64_t pieces = p.words() / 32, word_blocks = spread ? pieces : (pieces + kJoinWarps - 1) / kJoinWarps;
        const int64_t bias_blocks = a.bias_partial != nullptr ? (args->out + 31) / 32 : 0;
        const JoinArgs j{a.partial, a.bias_partial, a.in, a.out, a.tile_in, a.tiles_in, a.splits, p.words(), word_blocks, args->grad_weight, args->grad_bias};
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(static_cast<unsigned>(word_blocks + bias_blocks));
        config.blockDim = dim3(32 * kJoinWarps);
        config.stream = stream;
        cudaLaunchAttribute early{};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        config.attrs = &early;
        config.numAttrs = 1;
        error = cudaLaunchKernelEx(&config, spread ? fz_int8_weight_grad_join_kernel<true> : fz_int8_weight_grad_join_kernel<false>, j);
    }
    return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, "int8_weight_grad");
}
