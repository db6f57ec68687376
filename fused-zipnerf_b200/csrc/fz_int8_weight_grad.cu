// fz_int8_weight_grad.cu -- the weight and bias gradient of a linear layer from the 8-bit checkpoint of its input
// (zf_int8_weight_grad): grad_weight += grad^T (codes x scales), grad_bias += column sums of grad, on the tcgen05 tensor
// cores (kind::f16 on bf16, fp32 accumulators in tensor memory).
//
// The samples are the K dimension of this product, so both operands are MN-major. A CTA takes one tile of grad_weight (up
// to 256 outputs x 256 inputs) and a share of the samples, 64 at a time through a ring of stages:
//   warp 0 (one lane)  brings the stage's gradients by TMA tensor copies (128-byte swizzle, no multicast) where their rows
//                      lie on the 16-byte grid;
//   warps 2-9          read the stage's codes (a stage ahead, into registers), turn them into bf16 values codes x scale
//                      and write them as the B operand; gradients off the grid they bring too; they also sum the bias;
//   warp 1 (one lane)  issues the MMAs.
// With power-of-two scales codes x scale is a bf16 number, so both operands are exact and only the sums round.
//
// Each CTA leaves its sums in the workspace, in the order of its tensor-memory reads; the join kernel adds the shares of a
// tile in their order, so that results do not depend on timing.
//
// Bounded waits and the status as in fz_int8_linear.cu.
#include "zf_int8.h"
#include "fz_status.h"
#include "fz_tcgen05.cuh"
#include "fz_tma.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <cstdint>

namespace zf::int8_weight_grad {

using namespace zf::nerf_mlp;  // the tcgen05 building blocks

constexpr int kRows = 64;                    // samples of a stage
constexpr int kAtom = 64;                    // columns of a 128-byte-swizzled atom
constexpr int kAtomBytes = kRows * 128;
constexpr int kMaxTile = 256;                // outputs (two M = 128 halves) and inputs of a tile
constexpr int kOperandBytes = kMaxTile / kAtom * kAtomBytes;  // 32 KB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kStages = 3;
constexpr int kWorkers = 8;                  // warps that convert, and read the accumulators
constexpr int kFirstWorker = 2;
constexpr int kThreads = 32 * (kFirstWorker + kWorkers);
constexpr int kHeaderBytes = 1024;           // barriers
constexpr int kBiasOffset = kHeaderBytes;    // 8 x 256 partial bias sums
constexpr int kRingOffset = kBiasOffset + kWorkers * kMaxTile * 4;
constexpr int kSmemBytes = kRingOffset + kStages * kStageBytes;
constexpr uint32_t kTmemColumns = 512;
static_assert(kRingOffset % 1024 == 0, "the swizzled ring starts on a 1024-byte boundary");
static_assert(kSmemBytes <= 227 * 1024, "one CTA per SM");

struct Args {
    CUtensorMap grad_map;    // grad [n, out] bf16, boxes of 64 samples x 64 columns (on the 16-byte grid)
    const uint16_t* grad;
    int64_t grad_stride;
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    int n, in, out;
    int tile_out, tile_in;   // multiples of 64, at most 256
    int tiles_out, tiles_in;
    int splits;
    int stages_total;        // stages over all samples
    float* partial;          // [splits][tiles][tile_in / 4][m_rows] float4
    float* bias_partial;     // [splits][out], or null
    int* status;
};

// rows of the accumulators of a tile: 128 or 256
__host__ __device__ __forceinline__ int m_rows(const int tile_out) { return tile_out > 128 ? 256 : 128; }

// four codes (one word) as values
__device__ __forceinline__ void values_of(const uint32_t word, const float scale, float (&v)[4]) {
    const uint32_t biased = word ^ 0x80808080u;  // code + 128
    #pragma unroll
    for (int e = 0; e < 4; e++) {
        // 2^23 + (code + 128), exactly, without a conversion instruction
        const float f = __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7440u + e));
        v[e] = (f - 8388736.0f) * scale;
    }
}

template <bool kOnGrid>
__global__ void __launch_bounds__(kThreads, 1) fz_int8_weight_grad_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + 516);
    const uint32_t bar0 = smem_address(smem);
    auto grad_bar = [&](const uint32_t i) { return bar0 + 8u * i; };                 // a stage's gradients have landed
    auto full_bar = [&](const uint32_t i) { return bar0 + 8u * (kStages + i); };     // the workers have written their part
    auto empty_bar = [&](const uint32_t i) { return bar0 + 8u * (2 * kStages + i); };
    const uint32_t done_bar = bar0 + 8u * (3 * kStages);
    const uint32_t ring = bar0 + kRingOffset;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int tile = blockIdx.x % (a.tiles_out * a.tiles_in), split = blockIdx.x / (a.tiles_out * a.tiles_in);
    const int out0 = tile / a.tiles_in * a.tile_out, in0 = tile % a.tiles_in * a.tile_in;
    const int first = static_cast<int>(static_cast<int64_t>(a.stages_total) * split / a.splits);
    const int stages = static_cast<int>(static_cast<int64_t>(a.stages_total) * (split + 1) / a.splits) - first;
    const int halves = m_rows(a.tile_out) / 128;
    const int grad_atoms = (min(a.tile_out, a.out - out0) + kAtom - 1) / kAtom, in_atoms = a.tile_in / kAtom;
    const bool bias = a.bias_partial != nullptr && in0 == 0;

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(tmem_slot)), "r"(kTmemColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; i++) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(grad_bar(i)), "r"(1));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full_bar(i)), "r"(kWorkers));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty_bar(i)), "r"(1 + (kOnGrid && bias ? kWorkers : 0)));
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(done_bar), "r"(1));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        *abort = 0;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (kOnGrid && lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&a.grad_map)) : "memory");
            int issued = 0;
            for (int i = 0; i < stages; i++) {
                const uint32_t slot = i % kStages;
                if (i >= kStages && !wait_phase(empty_bar(slot), (i / kStages - 1) & 1u, abort)) break;
                expect_bytes(grad_bar(slot), static_cast<uint32_t>(grad_atoms * kAtomBytes));
                for (int g = 0; g < grad_atoms; g++) {
                    tma_load_2d(ring + slot * kStageBytes + g * kAtomBytes, &a.grad_map, out0 + g * kAtom, (first + i) * kRows, grad_bar(slot));
                }
                issued = i + 1;
            }
            // every copy issued has landed before the CTA's shared memory can go to another CTA
            for (int i = issued > kStages ? issued - kStages : 0; i < issued; i++) drain_phase(grad_bar(i % kStages), (i / kStages) & 1u);
        }
    }
    else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = instr_descriptor(kTileRows, a.tile_in, true, true);
            for (int i = 0; i < stages; i++) {
                const uint32_t slot = i % kStages, parity = (i / kStages) & 1u;
                if (kOnGrid && !wait_phase(grad_bar(slot), parity, abort)) break;
                if (!wait_phase(full_bar(slot), parity, abort)) break;
                fence_after_sync();
                const uint32_t at = ring + slot * kStageBytes;
                for (int k = 0; k < kRows / kMmaK; k++) {
                    // 16 samples: two 8-row groups further; an M half: two 64-column atoms further
                    const uint64_t b = mn_sw128_descriptor(at + kOperandBytes + k * 2048, kRows);
                    for (int h = 0; h < halves; h++) {
                        mma(tmem + h * kMaxTile, mn_sw128_descriptor(at + h * 2 * kAtomBytes + k * 2048, kRows), b, idesc, (i > 0 || k > 0) ? 1u : 0u);
                    }
                }
                commit(empty_bar(slot));
            }
            commit(done_bar);
        }
    }
    else {
        const int w = warp - kFirstWorker;
        // codes: warp w's rows are 8 w .. 8 w + 7 of a stage; lane l holds row l % 8 and the 16 codes l / 8 of each atom, so
        // that eight lanes of a shared-memory store lie in eight different places of the swizzle
        const int own_row = 8 * w + lane % 8, own_code = 16 * (lane / 8);
        uint4 next[kMaxTile / kAtom];
        float next_scale = 0.0f;
        auto fetch = [&](const int i) {
            const int64_t row = static_cast<int64_t>(first + i) * kRows + own_row;
            next_scale = row < a.n ? __ldg(a.scales + row) : 0.0f;
            const int8_t* codes = a.codes + row * a.codes_stride + in0;
            #pragma unroll
            for (int j = 0; j < kMaxTile / kAtom; j++) {
                const int c = kAtom * j + own_code;
                next[j] = make_uint4(0, 0, 0, 0);
                if (j < in_atoms && row < a.n && in0 + c < a.in) {
                    // 16 bytes from a multiple of 16 stay inside the row's stride; the last row may end with its codes
                    if (in0 + c + 16 <= a.in || row + 1 < a.n) next[j] = __ldg(reinterpret_cast<const uint4*>(codes + c));
                    else {
                        uint32_t words[4] = {};
                        #pragma unroll
                        for (int e = 0; e < 16; e++) {
                            if (in0 + c + e < a.in) words[e / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(codes[c + e])) << (8 * (e % 4));
                        }
                        next[j] = make_uint4(words[0], words[1], words[2], words[3]);
                    }
                }
            }
        };
        float sums[8] = {};  // bias: on the grid the 8 columns of 16-byte word `lane`, else columns lane + 32 j
        bool ok = true;
        if (stages > 0) fetch(0);
        for (int i = 0; i < stages; i++) {
            const uint32_t slot = i % kStages, parity = (i / kStages) & 1u;
            uint4 held[kMaxTile / kAtom];
            #pragma unroll
            for (int j = 0; j < kMaxTile / kAtom; j++) held[j] = next[j];
            const float scale = next_scale;
            if (i + 1 < stages) fetch(i + 1);
            if (i >= kStages && !(ok = wait_phase(empty_bar(slot), parity ^ 1u, abort))) break;
            uint8_t* stage = smem + kRingOffset + slot * kStageBytes;
            uint8_t* operand = stage + kOperandBytes + own_row * 128;
            #pragma unroll
            for (int j = 0; j < kMaxTile / kAtom; j++) {
                if (j >= in_atoms) break;
                const uint32_t words[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
                #pragma unroll
                for (int p = 0; p < 2; p++) {
                    float lo[4], hi[4];
                    values_of(words[2 * p], scale, lo);
                    values_of(words[2 * p + 1], scale, hi);
                    *reinterpret_cast<uint4*>(operand + j * kAtomBytes + (((own_code / 8 + p) ^ (own_row & 7)) << 4)) =
                        make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]));
                }
            }
            if constexpr (!kOnGrid) {
                // gradients off the 16-byte grid: warp w's rows w + 8 r, lane l's columns l + 32 j
                const int columns = min(a.tile_out, a.out - out0);
                float stage_sums[8] = {};
                #pragma unroll
                for (int r = 0; r < kRows / kWorkers; r++) {
                    const int own = w + kWorkers * r;
                    const int64_t row = static_cast<int64_t>(first + i) * kRows + own;
                    const uint16_t* grad = a.grad + row * a.grad_stride + out0;
                    uint16_t v[8];
                    #pragma unroll
                    for (int j = 0; j < 8; j++) v[j] = row < a.n && lane + 32 * j < columns ? __ldg(grad + lane + 32 * j) : static_cast<uint16_t>(0);
                    #pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int c = lane + 32 * j;
                        if (c < kAtom * grad_atoms) {
                            *reinterpret_cast<uint16_t*>(stage + c / kAtom * kAtomBytes + own * 128 + (((c % kAtom / 8) ^ (own & 7)) << 4) + c % 8 * 2) = v[j];
                        }
                        stage_sums[j] += __uint_as_float(static_cast<uint32_t>(v[j]) << 16);
                    }
                }
                #pragma unroll
                for (int j = 0; j < 8; j++) sums[j] += stage_sums[j];
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) arrive(full_bar(slot));
            if (kOnGrid && bias) {
                if (!(ok = wait_phase(grad_bar(slot), parity, abort))) break;
                // warp w's rows w + 8 r: the sum of eight rows first, so that the long sum has few steps
                float stage_sums[8] = {};
                if (lane / 8 < grad_atoms) {
                    #pragma unroll
                    for (int r = 0; r < kRows / kWorkers; r++) {
                        const int row = w + kWorkers * r;  // row & 7 == w
                        const uint4 v = *reinterpret_cast<const uint4*>(stage + lane / 8 * kAtomBytes + row * 128 + (((lane % 8) ^ w) << 4));
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
                __syncwarp();
                if (lane == 0) arrive(empty_bar(slot));
            }
        }
        // the accumulators, 4 columns of a row per 16-byte word, neighbouring rows next to one another
        ok = __all_sync(0xFFFFFFFFu, ok && wait_phase(done_bar, 0, abort));
        fence_after_sync();
        if (ok) {
            const int rows = m_rows(a.tile_out), group = w / 4, quadrant = warp % 4;
            float4* to = reinterpret_cast<float4*>(a.partial) +
                         (static_cast<int64_t>(split) * a.tiles_out * a.tiles_in + tile) * (a.tile_in / 4) * rows + 32 * quadrant + lane;
            // two halves: a group of four warps each; one: the groups take alternate 32-column pieces
            const int half = halves == 2 ? group : 0;
            for (int c = halves == 2 ? 0 : 32 * group; c < a.tile_in; c += halves == 2 ? 32 : 64) {
                uint32_t r[32];
                issue_load<32>(tmem + (static_cast<uint32_t>(32 * quadrant) << 16) + half * kMaxTile + c, r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                #pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    // without a stage there was no MMA: the sums are zero
                    const float4 v = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
                    to[static_cast<int64_t>((c + j) / 4) * rows + 128 * half] = stages > 0 ? v : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
        }
        if (bias) {
            float* partial = reinterpret_cast<float*>(smem + kBiasOffset) + w * kMaxTile;
            #pragma unroll
            for (int e = 0; e < 8; e++) partial[kOnGrid ? 8 * lane + e : lane + 32 * e] = sums[e];
        }
    }

    fence_before_sync();
    __syncthreads();
    if (bias && threadIdx.x < kMaxTile && threadIdx.x < min(a.tile_out, a.out - out0)) {
        const float* partial = reinterpret_cast<const float*>(smem + kBiasOffset) + threadIdx.x;
        float sum = 0.0f;
        #pragma unroll
        for (int w = 0; w < kWorkers; w++) sum += partial[w * kMaxTile];
        a.bias_partial[static_cast<int64_t>(split) * a.out + out0 + threadIdx.x] = sum;
    }
    if (threadIdx.x == 32) drain_phase(done_bar, 0);  // no MMA still writes the tensor memory freed below
    if (threadIdx.x == 0 && *abort) atomicExch(a.status, kWaitTimeout);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
}

// grad_weight += the shares' sums: 32 words (4 columns of a row) per block of 8 warps, each warp every eighth share, then
// the eight sums in their order; the blocks past the tiles do the same for the bias
constexpr int kJoinWarps = 8;

struct JoinArgs {
    const float* partial;
    const float* bias_partial;
    int in, out, tile_out, tile_in, tiles_in, splits;
    int64_t words;           // of one share
    int64_t word_blocks;
    float* grad_weight;
    float* grad_bias;
};

__global__ void __launch_bounds__(32 * kJoinWarps) fz_int8_weight_grad_join_kernel(const JoinArgs a) {
    __shared__ float4 parts[kJoinWarps][32];
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
    const int64_t word = blockIdx.x * int64_t{32} + lane;
    const int rows = m_rows(a.tile_out);
    const int64_t per_tile = static_cast<int64_t>(a.tile_in / 4) * rows;
    const int64_t tile = word / per_tile;
    const int within = static_cast<int>(word - tile * per_tile);
    const int64_t o = tile / a.tiles_in * a.tile_out + within % rows, k = tile % a.tiles_in * a.tile_in + within / rows * 4;
    const bool live = word < a.words && within % rows < a.tile_out && o < a.out && k < a.in;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (live) {
        const float4* from = reinterpret_cast<const float4*>(a.partial) + word;
        #pragma unroll 4
        for (int s = warp; s < a.splits; s += kJoinWarps) {
            const float4 v = __ldcs(from + s * a.words);
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
    }
    parts[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && live) {
        #pragma unroll
        for (int w = 1; w < kJoinWarps; w++) {
            const float4 v = parts[w][lane];
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        float* to = a.grad_weight + o * a.in + k;
        const float part[4] = {sum.x, sum.y, sum.z, sum.w};
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            if (k + e < a.in) to[e] += part[e];
        }
    }
}

struct Plan {
    int tile_out, tile_in, tiles_out, tiles_in, splits, stages_total;
    int64_t words() const { return static_cast<int64_t>(tiles_out) * tiles_in * (tile_in / 4) * m_rows(tile_out); }
};

// columns in equal shares of at most 256, whole 64-column atoms
int share_of(const int64_t columns) {
    const int64_t shares = (columns + kMaxTile - 1) / kMaxTile;
    return static_cast<int>(((columns + shares - 1) / shares + kAtom - 1) / kAtom * kAtom);
}

constexpr int kPlanSms = 148;     // multiprocessors the plan counts on (the workspace's size does not depend on the device)
constexpr int kMinStages = 4;     // samples of a share: enough that its sums' way through the workspace stays small

Plan plan_of(const int64_t n, const int64_t in, const int64_t out) {
    Plan p{};
    p.tile_out = share_of(out);
    p.tile_in = share_of(in);
    p.tiles_out = static_cast<int>((out + p.tile_out - 1) / p.tile_out);
    p.tiles_in = static_cast<int>((in + p.tile_in - 1) / p.tile_in);
    p.stages_total = static_cast<int>((n + kRows - 1) / kRows);
    const int64_t tiles = static_cast<int64_t>(p.tiles_out) * p.tiles_in;
    const int64_t most = std::max<int64_t>(1, p.stages_total / kMinStages);
    if (tiles < kPlanSms) p.splits = static_cast<int>(std::min<int64_t>(most, kPlanSms / tiles));
    else {
        // more tiles than multiprocessors: up to four shares where the last wave is fuller for it
        auto waves = [&](const int64_t s) { return static_cast<double>((tiles * s + kPlanSms - 1) / kPlanSms) / static_cast<double>(s); };
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

template <bool kOnGrid>
cudaError_t launch(const Args& a, const unsigned blocks, cudaStream_t stream) {
    const cudaError_t error = cudaFuncSetAttribute(fz_int8_weight_grad_kernel<kOnGrid>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
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
    if (args->workspace == nullptr || reinterpret_cast<uintptr_t>(args->workspace) % 16 != 0
        || args->workspace_bytes < zf_int8_weight_grad_workspace_size(args->n, args->in, args->out)) {
        return invalid("int8_weight_grad: workspace too small");
    }
    const Plan p = plan_of(args->n, args->in, args->out);
    Args a{};
    a.grad = args->grad;
    a.grad_stride = args->grad_stride;
    a.codes = args->codes;
    a.codes_stride = args->codes_stride;
    a.scales = args->scales;
    a.n = static_cast<int>(args->n);
    a.in = static_cast<int>(args->in);
    a.out = static_cast<int>(args->out);
    a.tile_out = p.tile_out;
    a.tile_in = p.tile_in;
    a.tiles_out = p.tiles_out;
    a.tiles_in = p.tiles_in;
    a.splits = p.splits;
    a.stages_total = p.stages_total;
    a.partial = static_cast<float*>(args->workspace);
    a.bias_partial = args->grad_bias != nullptr ? a.partial + p.splits * p.words() * 4 : nullptr;
    a.status = args->status;
    const bool on_grid = reinterpret_cast<uintptr_t>(args->grad) % 16 == 0 && args->grad_stride % 8 == 0;
    if (on_grid && !encode_grad(&a.grad_map, args->grad, args->out, args->grad_stride, args->n)) return zf::set_error(ZF_ERROR_CUDA, "int8_weight_grad: no tensor map");
    const unsigned blocks = static_cast<unsigned>(p.splits * p.tiles_out * p.tiles_in);
    cudaError_t error = on_grid ? launch<true>(a, blocks, stream) : launch<false>(a, blocks, stream);
    if (error == cudaSuccess) {
        const int64_t word_blocks = (p.words() + 31) / 32, bias_blocks = a.bias_partial != nullptr ? (args->out + 31) / 32 : 0;
        const JoinArgs j{a.partial, a.bias_partial, a.in, a.out, a.tile_out, a.tile_in, a.tiles_in, a.splits, p.words(), word_blocks, args->grad_weight,
                         args->grad_bias};
        fz_int8_weight_grad_join_kernel<<<static_cast<unsigned>(word_blocks + bias_blocks), 32 * kJoinWarps, 0, stream>>>(j);
        error = cudaGetLastError();
    }
    return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, "int8_weight_grad");
}
