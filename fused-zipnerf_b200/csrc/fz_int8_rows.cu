// fz_int8_rows.cu -- the row operators of include/zf_int8.h: quantization and restoring of rows, the add + RMS norm with
// 8-bit output, and the norm's backward from its 8-bit output. All of them stream rows once through registers: they
// move a few bytes per element and do a few operations on each, so device memory bounds them.
//
// A row belongs to a team of kTeam threads (8 lanes, a warp, or a block of 256) of which each holds kHeld elements in
// registers between the row's reductions, so every input is read once and every output written once. Rows longer than
// the widest team holds are walked three times by a block (fz_long_* kernels).
//
// Compiled without fast math: the quotients are IEEE ones and subnormal inputs are kept, so that the codes are those of
// the definition.
#include "zf_int8.h"
#include "fz_status.h"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

namespace zf::int8_rows {

constexpr int kBlock = 256;
constexpr float kLargestCode = 127.0f;
constexpr float kSmallestScale = 0x1p-126f;
constexpr uint32_t kInfinityBits = 0x7F800000u;

// element type tags: what a tensor holds (kNone: there is no such tensor)
enum Type : int { kF32 = ZF_FLOAT32, kBf16 = ZF_BFLOAT16, kNone = 2 };

template <int kType>
constexpr int kSize = kType == kF32 ? 4 : 2;

template <int kType>
__device__ __forceinline__ float load_one(const void* row, const int64_t j) {
    if constexpr (kType == kF32) return static_cast<const float*>(row)[j];
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[j]);
}

template <int kType>
__device__ __forceinline__ void store_one(void* row, const int64_t j, const float v) {
    if constexpr (kType == kF32) static_cast<float*>(row)[j] = v;
    else static_cast<__nv_bfloat16*>(row)[j] = __float2bfloat16_rn(v);
}

// eight elements at the 16-byte aligned address of element j
template <int kType>
__device__ __forceinline__ void load_eight(const void* row, const int64_t j, float* v) {
    if constexpr (kType == kF32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(row) + j);
        const float4 a = p[0], b = p[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    else {
        const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + j);
        const uint32_t words[4] = {a.x, a.y, a.z, a.w};
        #pragma unroll
        for (int q = 0; q < 4; q++) {
            v[2 * q] = __uint_as_float(words[q] << 16);
            v[2 * q + 1] = __uint_as_float(words[q] & 0xFFFF0000u);
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16(const float lo, const float hi) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&pair);
}

template <int kType>
__device__ __forceinline__ void store_eight(void* row, const int64_t j, const float* v) {
    if constexpr (kType == kF32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(row) + j);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + j) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
}

__device__ __forceinline__ void load_eight_codes(const int8_t* row, const int64_t j, float* v) {
    const uint2 a = *reinterpret_cast<const uint2*>(row + j);
    const uint32_t words[2] = {a.x, a.y};
    #pragma unroll
    for (int e = 0; e < 8; e++) v[e] = static_cast<float>(static_cast<int8_t>(words[e / 4] >> (8 * (e % 4))));
}

// reductions over the row's team; every thread of the team gets the result. `shared` holds one word per warp and is
// free for the next reduction after `barrier`-separated use: the three words of a row alternate between three slots.
template <int kTeam>
struct Team {
    uint32_t (*shared)[kBlock / 32];

    __device__ __forceinline__ uint32_t mask() const {
        if constexpr (kTeam >= 32) return 0xFFFFFFFFu;
        else return ((1u << kTeam) - 1u) << (threadIdx.x % 32 / kTeam * kTeam);
    }

    __device__ __forceinline__ float sum(float v, const int slot) const {
        #pragma unroll
        for (int s = (kTeam < 32 ? kTeam : 32) / 2; s > 0; s /= 2) v += __shfl_xor_sync(mask(), v, s);
        if constexpr (kTeam > 32) {
            if (threadIdx.x % 32 == 0) shared[slot][threadIdx.x / 32] = __float_as_uint(v);
            __syncthreads();
            v = 0.0f;
            #pragma unroll
            for (int w = 0; w < kTeam / 32; w++) v += __uint_as_float(shared[slot][w]);
        }
        return v;
    }

    __device__ __forceinline__ uint32_t max(uint32_t v, const int slot) const {
        v = __reduce_max_sync(mask(), v);
        if constexpr (kTeam > 32) {
            if (threadIdx.x % 32 == 0) shared[slot][threadIdx.x / 32] = v;
            __syncthreads();
            #pragma unroll
            for (int w = 0; w < kTeam / 32; w++) v = ::max(v, shared[slot][w]);
        }
        return v;
    }
};

__device__ __forceinline__ uint32_t magnitude_bits(const float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// the scale of a row from the largest magnitude's bits (which order like the magnitudes, infinities and NaN above every
// finite value), and the factor that turns values into codes
__device__ __forceinline__ float row_scale(const uint32_t largest, const bool power_of_two, float& to_codes) {
    to_codes = 0.0f;
    if (largest == 0) return 0.0f;
    if (largest >= kInfinityBits) return __uint_as_float(0x7FFFFFFFu);
    float scale = fmaxf(__fdiv_rn(__uint_as_float(largest), kLargestCode), kSmallestScale);
    if (power_of_two) {
        // the next power of two unless it is one: the quotient is at most 2^121, so the exponent has room
        const uint32_t bits = __float_as_uint(scale);
        scale = __uint_as_float((bits + 0x007FFFFFu) & 0xFF800000u);
    }
    to_codes = __frcp_rn(scale);
    return scale;
}

// x / scale to the nearest integer, ties to even. The product with the reciprocal is within 2 ulp of the quotient: at
// most 127 (1 + 2^-22), so it cannot round to 128; the clamp keeps that true by construction.
__device__ __forceinline__ int to_code(const float v, const float to_codes) {
    return max(-127, min(127, __float2int_rn(v * to_codes)));
}

struct QuantizeArgs {
    const void* x;
    int64_t x_stride;
    const void* residual;
    int64_t residual_stride;
    const float* weight;
    int64_t n, d;
    float eps;
    bool power_of_two;
    int8_t* codes;
    int64_t codes_stride;
    float* scales;
    void* sum;
    int64_t sum_stride;
    float* rstd;
};

template <int kType>
__device__ __forceinline__ const void* row_of(const void* base, const int64_t row, const int64_t stride) {
    return static_cast<const uint8_t*>(base) + row * stride * kSize<kType>;
}
template <int kType>
__device__ __forceinline__ void* row_of(void* base, const int64_t row, const int64_t stride) {
    return static_cast<uint8_t*>(base) + row * stride * kSize<kType>;
}

// element i of thread t of a team: kVector: eight neighbouring elements per 16-byte (bf16) access, else one at a time
// with neighbouring threads on neighbouring elements
template <bool kVector, int kTeam>
__device__ __forceinline__ int element(const int t, const int i) {
    if constexpr (kVector) return (i / 8) * (8 * kTeam) + 8 * t + i % 8;
    else return i * kTeam + t;
}

template <int kType, bool kVector, int kTeam, int kHeld>
__device__ __forceinline__ void load_row(const void* row, const int d, const int t, float (&v)[kHeld]) {
    if constexpr (kVector) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += 8) {
            const int j = element<true, kTeam>(t, i);
            if (j + 8 <= d) load_eight<kType>(row, j, v + i);
            else {
                #pragma unroll
                for (int e = 0; e < 8; e++) v[i + e] = j + e < d ? load_one<kType>(row, j + e) : 0.0f;
            }
        }
    }
    else {
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            const int j = element<false, kTeam>(t, i);
            v[i] = j < d ? load_one<kType>(row, j) : 0.0f;
        }
    }
}

template <int kType, bool kVector, int kTeam, int kHeld>
__device__ __forceinline__ void store_row(void* row, const int d, const int t, const float (&v)[kHeld]) {
    if constexpr (kVector) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += 8) {
            const int j = element<true, kTeam>(t, i);
            if (j + 8 <= d) store_eight<kType>(row, j, v + i);
            else {
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (j + e < d) store_one<kType>(row, j + e, v[i + e]);
                }
            }
        }
    }
    else {
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            const int j = element<false, kTeam>(t, i);
            if (j < d) store_one<kType>(row, j, v[i]);
        }
    }
}

template <bool kVector, int kTeam, int kHeld>
__device__ __forceinline__ void load_codes(const int8_t* row, const int d, const int t, float (&v)[kHeld]) {
    if constexpr (kVector) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += 8) {
            const int j = element<true, kTeam>(t, i);
            if (j + 8 <= d) load_eight_codes(row, j, v + i);
            else {
                #pragma unroll
                for (int e = 0; e < 8; e++) v[i + e] = j + e < d ? static_cast<float>(row[j + e]) : 0.0f;
            }
        }
    }
    else {
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            const int j = element<false, kTeam>(t, i);
            v[i] = j < d ? static_cast<float>(row[j]) : 0.0f;
        }
    }
}

// the rows of x (kNorm: the normalised rows of x + residual) as codes and scales
template <int kX, int kResidual, bool kNorm, bool kVector, int kTeam, int kHeld>
__global__ void __launch_bounds__(kBlock) fz_quantize_kernel(const QuantizeArgs a) {
    __shared__ uint32_t shared[2][kBlock / 32];
    const Team<kTeam> team{shared};
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kTeam) + threadIdx.x / kTeam;
    if (row >= a.n) return;
    float v[kHeld];
    load_row<kX, kVector, kTeam>(row_of<kX>(a.x, row, a.x_stride), d, t, v);
    bool overflow = false;
    if constexpr (kNorm) {
        if constexpr (kResidual != kNone) {
            float r[kHeld];
            load_row<kResidual, kVector, kTeam>(row_of<kResidual>(a.residual, row, a.residual_stride), d, t, r);
            #pragma unroll
            for (int i = 0; i < kHeld; i++) v[i] += r[i];
            store_row<kResidual, kVector, kTeam>(row_of<kResidual>(a.sum, row, a.sum_stride), d, t, v);
        }
        float squares = 0.0f;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) squares = fmaf(v[i], v[i], squares);
        squares = team.sum(squares, 0);
        overflow = !(squares <= FLT_MAX);
        const float rstd = overflow ? __uint_as_float(0x7FFFFFFFu) : __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(squares, static_cast<float>(d)) + a.eps));
        if (t == 0 && a.rstd != nullptr) a.rstd[row] = rstd;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) v[i] *= rstd;
        if (a.weight != nullptr) {
            #pragma unroll
            for (int i = 0; i < kHeld; i++) {
                const int j = element<kVector, kTeam>(t, i);
                if (j < d) v[i] *= __ldg(a.weight + j);
            }
        }
    }
    uint32_t largest = 0;
    #pragma unroll
    for (int i = 0; i < kHeld; i++) largest = max(largest, magnitude_bits(v[i]));
    largest = team.max(largest, 1);
    if (overflow) largest = kInfinityBits;
    float to_codes;
    const float scale = row_scale(largest, a.power_of_two, to_codes);
    if (t == 0) a.scales[row] = scale;
    const bool finite = largest < kInfinityBits;
    int8_t* codes = a.codes + row * a.codes_stride;
    if constexpr (kVector) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += 8) {
            const int j = element<true, kTeam>(t, i);
            uint32_t words[2] = {0, 0};
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                if (finite) words[e / 4] |= (static_cast<uint32_t>(to_code(v[i + e], to_codes)) & 0xFFu) << (8 * (e % 4));
            }
            if (j + 8 <= d) *reinterpret_cast<uint2*>(codes + j) = make_uint2(words[0], words[1]);
            else {
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (j + e < d) codes[j + e] = static_cast<int8_t>(words[e / 4] >> (8 * (e % 4)));
                }
            }
        }
    }
    else {
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            const int j = element<false, kTeam>(t, i);
            if (j < d) codes[j] = static_cast<int8_t>(finite ? to_code(v[i], to_codes) : 0);
        }
    }
}

// rows longer than a team holds: a block reads the row once per reduction and once more for the codes
template <int kX, int kResidual, bool kNorm>
__global__ void __launch_bounds__(kBlock) fz_long_quantize_kernel(const QuantizeArgs a) {
    __shared__ uint32_t shared[2][kBlock / 32];
    const Team<kBlock> team{shared};
    const int64_t row = blockIdx.x;
    const void* x = row_of<kX>(a.x, row, a.x_stride);
    const void* residual = kResidual != kNone ? row_of<kResidual>(a.residual, row, a.residual_stride) : nullptr;
    auto value = [&](const int64_t j) {
        float v = load_one<kX>(x, j);
        if constexpr (kResidual != kNone) v += load_one<kResidual>(residual, j);
        return v;
    };
    float rstd = 1.0f;
    bool overflow = false;
    if constexpr (kNorm) {
        float squares = 0.0f;
        for (int64_t j = threadIdx.x; j < a.d; j += kBlock) {
            const float v = value(j);
            squares = fmaf(v, v, squares);
        }
        squares = team.sum(squares, 0);
        overflow = !(squares <= FLT_MAX);
        rstd = overflow ? __uint_as_float(0x7FFFFFFFu) : __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(squares, static_cast<float>(a.d)) + a.eps));
        if (threadIdx.x == 0 && a.rstd != nullptr) a.rstd[row] = rstd;
    }
    auto scaled = [&](const float v, const int64_t j) {
        if constexpr (!kNorm) return v;
        else return a.weight != nullptr ? v * rstd * __ldg(a.weight + j) : v * rstd;
    };
    uint32_t largest = 0;
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) largest = max(largest, magnitude_bits(scaled(value(j), j)));
    largest = team.max(largest, 1);
    if (overflow) largest = kInfinityBits;
    float to_codes;
    const float scale = row_scale(largest, a.power_of_two, to_codes);
    if (threadIdx.x == 0) a.scales[row] = scale;
    const bool finite = largest < kInfinityBits;
    int8_t* codes = a.codes + row * a.codes_stride;
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) {
        const float v = value(j);
        // each thread reads an element of the residual for the last time before it writes the same element of the sum
        if constexpr (kResidual != kNone) store_one<kResidual>(row_of<kResidual>(a.sum, row, a.sum_stride), j, v);
        codes[j] = static_cast<int8_t>(finite ? to_code(scaled(v, j), to_codes) : 0);
    }
}

struct RestoreArgs {
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    int64_t n, d;
    void* out;
    int64_t out_stride;
};

// codes * scales, eight (kVector) or one element per thread at a time; blocks of 256 threads over (row, chunk) pairs
template <int kOut, bool kVector>
__global__ void __launch_bounds__(kBlock) fz_dequantize_kernel(const RestoreArgs a) {
    constexpr int kChunk = kVector ? 8 : 1;
    const int64_t chunks = (a.d + kChunk - 1) / kChunk;
    const int64_t total = a.n * chunks;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t row = i / chunks, j = (i - row * chunks) * kChunk;
        const float scale = __ldg(a.scales + row);
        const int8_t* codes = a.codes + row * a.codes_stride;
        void* out = row_of<kOut>(a.out, row, a.out_stride);
        if constexpr (kVector) {
            if (j + 8 <= a.d) {
                float v[8];
                load_eight_codes(codes, j, v);
                #pragma unroll
                for (int e = 0; e < 8; e++) v[e] *= scale;
                store_eight<kOut>(out, j, v);
            }
            else {
                for (int64_t e = j; e < a.d; e++) store_one<kOut>(out, e, static_cast<float>(codes[e]) * scale);
            }
        }
        else store_one<kOut>(out, j, static_cast<float>(codes[j]) * scale);
    }
}

struct BackwardArgs {
    const void* grad;
    int64_t grad_stride;
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    const float* rstd;
    const void* grad_residual;
    int64_t grad_residual_stride;
    int64_t n, d;
    void* grad_x;
    int64_t grad_x_stride;
};

// grad_x = rstd (grad - y mean(grad y)) + grad_residual, y = codes * scale
template <int kGrad, int kResidual, bool kVector, int kTeam, int kHeld>
__global__ void __launch_bounds__(kBlock) fz_norm_backward_kernel(const BackwardArgs a) {
    constexpr int kOut = kResidual != kNone ? kResidual : kGrad;
    __shared__ uint32_t shared[1][kBlock / 32];
    const Team<kTeam> team{shared};
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / kTeam) + threadIdx.x / kTeam;
    if (row >= a.n) return;
    float g[kHeld], y[kHeld];
    load_row<kGrad, kVector, kTeam>(row_of<kGrad>(a.grad, row, a.grad_stride), d, t, g);
    load_codes<kVector, kTeam>(a.codes + row * a.codes_stride, d, t, y);
    float r[kResidual != kNone ? kHeld : 1];
    if constexpr (kResidual != kNone) load_row<kResidual, kVector, kTeam>(row_of<kResidual>(a.grad_residual, row, a.grad_residual_stride), d, t, r);
    const float scale = __ldg(a.scales + row), rstd = __ldg(a.rstd + row);
    float dot = 0.0f;
    #pragma unroll
    for (int i = 0; i < kHeld; i++) {
        y[i] *= scale;
        dot = fmaf(g[i], y[i], dot);
    }
    const float mean = __fdiv_rn(team.sum(dot, 0), static_cast<float>(d));
    #pragma unroll
    for (int i = 0; i < kHeld; i++) {
        g[i] = rstd * fmaf(-y[i], mean, g[i]);
        if constexpr (kResidual != kNone) g[i] += r[i];
    }
    store_row<kOut, kVector, kTeam>(row_of<kOut>(a.grad_x, row, a.grad_x_stride), d, t, g);
}

template <int kGrad, int kResidual>
__global__ void __launch_bounds__(kBlock) fz_long_norm_backward_kernel(const BackwardArgs a) {
    constexpr int kOut = kResidual != kNone ? kResidual : kGrad;
    __shared__ uint32_t shared[1][kBlock / 32];
    const Team<kBlock> team{shared};
    const int64_t row = blockIdx.x;
    const void* grad = row_of<kGrad>(a.grad, row, a.grad_stride);
    const int8_t* codes = a.codes + row * a.codes_stride;
    const float scale = __ldg(a.scales + row), rstd = __ldg(a.rstd + row);
    float dot = 0.0f;
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) dot = fmaf(load_one<kGrad>(grad, j), static_cast<float>(codes[j]) * scale, dot);
    const float mean = __fdiv_rn(team.sum(dot, 0), static_cast<float>(a.d));
    void* out = row_of<kOut>(a.grad_x, row, a.grad_x_stride);
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) {
        float g = rstd * fmaf(-static_cast<float>(codes[j]) * scale, mean, load_one<kGrad>(grad, j));
        if constexpr (kResidual != kNone) g += load_one<kResidual>(row_of<kResidual>(a.grad_residual, row, a.grad_residual_stride), j);
        store_one<kOut>(out, j, g);
    }
}

// ---------------------------------------------------------------------------------------------------------------------

bool aligned(const void* p, const int64_t stride, const int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}
bool valid_type(const int type) { return type == ZF_FLOAT32 || type == ZF_BFLOAT16; }
int size_of(const int type) { return type == ZF_FLOAT32 ? 4 : 2; }
bool valid_codes(const void* codes, const int64_t stride, const int64_t d) {
    return codes != nullptr && reinterpret_cast<uintptr_t>(codes) % 16 == 0 && stride % 16 == 0 && stride >= d;
}
bool valid_rows(const void* p, const int type, const int64_t stride, const int64_t d) {
    return p != nullptr && valid_type(type) && stride >= d && reinterpret_cast<uintptr_t>(p) % size_of(type) == 0;
}

constexpr int64_t kMaxRows = (int64_t{1} << 31) - 1;  // one block per row at the most

// the team that holds rows of d elements: team threads of which each holds `held` elements
template <typename Launch, typename LaunchLong>
void with_team(const int64_t d, const Launch& launch, const LaunchLong& launch_long) {
    using std::integral_constant;
    if (d <= 64) launch(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (d <= 256) launch(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (d <= 1024) launch(integral_constant<int, 32>{}, integral_constant<int, 32>{});
    else if (d <= 4096) launch(integral_constant<int, 256>{}, integral_constant<int, 16>{});
    else if (d <= 8192) launch(integral_constant<int, 256>{}, integral_constant<int, 32>{});
    else launch_long();
}

template <int kX, int kResidual, bool kNorm>
cudaError_t launch_quantize(const QuantizeArgs& a, const bool vector, cudaStream_t stream) {
    with_team(
        a.d,
        [&](const auto team, const auto held) {
            constexpr int kTeam = decltype(team)::value, kHeld = decltype(held)::value;
            constexpr int kRows = kBlock / kTeam;
            const unsigned blocks = static_cast<unsigned>((a.n + kRows - 1) / kRows);
            if (vector) fz_quantize_kernel<kX, kResidual, kNorm, true, kTeam, kHeld><<<blocks, kBlock, 0, stream>>>(a);
            else fz_quantize_kernel<kX, kResidual, kNorm, false, kTeam, kHeld><<<blocks, kBlock, 0, stream>>>(a);
        },
        [&] { fz_long_quantize_kernel<kX, kResidual, kNorm><<<static_cast<unsigned>(a.n), kBlock, 0, stream>>>(a); });
    return cudaGetLastError();
}

template <int kGrad, int kResidual>
cudaError_t launch_backward(const BackwardArgs& a, const bool vector, cudaStream_t stream) {
    with_team(
        a.d,
        [&](const auto team, const auto held) {
            constexpr int kTeam = decltype(team)::value, kHeld = decltype(held)::value;
            constexpr int kRows = kBlock / kTeam;
            const unsigned blocks = static_cast<unsigned>((a.n + kRows - 1) / kRows);
            if (vector) fz_norm_backward_kernel<kGrad, kResidual, true, kTeam, kHeld><<<blocks, kBlock, 0, stream>>>(a);
            else fz_norm_backward_kernel<kGrad, kResidual, false, kTeam, kHeld><<<blocks, kBlock, 0, stream>>>(a);
        },
        [&] { fz_long_norm_backward_kernel<kGrad, kResidual><<<static_cast<unsigned>(a.n), kBlock, 0, stream>>>(a); });
    return cudaGetLastError();
}

int finish(const cudaError_t error, const char* what) { return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, what); }

int invalid(const char* message) { return zf::set_error(ZF_ERROR_INVALID_ARGUMENT, message); }

}  // namespace zf::int8_rows

int zf_quantize_rows(const zf_quantize_rows_args* args, cudaStream_t stream) {
    using namespace zf::int8_rows;
    if (args == nullptr || args->n < 0 || args->d <= 0 || args->n > kMaxRows) return invalid("quantize_rows: invalid sizes");
    if (args->n == 0) return ZF_OK;
    if (!valid_rows(args->x, args->x_dtype, args->x_stride, args->d)) return invalid("quantize_rows: invalid x");
    if (!valid_codes(args->codes, args->codes_stride, args->d) || args->scales == nullptr) {
        return invalid("quantize_rows: codes must be 16-byte aligned with a row stride that is a multiple of 16");
    }
    QuantizeArgs a{};
    a.x = args->x;
    a.x_stride = args->x_stride;
    a.n = args->n;
    a.d = args->d;
    a.power_of_two = args->power_of_two != 0;
    a.codes = args->codes;
    a.codes_stride = args->codes_stride;
    a.scales = args->scales;
    const bool vector = aligned(args->x, args->x_stride, size_of(args->x_dtype));
    return finish(args->x_dtype == ZF_FLOAT32 ? launch_quantize<kF32, kNone, false>(a, vector, stream) : launch_quantize<kBf16, kNone, false>(a, vector, stream),
                  "quantize_rows");
}

int zf_dequantize_rows(const zf_dequantize_rows_args* args, cudaStream_t stream) {
    using namespace zf::int8_rows;
    if (args == nullptr || args->n < 0 || args->d <= 0 || args->n > kMaxRows) return invalid("dequantize_rows: invalid sizes");
    if (args->n == 0) return ZF_OK;
    if (!valid_codes(args->codes, args->codes_stride, args->d) || args->scales == nullptr) {
        return invalid("dequantize_rows: codes must be 16-byte aligned with a row stride that is a multiple of 16");
    }
    if (!valid_rows(args->out, args->out_dtype, args->out_stride, args->d)) return invalid("dequantize_rows: invalid output");
    int device = 0, n_sms = 0;
    cudaError_t error = cudaGetDevice(&device);
    if (error == cudaSuccess) error = cudaDeviceGetAttribute(&n_sms, cudaDevAttrMultiProcessorCount, device);
    if (error != cudaSuccess) return zf::set_cuda_error(error, "device query");
    const RestoreArgs a{args->codes, args->codes_stride, args->scales, args->n, args->d, args->out, args->out_stride};
    const bool vector = aligned(args->out, args->out_stride, size_of(args->out_dtype));
    const int64_t chunks = args->n * (vector ? (args->d + 7) / 8 : args->d);
    const int64_t needed = (chunks + kBlock - 1) / kBlock, most = static_cast<int64_t>(n_sms) * 32;
    const unsigned blocks = static_cast<unsigned>(needed < most ? needed : most);
    if (args->out_dtype == ZF_FLOAT32) {
        if (vector) fz_dequantize_kernel<kF32, true><<<blocks, kBlock, 0, stream>>>(a);
        else fz_dequantize_kernel<kF32, false><<<blocks, kBlock, 0, stream>>>(a);
    }
    else {
        if (vector) fz_dequantize_kernel<kBf16, true><<<blocks, kBlock, 0, stream>>>(a);
        else fz_dequantize_kernel<kBf16, false><<<blocks, kBlock, 0, stream>>>(a);
    }
    return finish(cudaGetLastError(), "dequantize_rows");
}

int zf_rms_norm_int8(const zf_rms_norm_int8_args* args, cudaStream_t stream) {
    using namespace zf::int8_rows;
    if (args == nullptr || args->n < 0 || args->d <= 0 || args->n > kMaxRows) return invalid("rms_norm_int8: invalid sizes");
    if (!(args->eps >= FLT_MIN && args->eps <= FLT_MAX)) return invalid("rms_norm_int8: eps must be positive");
    if ((args->residual == nullptr) != (args->sum == nullptr) && args->n > 0) return invalid("rms_norm_int8: residual and sum go together");
    if (args->n == 0) return ZF_OK;
    if (!valid_rows(args->x, args->x_dtype, args->x_stride, args->d)) return invalid("rms_norm_int8: invalid x");
    if (args->residual != nullptr && (!valid_rows(args->residual, args->residual_dtype, args->residual_stride, args->d)
                                      || !valid_rows(args->sum, args->residual_dtype, args->sum_stride, args->d))) {
        return invalid("rms_norm_int8: invalid residual or sum");
    }
    if (!valid_codes(args->codes, args->codes_stride, args->d) || args->scales == nullptr) {
        return invalid("rms_norm_int8: codes must be 16-byte aligned with a row stride that is a multiple of 16");
    }
    const QuantizeArgs a{args->x, args->x_stride, args->residual, args->residual_stride, args->weight, args->n, args->d, args->eps,
                         args->power_of_two != 0, args->codes, args->codes_stride, args->scales, args->sum, args->sum_stride, args->rstd};
    const bool residual = args->residual != nullptr;
    const int size = size_of(args->residual_dtype);
    const bool vector = aligned(args->x, args->x_stride, size_of(args->x_dtype))
                        && (!residual || (aligned(args->residual, args->residual_stride, size) && aligned(args->sum, args->sum_stride, size)));
    cudaError_t error;
    if (args->x_dtype == ZF_FLOAT32) {
        error = !residual ? launch_quantize<kF32, kNone, true>(a, vector, stream)
                : args->residual_dtype == ZF_FLOAT32 ? launch_quantize<kF32, kF32, true>(a, vector, stream)
                                                     : launch_quantize<kF32, kBf16, true>(a, vector, stream);
    }
    else {
        error = !residual ? launch_quantize<kBf16, kNone, true>(a, vector, stream)
                : args->residual_dtype == ZF_FLOAT32 ? launch_quantize<kBf16, kF32, true>(a, vector, stream)
                                                     : launch_quantize<kBf16, kBf16, true>(a, vector, stream);
    }
    return finish(error, "rms_norm_int8");
}

int zf_rms_norm_int8_backward(const zf_rms_norm_int8_backward_args* args, cudaStream_t stream) {
    using namespace zf::int8_rows;
    if (args == nullptr || args->n < 0 || args->d <= 0 || args->n > kMaxRows) return invalid("rms_norm_int8_backward: invalid sizes");
    if (args->n == 0) return ZF_OK;
    if (!valid_rows(args->grad, args->grad_dtype, args->grad_stride, args->d)) return invalid("rms_norm_int8_backward: invalid grad");
    const bool residual = args->grad_residual != nullptr;
    if (residual && !valid_rows(args->grad_residual, args->grad_residual_dtype, args->grad_residual_stride, args->d)) {
        return invalid("rms_norm_int8_backward: invalid grad_residual");
    }
    if (!valid_codes(args->codes, args->codes_stride, args->d) || args->scales == nullptr || args->rstd == nullptr) {
        return invalid("rms_norm_int8_backward: codes must be 16-byte aligned with a row stride that is a multiple of 16");
    }
    const int out_dtype = residual ? args->grad_residual_dtype : args->grad_dtype;
    if (!valid_rows(args->grad_x, out_dtype, args->grad_x_stride, args->d)) return invalid("rms_norm_int8_backward: invalid grad_x");
    const BackwardArgs a{args->grad, args->grad_stride, args->codes, args->codes_stride, args->scales, args->rstd, args->grad_residual,
                         args->grad_residual_stride, args->n, args->d, args->grad_x, args->grad_x_stride};
    const bool vector = aligned(args->grad, args->grad_stride, size_of(args->grad_dtype)) && aligned(args->grad_x, args->grad_x_stride, size_of(out_dtype))
                        && (!residual || aligned(args->grad_residual, args->grad_residual_stride, size_of(args->grad_residual_dtype)));
    cudaError_t error;
    if (args->grad_dtype == ZF_FLOAT32) {
        error = !residual ? launch_backward<kF32, kNone>(a, vector, stream)
                : args->grad_residual_dtype == ZF_FLOAT32 ? launch_backward<kF32, kF32>(a, vector, stream)
                                                          : launch_backward<kF32, kBf16>(a, vector, stream);
    }
    else {
        error = !residual ? launch_backward<kBf16, kNone>(a, vector, stream)
                : args->grad_residual_dtype == ZF_FLOAT32 ? launch_backward<kBf16, kF32>(a, vector, stream)
                                                          : launch_backward<kBf16, kBf16>(a, vector, stream);
    }
    return finish(error, "rms_norm_int8_backward");
}
