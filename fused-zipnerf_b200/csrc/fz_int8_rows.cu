// fz_int8_rows.cu -- the row operators of include/zf_int8.h: quantization and restoring of rows, the add + RMS norm with
// 8-bit output, and the norm's backward from its 8-bit output. All of them stream rows once through registers: they
// move a few bytes per element and do a few operations on each, so device memory bounds them.
//
// A row belongs to a team of kTeam threads (8 lanes, a warp, or a block of 256) of which each holds kHeld elements in
// registers between the row's reductions, so every input is read once and every output written once. A team takes
// kBatch rows at a time and issues all of their loads, of every operand, before it touches the first value: a conversion
// behind a load waits for it, and with one load at a time per thread the memory's latency bound these kernels. Rows longer than the widest team holds are walked three times by a block (fz_long_* kernels).
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

__device__ __forceinline__ uint32_t pack_bf16(const float lo, const float hi) {
    const __nv_bfloat162 pair = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&pair);
}

// eight elements at the 16-byte aligned address of element j
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

// reductions over the row's team; every thread of the team gets the result. A block's reduction leaves one word per warp
// in `shared[slot]`; two reductions in a row use different slots, so that the barrier of the second lies between the
// reads of the first and the next writes to its slot.
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
// finite value), and the factor that turns values into codes: the scale's reciprocal, exact for powers of two, else
// within an ulp
__device__ __forceinline__ float row_scale(const uint32_t largest, const bool power_of_two, float& to_codes) {
    to_codes = 0.0f;
    if (largest == 0) return 0.0f;
    if (largest >= kInfinityBits) return __uint_as_float(0x7FFFFFFFu);
    if (power_of_two) {
        // largest / 127 = m 2^e / 127 with 127 = 1.984375 x 2^6: at most 2^(e - 6) exactly when m is at most 1.984375
        const int exponent = max(static_cast<int>((largest + 0x00020000u - 1u) >> 23) - 6, 1);
        to_codes = __uint_as_float(static_cast<uint32_t>(254 - exponent) << 23);
        return __uint_as_float(static_cast<uint32_t>(exponent) << 23);
    }
    const float scale = fmaxf(__fdiv_rn(__uint_as_float(largest), kLargestCode), kSmallestScale);
    asm("rcp.approx.f32 %0, %1;" : "=f"(to_codes) : "f"(scale));
    return scale;
}

// x / scale to the nearest integer, ties to even, in the low byte: the sum with 1.5 x 2^23 leaves the integer in the low
// bits of the significand, and the product is not rounded before. The product with the reciprocal is within 2 ulp of the
// quotient: at most 127 (1 + 2^-21), so it cannot round to 128.
__device__ __forceinline__ uint32_t to_code(const float v, const float to_codes) { return __float_as_uint(fmaf(v, to_codes, 12582912.0f)); }

// the low bytes of four words
__device__ __forceinline__ uint32_t pack_codes(const uint32_t a, const uint32_t b, const uint32_t c, const uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040u), __byte_perm(c, d, 0x0040u), 0x5410u);
}

// the larger magnitude (with some sign), NaN if one is
__device__ __forceinline__ float larger_magnitude(const float a, const float b) {
    float out;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(out) : "f"(a), "f"(b));
    return out;
}

struct QuantizeArgs {
    const void* x;
    int64_t x_stride;
    const void* residual;
    int64_t residual_stride;
    const float* weight;
    int64_t n, d;
    float one_over_d, eps;
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

// a thread's elements of a row as they lie in memory: fetch only loads, value(i) converts. Elements past d are zero.
template <int kType, bool kVector, int kTeam, int kHeld>
struct Held {
    static constexpr int kPerWord = kVector && kType == kBf16 ? 2 : 1;
    uint32_t words[kHeld / kPerWord];

    __device__ __forceinline__ void fetch(const void* row, const int d, const int t) {
        if constexpr (kVector) {
            #pragma unroll
            for (int i = 0; i < kHeld; i += 8) {
                const int j = element<true, kTeam>(t, i);
                constexpr int kLoads = kType == kF32 ? 2 : 1;
                const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + static_cast<int64_t>(j) * kSize<kType>);
                #pragma unroll
                for (int q = 0; q < kLoads; q++) {
                    const uint4 v = j + 8 <= d ? __ldg(from + q) : make_uint4(0, 0, 0, 0);
                    uint32_t* to = words + i / kPerWord + 4 * q;
                    to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
                }
            }
            if (d % 8 != 0) fetch_tail(row, d, t);
        }
        else {
            #pragma unroll
            for (int i = 0; i < kHeld; i++) {
                const int j = element<false, kTeam>(t, i);
                words[i] = j < d ? bits(row, j) : 0u;
            }
        }
    }

    __device__ __forceinline__ float value(const int i) const {
        if constexpr (kType == kF32) return __uint_as_float(words[i]);
        else if constexpr (kVector) return __uint_as_float(i % 2 ? words[i / 2] & 0xFFFF0000u : words[i / 2] << 16);
        else return __uint_as_float(words[i] << 16);
    }

private:
    static __device__ __forceinline__ uint32_t bits(const void* row, const int j) {
        if constexpr (kType == kF32) return __ldg(static_cast<const uint32_t*>(row) + j);
        else return __ldg(static_cast<const uint16_t*>(row) + j);
    }
    // the last d % 8 elements
    __device__ __forceinline__ void fetch_tail(const void* row, const int d, const int t) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += 8) {
            const int j = element<true, kTeam>(t, i);
            if (j >= d || j + 8 <= d) continue;
            #pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t v = j + e < d ? bits(row, j + e) : 0u;
                if constexpr (kType == kF32) words[i + e] = v;
                else words[(i + e) / 2] |= v << (e % 2 * 16);
            }
        }
    }
};

// the same for codes
template <bool kVector, int kTeam, int kHeld>
struct HeldCodes {
    uint32_t words[kVector ? kHeld / 4 : kHeld];

    __device__ __forceinline__ void fetch(const int8_t* row, const int d, const int t) {
        if constexpr (kVector) {
            #pragma unroll
            for (int i = 0; i < kHeld; i += 8) {
                const int j = element<true, kTeam>(t, i);
                const uint2 v = j + 8 <= d ? __ldg(reinterpret_cast<const uint2*>(row + j)) : make_uint2(0, 0);
                words[i / 4] = v.x, words[i / 4 + 1] = v.y;
            }
            if (d % 8 != 0) {
                #pragma unroll
                for (int i = 0; i < kHeld; i += 8) {
                    const int j = element<true, kTeam>(t, i);
                    if (j >= d || j + 8 <= d) continue;
                    #pragma unroll
                    for (int e = 0; e < 8; e++) {
                        if (j + e < d) words[(i + e) / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(row + j + e))) << (8 * (e % 4));
                    }
                }
            }
        }
        else {
            #pragma unroll
            for (int i = 0; i < kHeld; i++) {
                const int j = element<false, kTeam>(t, i);
                words[i] = j < d ? static_cast<uint8_t>(__ldg(row + j)) : 0u;
            }
        }
    }

    // 2^23 + (code + 128) as a float without a conversion instruction, less 2^23 + 128: exact
    __device__ __forceinline__ float value(const int i) const {
        const uint32_t biased = (kVector ? words[i / 4] : words[i]) ^ (kVector ? 0x80808080u : 0x80u);
        return __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7440u + (kVector ? i % 4 : 0))) - 8388736.0f;
    }
};

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

// rows that a team fetches before it works on the first: about 32 elements of each operand per thread
template <int kHeld, int kOperands>
constexpr int kBatch = kHeld * kOperands >= 32 ? 1 : 32 / (kHeld * kOperands);

// the rows of x (kNorm: the normalised rows of x + residual) as codes and scales
template <int kX, int kResidual, bool kNorm, bool kVector, int kTeam, int kHeld>
__global__ void __launch_bounds__(kBlock) fz_quantize_kernel(const QuantizeArgs a) {
    constexpr int kRows = kBatch<kHeld, kResidual != kNone ? 2 : 1>;
    __shared__ uint32_t shared[2][kBlock / 32];
    const Team<kTeam> team{shared};
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    // a team's rows: kBlock / kTeam teams of a block side by side, kRows times
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kBlock / kTeam * kRows) + threadIdx.x / kTeam;
    auto row_at = [&](const int b) { return first + b * (kBlock / kTeam); };
    Held<kX, kVector, kTeam, kHeld> x[kRows];
    Held<kResidual != kNone ? kResidual : kX, kVector, kTeam, kHeld> r[kRows];
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        const int64_t row = min(row_at(b), a.n - 1);  // rows past the last repeat it and write nothing
        x[b].fetch(row_of<kX>(a.x, row, a.x_stride), d, t);
        if constexpr (kResidual != kNone) r[b].fetch(row_of<kResidual>(a.residual, row, a.residual_stride), d, t);
    }
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        const int64_t row = row_at(b);
        if (row >= a.n) return;
        float v[kHeld];
        #pragma unroll
        for (int i = 0; i < kHeld; i++) v[i] = x[b].value(i);
        bool overflow = false;
        if constexpr (kNorm) {
            if constexpr (kResidual != kNone) {
                #pragma unroll
                for (int i = 0; i < kHeld; i++) v[i] += r[b].value(i);
                store_row<kResidual, kVector, kTeam>(row_of<kResidual>(a.sum, row, a.sum_stride), d, t, v);
            }
            float squares = 0.0f;
            #pragma unroll
            for (int i = 0; i < kHeld; i++) squares = fmaf(v[i], v[i], squares);
            squares = team.sum(squares, 0);
            overflow = !(squares <= FLT_MAX);
            const float rstd = overflow ? __uint_as_float(0x7FFFFFFFu) : __frsqrt_rn(squares * a.one_over_d + a.eps);
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
        float magnitude = 0.0f;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) magnitude = larger_magnitude(magnitude, v[i]);
        uint32_t largest = team.max(magnitude_bits(magnitude), kNorm ? 1 : b % 2);
        if (overflow) largest = kInfinityBits;
        float to_codes;
        const float scale = row_scale(largest, a.power_of_two, to_codes);
        if (t == 0) a.scales[row] = scale;
        // no code is 0x80 or above 127 in magnitude; those of a row that is not finite are zero
        const uint32_t keep = largest < kInfinityBits ? 0xFFFFFFFFu : 0u;
        int8_t* codes = a.codes + row * a.codes_stride;
        if constexpr (kVector) {
            #pragma unroll
            for (int i = 0; i < kHeld; i += 8) {
                const int j = element<true, kTeam>(t, i);
                uint32_t words[2];
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float* u = &v[i + 4 * h];
                    words[h] = pack_codes(to_code(u[0], to_codes), to_code(u[1], to_codes), to_code(u[2], to_codes), to_code(u[3], to_codes)) & keep;
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
                if (j < d) codes[j] = static_cast<int8_t>(to_code(v[i], to_codes) & keep);
            }
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
        rstd = overflow ? __uint_as_float(0x7FFFFFFFu) : __frsqrt_rn(squares * a.one_over_d + a.eps);
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
        codes[j] = static_cast<int8_t>(finite ? to_code(scaled(v, j), to_codes) : 0u);
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

// codes * scales. kVector: a team per row as above, eight elements per access. Else the output, contiguous but with rows
// off the 16-byte grid, is written as one sequence of 16-byte words, whose elements' rows and columns one division per
// word finds; or (kWord = 1) any other layout, element by element.
template <int kOut, int kTeam, int kHeld>
__global__ void __launch_bounds__(kBlock) fz_dequantize_kernel(const RestoreArgs a) {
    constexpr int kRows = kBatch<kHeld, 1>;
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kBlock / kTeam * kRows) + threadIdx.x / kTeam;
    auto row_at = [&](const int b) { return first + b * (kBlock / kTeam); };
    HeldCodes<true, kTeam, kHeld> codes[kRows];
    float scales[kRows];
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        const int64_t row = min(row_at(b), a.n - 1);
        codes[b].fetch(a.codes + row * a.codes_stride, d, t);
        scales[b] = __ldg(a.scales + row);
    }
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        if (row_at(b) >= a.n) return;
        float v[kHeld];
        #pragma unroll
        for (int i = 0; i < kHeld; i++) v[i] = codes[b].value(i) * scales[b];
        store_row<kOut, true, kTeam>(row_of<kOut>(a.out, row_at(b), a.out_stride), d, t, v);
    }
}

template <int kOut, int kWord>
__global__ void __launch_bounds__(kBlock) fz_dequantize_flat_kernel(const RestoreArgs a) {
    const int64_t total = a.n * a.d;
    for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * kWord; at < total; at += static_cast<int64_t>(gridDim.x) * kBlock * kWord) {
        int64_t row = total <= UINT32_MAX ? static_cast<uint32_t>(at) / static_cast<uint32_t>(a.d) : at / a.d;
        int64_t j = at - row * a.d;
        float v[kWord];
        #pragma unroll
        for (int e = 0; e < kWord; e++) {
            v[e] = at + e < total ? static_cast<float>(a.codes[row * a.codes_stride + j]) * __ldg(a.scales + row) : 0.0f;
            if (++j == a.d) j = 0, row++;
        }
        if constexpr (kWord == 8) {
            if (at + 8 <= total) store_eight<kOut>(a.out, at, v);
            else {
                #pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (at + e < total) store_one<kOut>(a.out, at + e, v[e]);
                }
            }
        }
        else store_one<kOut>(row_of<kOut>(a.out, at / a.d, a.out_stride), at % a.d, v[0]);
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
    float one_over_d;
    void* grad_x;
    int64_t grad_x_stride;
};

// grad_x = rstd (grad - y mean(grad y)) + grad_residual, y = codes * scale
template <int kGrad, int kResidual, bool kVector, int kTeam, int kHeld>
__global__ void __launch_bounds__(kBlock) fz_norm_backward_kernel(const BackwardArgs a) {
    constexpr int kOut = kResidual != kNone ? kResidual : kGrad;
    constexpr int kRows = kBatch<kHeld, 2>;
    __shared__ uint32_t shared[2][kBlock / 32];
    const Team<kTeam> team{shared};
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kBlock / kTeam * kRows) + threadIdx.x / kTeam;
    auto row_at = [&](const int b) { return first + b * (kBlock / kTeam); };
    Held<kGrad, kVector, kTeam, kHeld> grad[kRows];
    HeldCodes<kVector, kTeam, kHeld> codes[kRows];
    Held<kOut, kVector, kTeam, kHeld> r[kRows];
    float scales[kRows], rstds[kRows];
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        const int64_t row = min(row_at(b), a.n - 1);  // rows past the last repeat it and write nothing
        grad[b].fetch(row_of<kGrad>(a.grad, row, a.grad_stride), d, t);
        codes[b].fetch(a.codes + row * a.codes_stride, d, t);
        if constexpr (kResidual != kNone) r[b].fetch(row_of<kResidual>(a.grad_residual, row, a.grad_residual_stride), d, t);
        scales[b] = __ldg(a.scales + row);
        rstds[b] = __ldg(a.rstd + row);
    }
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        const int64_t row = row_at(b);
        if (row >= a.n) return;
        float g[kHeld], y[kHeld];
        float dot = 0.0f;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            g[i] = grad[b].value(i);
            y[i] = codes[b].value(i) * scales[b];
            dot = fmaf(g[i], y[i], dot);
        }
        const float mean = team.sum(dot, b % 2) * a.one_over_d;
        #pragma unroll
        for (int i = 0; i < kHeld; i++) {
            g[i] = rstds[b] * fmaf(-y[i], mean, g[i]);
            if constexpr (kResidual != kNone) g[i] += r[b].value(i);
        }
        store_row<kOut, kVector, kTeam>(row_of<kOut>(a.grad_x, row, a.grad_x_stride), d, t, g);
    }
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
    const float mean = team.sum(dot, 0) * a.one_over_d;
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
            constexpr int kRows = kBlock / kTeam * kBatch<kHeld, kResidual != kNone ? 2 : 1>;
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
            constexpr int kRows = kBlock / kTeam * kBatch<kHeld, 2>;
            const unsigned blocks = static_cast<unsigned>((a.n + kRows - 1) / kRows);
            if (vector) fz_norm_backward_kernel<kGrad, kResidual, true, kTeam, kHeld><<<blocks, kBlock, 0, stream>>>(a);
            else fz_norm_backward_kernel<kGrad, kResidual, false, kTeam, kHeld><<<blocks, kBlock, 0, stream>>>(a);
        },
        [&] { fz_long_norm_backward_kernel<kGrad, kResidual><<<static_cast<unsigned>(a.n), kBlock, 0, stream>>>(a); });
    return cudaGetLastError();
}

template <int kOut>
cudaError_t launch_restore(const RestoreArgs& a, const bool vector, cudaStream_t stream) {
    // words of eight elements, or single elements, spread over a few blocks per multiprocessor
    auto flat = [&](const int word) {
        const int64_t needed = (a.n * a.d + kBlock * word - 1) / (kBlock * word);
        return static_cast<unsigned>(needed < 4096 ? needed : 4096);
    };
    auto element_wise = [&] { fz_dequantize_flat_kernel<kOut, 1><<<flat(1), kBlock, 0, stream>>>(a); };
    if (vector) {
        with_team(
            a.d,
            [&](const auto team, const auto held) {
                constexpr int kTeam = decltype(team)::value, kHeld = decltype(held)::value;
                constexpr int kRows = kBlock / kTeam * kBatch<kHeld, 1>;
                fz_dequantize_kernel<kOut, kTeam, kHeld><<<static_cast<unsigned>((a.n + kRows - 1) / kRows), kBlock, 0, stream>>>(a);
            },
            [&] {
                if (a.out_stride == a.d) fz_dequantize_flat_kernel<kOut, 8><<<flat(8), kBlock, 0, stream>>>(a);
                else element_wise();
            });
    }
    else if (a.out_stride == a.d && reinterpret_cast<uintptr_t>(a.out) % 16 == 0) fz_dequantize_flat_kernel<kOut, 8><<<flat(8), kBlock, 0, stream>>>(a);
    else element_wise();
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
    const RestoreArgs a{args->codes, args->codes_stride, args->scales, args->n, args->d, args->out, args->out_stride};
    const bool vector = aligned(args->out, args->out_stride, size_of(args->out_dtype));
    return finish(args->out_dtype == ZF_FLOAT32 ? launch_restore<kF32>(a, vector, stream) : launch_restore<kBf16>(a, vector, stream), "dequantize_rows");
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
    const QuantizeArgs a{args->x, args->x_stride, args->residual, args->residual_stride, args->weight, args->n, args->d, 1.0f / static_cast<float>(args->d), args->eps,
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
                         args->grad_residual_stride, args->n, args->d, 1.0f / static_cast<float>(args->d), args->grad_x, args->grad_x_stride};
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
