// fz_int8_rows.cu -- the row operators of include/zf_int8.h: quantization and restoring of rows, the add + RMS norm with
// 8-bit output, and the norm's backward from its 8-bit output. All of them stream rows once through registers: they
// move a few bytes per element and do a few operations on each, so device memory bounds them.
//
// A row belongs to a team of kTeam threads (8 lanes, a warp, or a block of 256) of which each holds kHeld elements in
// registers between the row's reductions, so every input is read once and every output written once. A team takes
// kBatch rows at a time and issues all of their loads, of every operand, before it touches the first value: a conversion
// behind a load waits for it, and with one load at a time per thread the memory's latency bound these kernels. Rows longer than the widest team holds are walked three times by a block (fz_long_* kernels).
//
// Measured on one B200, 2,097,152 x 256 bf16: quantize 0.27 ms, restore 0.24 ms, add + norm 0.57 ms, norm backward 0.52 ms,
// 6.0 to 7.2 TB/s against the 6.5 that a copy moves; the norm issues an instruction in 74 % of the cycles, so it is close to
// that bound as well. Odd widths (1 element per access) reach 2 to 4 TB/s, bound by their many narrow accesses.
//
// Compiled without fast math: the scales are IEEE quotients and subnormal inputs are kept; the codes are those of the fp32
// quotients x / scale (to_codes_of).
#include "zf_int8.h"
#include "fz_status.h"
#include "fz_launch.h"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

namespace zf::int8_rows {

constexpr int kBlock = 256;
// threads of a team kernel's block: whole teams
template <int kTeam>
constexpr int kTeamBlock = kTeam > kBlock || (kTeam > 32 && kTeam < kBlock) ? kTeam : kBlock;
constexpr int kMaxWarps = 16;
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

// reductions over the team's threads, of kRows rows side by side (independent, so their latencies overlap, and a block has
// one barrier for all of them); every thread gets the results. A block leaves one word per warp and row in `shared`, which
// serves one reduction.
template <int kTeam, int kRows>
struct Team {
    static __device__ __forceinline__ uint32_t mask() {
        if constexpr (kTeam >= 32) return 0xFFFFFFFFu;
        else return ((1u << kTeam) - 1u) << (threadIdx.x % 32 / kTeam * kTeam);
    }

    static __device__ __forceinline__ void sum(float (&v)[kRows], uint32_t (&shared)[kRows][kMaxWarps]) {
        #pragma unroll
        for (int s = (kTeam < 32 ? kTeam : 32) / 2; s > 0; s /= 2) {
            #pragma unroll
            for (int b = 0; b < kRows; b++) v[b] += __shfl_xor_sync(mask(), v[b], s);
        }
        if constexpr (kTeam > 32) {
            #pragma unroll
            for (int b = 0; b < kRows; b++) {
                if (threadIdx.x % 32 == 0) shared[b][threadIdx.x / 32] = __float_as_uint(v[b]);
            }
            __syncthreads();
            #pragma unroll
            for (int b = 0; b < kRows; b++) {
                v[b] = 0.0f;
                #pragma unroll
                for (int w = 0; w < kTeam / 32; w++) v[b] += __uint_as_float(shared[b][w]);
            }
        }
    }

    static __device__ __forceinline__ void max(uint32_t (&v)[kRows], uint32_t (&shared)[kRows][kMaxWarps]) {
        #pragma unroll
        for (int b = 0; b < kRows; b++) v[b] = __reduce_max_sync(mask(), v[b]);
        if constexpr (kTeam > 32) {
            #pragma unroll
            for (int b = 0; b < kRows; b++) {
                if (threadIdx.x % 32 == 0) shared[b][threadIdx.x / 32] = v[b];
            }
            __syncthreads();
            #pragma unroll
            for (int b = 0; b < kRows; b++) {
                #pragma unroll
                for (int w = 0; w < kTeam / 32; w++) v[b] = ::max(v[b], shared[b][w]);
            }
        }
    }
};

__device__ __forceinline__ uint32_t magnitude_bits(const float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// what turns the values of a row into codes: the scale's reciprocal as the sum of two floats, the second zero for powers of two
struct Reciprocal {
    float high, low;
};

// the scale of a row from the largest magnitude's bits (which order like the magnitudes, infinities and NaN above every
// finite value), and its reciprocal
__device__ __forceinline__ float row_scale(const uint32_t largest, const bool power_of_two, Reciprocal& to_codes) {
    to_codes = {0.0f, 0.0f};
    if (largest == 0) return 0.0f;
    if (largest >= kInfinityBits) return __uint_as_float(0x7FFFFFFFu);
    if (power_of_two) {
        // largest / 127 = m 2^e / 127 with 127 = 1.984375 x 2^6: at most 2^(e - 6) exactly when m is at most 1.984375
        const int exponent = max(static_cast<int>((largest + 0x00020000u - 1u) >> 23) - 6, 1);
        to_codes.high = __uint_as_float(static_cast<uint32_t>(254 - exponent) << 23);
        return __uint_as_float(static_cast<uint32_t>(exponent) << 23);
    }
    const float scale = fmaxf(__fdiv_rn(__uint_as_float(largest), kLargestCode), kSmallestScale);
    to_codes.high = __frcp_rn(scale);
    // 1 - high scale is a float, so it is exact; 1 / scale = high / (1 - error)
    const float error = fmaf(-to_codes.high, scale, 1.0f);
    to_codes.low = to_codes.high * fmaf(error, error, error);
    return scale;
}

// two values as codes, x / scale (the fp32 quotient) to the nearest integer, ties to even, in the low bytes of the words: the
// sum with 1.5 x 2^23 leaves the integer in the low bits of the significand. The high part alone gives products up to 2 ulp
// from the quotient, and rows meet half steps often (in bf16 every x of half the largest magnitude is one). With both parts
// the product is the quotient but where that lies within 2^-46 of a rounding boundary, and its code is the quotient's for every
// significand of a scale, at every half step and the floats around it (all 7.5e9 compared on the host), for scales
// below 2^102, where the low part is a normal number. At most 127 (1 + 2^-23), so it cannot round to 128. Division itself,
// for values near a half step alone, made quantizing 2,097,152 x 256 bf16 415 us instead of 300 (the high part alone: 290).
__device__ __forceinline__ void to_codes_of(const float x, const float y, const Reciprocal& to_codes, uint32_t& x_code, uint32_t& y_code) {
    asm("{\n.reg .b64 v, high, low, p;\n"
        "mov.b64 v, {%2, %3};\nmov.b64 high, {%4, %4};\nmov.b64 low, {%5, %5};\n"
        "mul.rn.f32x2 p, v, low;\nfma.rn.f32x2 p, v, high, p;\n"
        "mov.b64 v, {0f4B400000, 0f4B400000};\nadd.rn.f32x2 p, p, v;\nmov.b64 {%0, %1}, p;\n}\n"
        : "=r"(x_code), "=r"(y_code)
        : "f"(x), "f"(y), "f"(to_codes.high), "f"(to_codes.low));
}

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

// element i of thread t of a team. kVector neighbouring elements go with one access, neighbouring threads on neighbouring
// accesses: 8 where the rows lie on the 16-byte grid, 2 where they lie on pairs of elements (an even width), else 1.
template <int kVector, int kTeam>
__device__ __forceinline__ int element(const int t, const int i) {
    return i / kVector * (kVector * kTeam) + kVector * t + i % kVector;
}

// one word of a row. kWritten: of a tensor whose memory may be an output's too (the sum over the residual, a gradient over its
// upstream gradients), which the non-coherent path must not read.
template <bool kWritten, typename T>
__device__ __forceinline__ T load_word(const T* p) {
    if constexpr (kWritten) return *p;
    else return __ldg(p);
}

// a thread's elements of a row as they lie in memory: fetch only loads, value(i) converts. Elements past d are zero.
template <int kType, int kVector, int kTeam, int kHeld, bool kWritten>
struct Held {
    static constexpr int kPerWord = kVector > 1 && kType == kBf16 ? 2 : 1;
    uint32_t words[kHeld / kPerWord];

    __device__ __forceinline__ void fetch(const void* row, const int d, const int t) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += kVector) {
            const int j = element<kVector, kTeam>(t, i);
            const uint8_t* from = static_cast<const uint8_t*>(row) + static_cast<int64_t>(j) * kSize<kType>;
            uint32_t* to = words + i / kPerWord;
            if constexpr (kVector == 8) {
                #pragma unroll
                for (int q = 0; q < 2 / kPerWord; q++) {
                    const uint4 v = j + 8 <= d ? load_word<kWritten>(reinterpret_cast<const uint4*>(from) + q) : make_uint4(0, 0, 0, 0);
                    to[4 * q] = v.x, to[4 * q + 1] = v.y, to[4 * q + 2] = v.z, to[4 * q + 3] = v.w;
                }
            }
            else if constexpr (kVector == 2 && kType == kF32) {
                const uint2 v = j + 2 <= d ? load_word<kWritten>(reinterpret_cast<const uint2*>(from)) : make_uint2(0, 0);
                to[0] = v.x, to[1] = v.y;
            }
            else if constexpr (kVector == 2) to[0] = j + 2 <= d ? load_word<kWritten>(reinterpret_cast<const uint32_t*>(from)) : 0u;
            else to[0] = j < d ? bits(row, j) : 0u;
        }
        if (kVector > 1 && d % kVector != 0) {  // the last elements, in the team's thread whose access they do not fill
            #pragma unroll
            for (int i = 0; i < kHeld; i += kVector) {
                const int j = element<kVector, kTeam>(t, i);
                if (j >= d || j + kVector <= d) continue;
                #pragma unroll
                for (int e = 0; e < kVector; e++) {
                    const uint32_t v = j + e < d ? bits(row, j + e) : 0u;
                    if constexpr (kPerWord == 1) words[i + e] = v;
                    else words[(i + e) / 2] |= v << (e % 2 * 16);
                }
            }
        }
    }

    __device__ __forceinline__ float value(const int i) const {
        if constexpr (kType == kF32) return __uint_as_float(words[i]);
        else if constexpr (kPerWord == 2) return __uint_as_float(i % 2 ? words[i / 2] & 0xFFFF0000u : words[i / 2] << 16);
        else return __uint_as_float(words[i] << 16);
    }

private:
    static __device__ __forceinline__ uint32_t bits(const void* row, const int j) {
        if constexpr (kType == kF32) return load_word<kWritten>(static_cast<const uint32_t*>(row) + j);
        else return load_word<kWritten>(static_cast<const uint16_t*>(row) + j);
    }
};

// the same for codes, kPerWord of them in a word
template <int kVector, int kTeam, int kHeld>
struct HeldCodes {
    static constexpr int kPerWord = kVector == 8 ? 4 : kVector;
    uint32_t words[kHeld / kPerWord];

    __device__ __forceinline__ void fetch(const int8_t* row, const int d, const int t) {
        #pragma unroll
        for (int i = 0; i < kHeld; i += kVector) {
            const int j = element<kVector, kTeam>(t, i);
            uint32_t* to = words + i / kPerWord;
            if constexpr (kVector == 8) {
                const uint2 v = j + 8 <= d ? __ldg(reinterpret_cast<const uint2*>(row + j)) : make_uint2(0, 0);
                to[0] = v.x, to[1] = v.y;
            }
            else if constexpr (kVector == 2) to[0] = j + 2 <= d ? __ldg(reinterpret_cast<const uint16_t*>(row + j)) : 0u;
            else to[0] = j < d ? static_cast<uint8_t>(__ldg(row + j)) : 0u;
        }
        if (kVector > 1 && d % kVector != 0) {
            #pragma unroll
            for (int i = 0; i < kHeld; i += kVector) {
                const int j = element<kVector, kTeam>(t, i);
                if (j >= d || j + kVector <= d) continue;
                #pragma unroll
                for (int e = 0; e < kVector; e++) {
                    if (j + e < d) words[(i + e) / kPerWord] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(row + j + e))) << (8 * (e % kPerWord));
                }
            }
        }
    }

    // 2^23 + (code + 128) as a float without a conversion instruction, less 2^23 + 128: exact
    __device__ __forceinline__ float value(const int i) const {
        return __uint_as_float(__byte_perm(words[i / kPerWord] ^ 0x80808080u, 0x4B000000u, 0x7440u + i % kPerWord)) - 8388736.0f;
    }
};

template <int kType, int kVector, int kTeam, int kHeld>
__device__ __forceinline__ void store_row(void* row, const int d, const int t, const float (&v)[kHeld]) {
    #pragma unroll
    for (int i = 0; i < kHeld; i += kVector) {
        const int j = element<kVector, kTeam>(t, i);
        if (j + kVector <= d) {
            if constexpr (kVector == 8) store_eight<kType>(row, j, v + i);
            else if constexpr (kVector == 2 && kType == kF32) *reinterpret_cast<float2*>(static_cast<float*>(row) + j) = make_float2(v[i], v[i + 1]);
            else if constexpr (kVector == 2) *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(row) + j) = pack_bf16(v[i], v[i + 1]);
            else store_one<kType>(row, j, v[i]);
        }
        else {
            #pragma unroll
            for (int e = 0; e + 1 < kVector; e++) {
                if (j + e < d) store_one<kType>(row, j + e, v[i + e]);
            }
        }
    }
}

// rows that a team reduces side by side: a block all of its batch (one barrier), fewer threads one after the other (a row's
// stores leave while the next is worked on: 5 to 10 % faster at 256 columns)
template <int kTeam, int kRows>
constexpr int kTogether = kTeam > 32 ? kRows : 1;

// rows that a team fetches before it works on the first: about 32 elements of each operand per thread
template <int kHeld, int kOperands>
constexpr int kBatch = kHeld * kOperands >= 32 ? 1 : 32 / (kHeld * kOperands);

// the rows of x (kNorm: the normalised rows of x + residual) as codes and scales
template <int kX, int kResidual, bool kNorm, int kVector, int kTeam, int kHeld>
__global__ void __launch_bounds__(kTeamBlock<kTeam>) fz_quantize_kernel(const QuantizeArgs a) {
    constexpr int kRows = kBatch<kHeld, kResidual != kNone ? 2 : 1>;
    __shared__ uint32_t shared[2][kTogether<kTeam, kRows>][kMaxWarps];
    constexpr int kSide = kTogether<kTeam, kRows>;
    using Rows = Team<kTeam, kSide>;
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    // a team's rows: the teams of a block side by side, kRows times
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kTeamBlock<kTeam> / kTeam * kRows) + threadIdx.x / kTeam;
    if (first >= a.n) return;  // a team without rows: the reductions are a team's own
    auto row_at = [&](const int b) { return first + b * (kTeamBlock<kTeam> / kTeam); };
    Held<kX, kVector, kTeam, kHeld, false> x[kRows];
    Held<kResidual != kNone ? kResidual : kX, kVector, kTeam, kHeld, true> r[kRows];
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        // rows past the last repeat the team's own first one, which no other team writes, and write nothing
        const int64_t row = row_at(b) < a.n ? row_at(b) : first;
        x[b].fetch(row_of<kX>(a.x, row, a.x_stride), d, t);
        if constexpr (kResidual != kNone) r[b].fetch(row_of<kResidual>(a.residual, row, a.residual_stride), d, t);
    }
    #pragma unroll
    for (int of = 0; of < kRows; of += kSide) {
        float v[kSide][kHeld];
        #pragma unroll
        for (int b = 0; b < kSide; b++) {
            #pragma unroll
            for (int i = 0; i < kHeld; i++) v[b][i] = kResidual != kNone ? x[of + b].value(i) + r[of + b].value(i) : x[of + b].value(i);
            if constexpr (kResidual != kNone) {
                if (row_at(of + b) < a.n) store_row<kResidual, kVector, kTeam>(row_of<kResidual>(a.sum, row_at(of + b), a.sum_stride), d, t, v[b]);
            }
        }
        bool overflow[kSide] = {};
        if constexpr (kNorm) {
            float squares[kSide] = {};
            #pragma unroll
            for (int b = 0; b < kSide; b++) {
                #pragma unroll
                for (int i = 0; i < kHeld; i++) squares[b] = fmaf(v[b][i], v[b][i], squares[b]);
            }
            Rows::sum(squares, shared[0]);
            #pragma unroll
            for (int b = 0; b < kSide; b++) {
                overflow[b] = !(squares[b] <= FLT_MAX);
                const float rstd = overflow[b] ? __uint_as_float(0x7FFFFFFFu) : __frsqrt_rn(squares[b] * a.one_over_d + a.eps);
                if (t == 0 && a.rstd != nullptr && row_at(of + b) < a.n) a.rstd[row_at(of + b)] = rstd;
                #pragma unroll
                for (int i = 0; i < kHeld; i++) v[b][i] *= rstd;
            }
            if (a.weight != nullptr) {
                #pragma unroll
                for (int i = 0; i < kHeld; i++) {
                    const int j = element<kVector, kTeam>(t, i);
                    const float weight = j < d ? __ldg(a.weight + j) : 0.0f;
                    #pragma unroll
                    for (int b = 0; b < kSide; b++) v[b][i] *= weight;
                }
            }
        }
        uint32_t largest[kSide];
        #pragma unroll
        for (int b = 0; b < kSide; b++) {
            float magnitude = 0.0f;
            #pragma unroll
            for (int i = 0; i < kHeld; i++) magnitude = larger_magnitude(magnitude, v[b][i]);
            largest[b] = magnitude_bits(magnitude);
        }
        Rows::max(largest, shared[1]);
        #pragma unroll
        for (int b = 0; b < kSide; b++) {
            const int64_t row = row_at(of + b);
            if (row >= a.n) return;
            if (overflow[b]) largest[b] = kInfinityBits;
            Reciprocal to_codes;
            const float scale = row_scale(largest[b], a.power_of_two, to_codes);
            if (t == 0) a.scales[row] = scale;
            const uint32_t keep = largest[b] < kInfinityBits ? 0xFFFFFFFFu : 0u;  // the codes of a row that is not finite are zero
            int8_t* codes = a.codes + row * a.codes_stride;
            constexpr int kPairs = kVector > 1 ? kVector : 2;
            uint32_t pairs[kPairs];
            #pragma unroll
            for (int i = 0; i < kHeld; i += kVector) {
                const int j = element<kVector, kTeam>(t, i);
                if (i % kPairs == 0) {
                    #pragma unroll
                    for (int e = 0; e < kPairs; e += 2) to_codes_of(v[b][i + e], v[b][i + e + 1], to_codes, pairs[e], pairs[e + 1]);
                }
                const uint32_t* words = pairs + i % kPairs;
                if (j + kVector <= d) {
                    if constexpr (kVector == 8) {
                        *reinterpret_cast<uint2*>(codes + j) =
                            make_uint2(pack_codes(words[0], words[1], words[2], words[3]) & keep, pack_codes(words[4], words[5], words[6], words[7]) & keep);
                    }
                    else if constexpr (kVector == 2) *reinterpret_cast<uint16_t*>(codes + j) = static_cast<uint16_t>(__byte_perm(words[0], words[1], 0x0040u) & keep);
                    else codes[j] = static_cast<int8_t>(words[0] & keep);
                }
                else {
                    #pragma unroll
                    for (int e = 0; e + 1 < kVector; e++) {
                        if (j + e < d) codes[j + e] = static_cast<int8_t>(words[e] & keep);
                    }
                }
            }
        }
    }
}

// rows longer than a team holds: a block reads the row once per reduction and once more for the codes
template <int kX, int kResidual, bool kNorm>
__global__ void __launch_bounds__(kBlock) fz_long_quantize_kernel(const QuantizeArgs a) {
    __shared__ uint32_t shared[2][1][kMaxWarps];
    using Row = Team<kBlock, 1>;
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
        float squares[1] = {0.0f};
        for (int64_t j = threadIdx.x; j < a.d; j += kBlock) {
            const float v = value(j);
            squares[0] = fmaf(v, v, squares[0]);
        }
        Row::sum(squares, shared[0]);
        overflow = !(squares[0] <= FLT_MAX);
        rstd = overflow ? __uint_as_float(0x7FFFFFFFu) : __frsqrt_rn(squares[0] * a.one_over_d + a.eps);
        if (threadIdx.x == 0 && a.rstd != nullptr) a.rstd[row] = rstd;
    }
    auto scaled = [&](const float v, const int64_t j) {
        if constexpr (!kNorm) return v;
        else return a.weight != nullptr ? v * rstd * __ldg(a.weight + j) : v * rstd;
    };
    uint32_t largest[1] = {0};
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) largest[0] = max(largest[0], magnitude_bits(scaled(value(j), j)));
    Row::max(largest, shared[1]);
    if (overflow) largest[0] = kInfinityBits;
    Reciprocal to_codes;
    const float scale = row_scale(largest[0], a.power_of_two, to_codes);
    if (threadIdx.x == 0) a.scales[row] = scale;
    const bool finite = largest[0] < kInfinityBits;
    int8_t* codes = a.codes + row * a.codes_stride;
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) {
        const float v = value(j);
        // each thread reads an element of the residual for the last time before it writes the same element of the sum
        if constexpr (kResidual != kNone) store_one<kResidual>(row_of<kResidual>(a.sum, row, a.sum_stride), j, v);
        uint32_t code, unused;
        to_codes_of(scaled(v, j), 0.0f, to_codes, code, unused);
        codes[j] = static_cast<int8_t>(finite ? code : 0u);
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
__global__ void __launch_bounds__(kTeamBlock<kTeam>) fz_dequantize_kernel(const RestoreArgs a) {
    constexpr int kRows = kBatch<kHeld, 1>;
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kTeamBlock<kTeam> / kTeam * kRows) + threadIdx.x / kTeam;
    auto row_at = [&](const int b) { return first + b * (kTeamBlock<kTeam> / kTeam); };
    HeldCodes<8, kTeam, kHeld> codes[kRows];
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
        store_row<kOut, 8, kTeam>(row_of<kOut>(a.out, row_at(b), a.out_stride), d, t, v);
    }
}

template <int kOut, int kWord>
__global__ void __launch_bounds__(kBlock) fz_dequantize_flat_kernel(const RestoreArgs a) {
    const int64_t total = a.n * a.d;
    for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * kWord; at < total; at += static_cast<int64_t>(gridDim.x) * kBlock * kWord) {
        int64_t row = total <= UINT32_MAX ? static_cast<uint32_t>(at) / static_cast<uint32_t>(a.d) : at / a.d;
        int64_t j = at - row * a.d;
        float v[kWord];
        if (kWord == 8 && j + 8 <= a.d && row + 1 < a.n) {
            // eight codes of one row, from the aligned words around them (the last may reach into the next row)
            const uint32_t* words = reinterpret_cast<const uint32_t*>(a.codes + row * a.codes_stride + (j & ~int64_t{3}));
            const uint32_t shift = static_cast<uint32_t>(j & 3) * 8;
            const uint32_t w0 = __ldg(words), w1 = __ldg(words + 1), w2 = shift != 0 ? __ldg(words + 2) : 0u;
            const uint32_t eight[2] = {__funnelshift_r(w0, w1, shift) ^ 0x80808080u, __funnelshift_r(w1, w2, shift) ^ 0x80808080u};
            const float scale = __ldg(a.scales + row);
            #pragma unroll
            for (int e = 0; e < kWord; e++) v[e] = (__uint_as_float(__byte_perm(eight[e / 4 % 2], 0x4B000000u, 0x7440u + e % 4)) - 8388736.0f) * scale;
        }
        else {
            #pragma unroll
            for (int e = 0; e < kWord; e++) {
                v[e] = at + e < total ? static_cast<float>(a.codes[row * a.codes_stride + j]) * __ldg(a.scales + row) : 0.0f;
                if (++j == a.d) j = 0, row++;
            }
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
template <int kGrad, int kResidual, int kVector, int kTeam, int kHeld>
__global__ void __launch_bounds__(kTeamBlock<kTeam>) fz_norm_backward_kernel(const BackwardArgs a) {
    constexpr int kOut = kResidual != kNone ? kResidual : kGrad;
    constexpr int kRows = kBatch<kHeld, 2>;
    constexpr int kSide = kTogether<kTeam, kRows>;
    __shared__ uint32_t shared[kSide][kMaxWarps];
    const int t = threadIdx.x % kTeam;
    const int d = static_cast<int>(a.d);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kTeamBlock<kTeam> / kTeam * kRows) + threadIdx.x / kTeam;
    if (first >= a.n) return;  // a team without rows: the reductions are a team's own
    auto row_at = [&](const int b) { return first + b * (kTeamBlock<kTeam> / kTeam); };
    Held<kGrad, kVector, kTeam, kHeld, true> grad[kRows];
    HeldCodes<kVector, kTeam, kHeld> codes[kRows];
    Held<kOut, kVector, kTeam, kHeld, true> r[kRows];
    float scales[kRows], rstds[kRows];
    #pragma unroll
    for (int b = 0; b < kRows; b++) {
        // rows past the last repeat the team's own first one, which no other team writes, and write nothing
        const int64_t row = row_at(b) < a.n ? row_at(b) : first;
        grad[b].fetch(row_of<kGrad>(a.grad, row, a.grad_stride), d, t);
        codes[b].fetch(a.codes + row * a.codes_stride, d, t);
        if constexpr (kResidual != kNone) r[b].fetch(row_of<kResidual>(a.grad_residual, row, a.grad_residual_stride), d, t);
        scales[b] = __ldg(a.scales + row);
        rstds[b] = __ldg(a.rstd + row);
    }
    #pragma unroll
    for (int of = 0; of < kRows; of += kSide) {
        float mean[kSide] = {};
        #pragma unroll
        for (int b = 0; b < kSide; b++) {
            #pragma unroll
            for (int i = 0; i < kHeld; i++) mean[b] = fmaf(grad[of + b].value(i), codes[of + b].value(i) * scales[of + b], mean[b]);
        }
        Team<kTeam, kSide>::sum(mean, shared);
        #pragma unroll
        for (int b = 0; b < kSide; b++) {
            const int64_t row = row_at(of + b);
            if (row >= a.n) return;
            mean[b] *= a.one_over_d;
            float g[kHeld];
            #pragma unroll
            for (int i = 0; i < kHeld; i++) {
                g[i] = rstds[of + b] * fmaf(-(codes[of + b].value(i) * scales[of + b]), mean[b], grad[of + b].value(i));
                if constexpr (kResidual != kNone) g[i] += r[of + b].value(i);
            }
            store_row<kOut, kVector, kTeam>(row_of<kOut>(a.grad_x, row, a.grad_x_stride), d, t, g);
        }
    }
}

template <int kGrad, int kResidual>
__global__ void __launch_bounds__(kBlock) fz_long_norm_backward_kernel(const BackwardArgs a) {
    constexpr int kOut = kResidual != kNone ? kResidual : kGrad;
    __shared__ uint32_t shared[1][kMaxWarps];
    const int64_t row = blockIdx.x;
    const void* grad = row_of<kGrad>(a.grad, row, a.grad_stride);
    const int8_t* codes = a.codes + row * a.codes_stride;
    const float scale = __ldg(a.scales + row), rstd = __ldg(a.rstd + row);
    float dot[1] = {0.0f};
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) dot[0] = fmaf(load_one<kGrad>(grad, j), static_cast<float>(codes[j]) * scale, dot[0]);
    Team<kBlock, 1>::sum(dot, shared);
    const float mean = dot[0] * a.one_over_d;
    void* out = row_of<kOut>(a.grad_x, row, a.grad_x_stride);
    for (int64_t j = threadIdx.x; j < a.d; j += kBlock) {
        float g = rstd * fmaf(-static_cast<float>(codes[j]) * scale, mean, load_one<kGrad>(grad, j));
        if constexpr (kResidual != kNone) g += load_one<kResidual>(row_of<kResidual>(a.grad_residual, row, a.grad_residual_stride), j);
        store_one<kOut>(out, j, g);
    }
}

// ---------------------------------------------------------------------------------------------------------------------

// elements per access that the rows of a tensor allow
int width_of(const void* p, const int64_t stride, const int size) {
    const uintptr_t address = reinterpret_cast<uintptr_t>(p);
    if (address % 16 == 0 && stride * size % 16 == 0) return 8;
    return address % (2 * size) == 0 && stride % 2 == 0 ? 2 : 1;
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

// the team that holds rows of d elements, of which each thread holds `held`. With wide accesses a few threads that hold
// more are faster (a reduction inside a warp needs no barrier; 48,336 x 592 bf16: 41 us in warps of 32 held, 54 in blocks of
// 128 threads); with narrow ones more threads are (48,335 x 585: 135 against 75 us), as a thread's accesses are many.
template <int kVector, typename Launch, typename LaunchLong>
void with_team(const int64_t d, const Launch& launch, const LaunchLong& launch_long) {
    using std::integral_constant;
    constexpr bool kWide = kVector == 8;
    if (d <= 64) launch(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (d <= 128) launch(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (d <= 256) launch(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (d <= 512) launch(integral_constant<int, 32>{}, integral_constant<int, 16>{});
    else if (d <= 1024) launch(integral_constant<int, kWide ? 32 : 128>{}, integral_constant<int, kWide ? 32 : 8>{});
    else if (d <= 2048) launch(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    else if (d <= 4096) launch(integral_constant<int, 256>{}, integral_constant<int, 16>{});
    else if (d <= 8192) launch(integral_constant<int, kWide ? 256 : 512>{}, integral_constant<int, kWide ? 32 : 16>{});
    else launch_long();
}

// elements per access: 8, 2 or 1
template <typename Launch>
void with_vector(const int vector, const Launch& launch) {
    using std::integral_constant;
    if (vector == 8) launch(integral_constant<int, 8>{});
    else if (vector == 2) launch(integral_constant<int, 2>{});
    else launch(integral_constant<int, 1>{});
}

template <int kX, int kResidual, bool kNorm>
cudaError_t launch_quantize(const QuantizeArgs& a, const int vector, cudaStream_t stream) {
    with_vector(vector, [&](const auto width) {
        constexpr int kVector = decltype(width)::value;
        with_team<kVector>(
            a.d,
            [&](const auto team, const auto held) {
                constexpr int kTeam = decltype(team)::value, kHeld = decltype(held)::value;
                constexpr int kRows = kTeamBlock<kTeam> / kTeam * kBatch<kHeld, kResidual != kNone ? 2 : 1>;
                const unsigned blocks = static_cast<unsigned>((a.n + kRows - 1) / kRows);
                fz_quantize_kernel<kX, kResidual, kNorm, kVector, kTeam, kHeld><<<blocks, kTeamBlock<kTeam>, 0, stream>>>(a);
            },
            [&] { fz_long_quantize_kernel<kX, kResidual, kNorm><<<static_cast<unsigned>(a.n), kBlock, 0, stream>>>(a); });
    });
    return cudaGetLastError();
}

template <int kGrad, int kResidual>
cudaError_t launch_backward(const BackwardArgs& a, const int vector, cudaStream_t stream) {
    with_vector(vector, [&](const auto width) {
        constexpr int kVector = decltype(width)::value;
        with_team<kVector>(
            a.d,
            [&](const auto team, const auto held) {
                constexpr int kTeam = decltype(team)::value, kHeld = decltype(held)::value;
                constexpr int kRows = kTeamBlock<kTeam> / kTeam * kBatch<kHeld, 2>;
                const unsigned blocks = static_cast<unsigned>((a.n + kRows - 1) / kRows);
                fz_norm_backward_kernel<kGrad, kResidual, kVector, kTeam, kHeld><<<blocks, kTeamBlock<kTeam>, 0, stream>>>(a);
            },
            [&] { fz_long_norm_backward_kernel<kGrad, kResidual><<<static_cast<unsigned>(a.n), kBlock, 0, stream>>>(a); });
    });
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
        with_team<8>(
            a.d,
            [&](const auto team, const auto held) {
                constexpr int kTeam = decltype(team)::value, kHeld = decltype(held)::value;
                constexpr int kRows = kTeamBlock<kTeam> / kTeam * kBatch<kHeld, 1>;
                fz_dequantize_kernel<kOut, kTeam, kHeld><<<static_cast<unsigned>((a.n + kRows - 1) / kRows), kTeamBlock<kTeam>, 0, stream>>>(a);
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
    if (!zf::aligned_as<float>(args->scales)) return invalid("quantize_rows: misaligned scales");
    QuantizeArgs a{};
    a.x = args->x;
    a.x_stride = args->x_stride;
    a.n = args->n;
    a.d = args->d;
    a.power_of_two = args->power_of_two != 0;
    a.codes = args->codes;
    a.codes_stride = args->codes_stride;
    a.scales = args->scales;
    const int vector = width_of(args->x, args->x_stride, size_of(args->x_dtype));
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
    if (!zf::aligned_as<float>(args->scales)) return invalid("dequantize_rows: misaligned scales");
    if (!valid_rows(args->out, args->out_dtype, args->out_stride, args->d)) return invalid("dequantize_rows: invalid output");
    const RestoreArgs a{args->codes, args->codes_stride, args->scales, args->n, args->d, args->out, args->out_stride};
    const bool vector = width_of(args->out, args->out_stride, size_of(args->out_dtype)) == 8;
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
    if (!zf::aligned_as<float>(args->scales, args->weight, args->rstd)) return invalid("rms_norm_int8: misaligned scales, weight or rstd");
    const QuantizeArgs a{args->x, args->x_stride, args->residual, args->residual_stride, args->weight, args->n, args->d, 1.0f / static_cast<float>(args->d), args->eps,
                         args->power_of_two != 0, args->codes, args->codes_stride, args->scales, args->sum, args->sum_stride, args->rstd};
    const bool residual = args->residual != nullptr;
    const int size = size_of(args->residual_dtype);
    int vector = width_of(args->x, args->x_stride, size_of(args->x_dtype));
    if (residual) vector = std::min({vector, width_of(args->residual, args->residual_stride, size), width_of(args->sum, args->sum_stride, size)});
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
    if (!zf::aligned_as<float>(args->scales, args->rstd)) return invalid("rms_norm_int8_backward: misaligned scales or rstd");
    const int out_dtype = residual ? args->grad_residual_dtype : args->grad_dtype;
    if (!valid_rows(args->grad_x, out_dtype, args->grad_x_stride, args->d)) return invalid("rms_norm_int8_backward: invalid grad_x");
    const BackwardArgs a{args->grad, args->grad_stride, args->codes, args->codes_stride, args->scales, args->rstd, args->grad_residual,
                         args->grad_residual_stride, args->n, args->d, 1.0f / static_cast<float>(args->d), args->grad_x, args->grad_x_stride};
    int vector = std::min(width_of(args->grad, args->grad_stride, size_of(args->grad_dtype)), width_of(args->grad_x, args->grad_x_stride, size_of(out_dtype)));
    if (residual) vector = std::min(vector, width_of(args->grad_residual, args->grad_residual_stride, size_of(args->grad_residual_dtype)));
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
