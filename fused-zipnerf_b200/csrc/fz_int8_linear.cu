// fz_int8_linear.cu -- the linear layer on int8 rows (zf_int8_linear): output = scales x weight_scales x (codes
// weight_codes^T) + bias, the integer products summed exactly.
#include "zf_int8.h"
#include "fz_status.h"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace zf::int8_linear {

constexpr int kTile = 64;       // rows and outputs of a block
constexpr int kDepth = 64;      // inputs per step
constexpr int kBlock = 256;     // each thread: 4 x 4 outputs

struct Args {
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    const int8_t* weight;
    int64_t weight_stride;
    const float* weight_scales;
    const float* bias;
    int64_t n, in, out;
    bool relu;
    void* output;
    int64_t output_stride;
};

// four codes at column k of a row (zeros past `in`)
__device__ __forceinline__ int four_codes(const int8_t* row, const int64_t k, const int64_t in) {
    if (k + 4 <= in) return *reinterpret_cast<const int*>(row + k);
    uint32_t v = 0;
    for (int e = 0; k + e < in; e++) v |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + e])) << (8 * e);
    return static_cast<int>(v);
}

template <typename Out>
__global__ void __launch_bounds__(kBlock) fz_int8_linear_kernel(const Args a) {
    __shared__ int x[kTile][kDepth / 4 + 1];
    __shared__ int w[kTile][kDepth / 4 + 1];
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile, out0 = static_cast<int64_t>(blockIdx.y) * kTile;
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    int sum[4][4] = {};
    for (int64_t k0 = 0; k0 < a.in; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth / 4; i += kBlock) {
            const int r = i / (kDepth / 4), c = i % (kDepth / 4);
            x[r][c] = row0 + r < a.n ? four_codes(a.codes + (row0 + r) * a.codes_stride, k0 + 4 * c, a.in) : 0;
            w[r][c] = out0 + r < a.out ? four_codes(a.weight + (out0 + r) * a.weight_stride, k0 + 4 * c, a.in) : 0;
        }
        __syncthreads();
        for (int c = 0; c < kDepth / 4; c++) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                #pragma unroll
                for (int j = 0; j < 4; j++) sum[i][j] = __dp4a(x[tr + 16 * i][c], w[tc + 16 * j][c], sum[i][j]);
            }
        }
        __syncthreads();
    }
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t r = row0 + tr + 16 * i;
        if (r >= a.n) continue;
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t o = out0 + tc + 16 * j;
            if (o >= a.out) continue;
            float v = static_cast<float>(sum[i][j]) * a.scales[r] * a.weight_scales[o];
            if (a.bias != nullptr) v += a.bias[o];
            if (a.relu && v < 0.0f) v = 0.0f;  // a comparison, so that a NaN stays one
            static_cast<Out*>(a.output)[r * a.output_stride + o] = static_cast<Out>(v);
        }
    }
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
    const int size = args->output_dtype == ZF_FLOAT32 ? 4 : 2;
    if ((args->output_dtype != ZF_FLOAT32 && args->output_dtype != ZF_BFLOAT16) || args->output == nullptr || args->output_stride < args->out
        || reinterpret_cast<uintptr_t>(args->output) % size != 0) {
        return invalid("int8_linear: invalid output");
    }
    const Args a{args->codes, args->codes_stride, args->scales, args->weight_codes, args->weight_stride, args->weight_scales, args->bias,
                 args->n, args->in, args->out, args->relu != 0, args->output, args->output_stride};
    const dim3 grid(static_cast<unsigned>((a.n + kTile - 1) / kTile), static_cast<unsigned>((a.out + kTile - 1) / kTile));
    if (grid.y > 65535) return invalid("int8_linear: invalid sizes");
    if (args->output_dtype == ZF_FLOAT32) fz_int8_linear_kernel<float><<<grid, kBlock, 0, stream>>>(a);
    else fz_int8_linear_kernel<__nv_bfloat16><<<grid, kBlock, 0, stream>>>(a);
    const cudaError_t error = cudaGetLastError();
    return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, "int8_linear");
}
