// fz_int8_weight_grad.cu -- the weight and bias gradient of a linear layer from the 8-bit checkpoint of its input
// (zf_int8_weight_grad): grad_weight += grad^T (codes x scales), grad_bias += column sums of grad.
#include "zf_int8.h"
#include "fz_status.h"

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

namespace zf::int8_weight_grad {

constexpr int kTile = 64;       // outputs and inputs of a block's part of grad_weight
constexpr int kRows = 32;       // samples per step
constexpr int kBlock = 256;     // each thread: 4 x 4 elements
constexpr int kMaxSplits = 256;

struct Args {
    const __nv_bfloat16* grad;
    int64_t grad_stride;
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    int64_t n, in, out;
    float* partial;         // [splits, out, in]
    float* bias_partial;    // [splits, out], or null
};

// split blockIdx.z of the samples: its part of the sums over a tile of grad_weight
__global__ void __launch_bounds__(kBlock) fz_int8_weight_grad_kernel(const Args a) {
    __shared__ float g[kRows][kTile], x[kRows][kTile];
    const int64_t out0 = static_cast<int64_t>(blockIdx.y) * kTile, in0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int64_t share = (a.n + gridDim.z - 1) / gridDim.z;
    const int64_t first = blockIdx.z * share, last = min(a.n, first + share);
    const int to = threadIdx.x / 16, ti = threadIdx.x % 16;
    float sum[4][4] = {}, bias = 0.0f;
    for (int64_t r0 = first; r0 < last; r0 += kRows) {
        for (int i = threadIdx.x; i < kRows * kTile; i += kBlock) {
            const int r = i / kTile, c = i % kTile;
            const int64_t row = r0 + r;
            g[r][c] = row < last && out0 + c < a.out ? __bfloat162float(a.grad[row * a.grad_stride + out0 + c]) : 0.0f;
            const float v = row < last && in0 + c < a.in ? static_cast<float>(a.codes[row * a.codes_stride + in0 + c]) * a.scales[row] : 0.0f;
            x[r][c] = __bfloat162float(__float2bfloat16_rn(v));
        }
        __syncthreads();
        for (int r = 0; r < kRows; r++) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                #pragma unroll
                for (int j = 0; j < 4; j++) sum[i][j] = fmaf(g[r][to + 16 * i], x[r][ti + 16 * j], sum[i][j]);
            }
            if (threadIdx.x < kTile) bias += g[r][threadIdx.x];
        }
        __syncthreads();
    }
    float* partial = a.partial + blockIdx.z * a.out * a.in;
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t o = out0 + to + 16 * i, k = in0 + ti + 16 * j;
            if (o < a.out && k < a.in) partial[o * a.in + k] = sum[i][j];
        }
    }
    if (a.bias_partial != nullptr && blockIdx.x == 0 && threadIdx.x < kTile && out0 + threadIdx.x < a.out) {
        a.bias_partial[blockIdx.z * a.out + out0 + threadIdx.x] = bias;
    }
}

// target[i] += the splits' sums in their order
__global__ void __launch_bounds__(kBlock) fz_int8_weight_grad_join_kernel(const float* partial, const int splits, const int64_t count, float* target) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x;
    if (i >= count) return;
    float sum = 0.0f;
    for (int s = 0; s < splits; s++) sum += partial[s * count + i];
    target[i] += sum;
}

int splits_of(const int64_t n, const int64_t in, const int64_t out) {
    const int64_t tiles = ((in + kTile - 1) / kTile) * ((out + kTile - 1) / kTile);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kMaxSplits, (n + 4 * kRows - 1) / (4 * kRows), (1184 + tiles - 1) / tiles})));
}

int invalid(const char* message) { return zf::set_error(ZF_ERROR_INVALID_ARGUMENT, message); }

}  // namespace zf::int8_weight_grad

int64_t zf_int8_weight_grad_workspace_size(const int64_t n, const int64_t in, const int64_t out) {
    using namespace zf::int8_weight_grad;
    if (n <= 0 || in <= 0 || out <= 0) return 0;
    return splits_of(n, in, out) * (in + 1) * out * 4;
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
    const int splits = splits_of(args->n, args->in, args->out);
    float* partial = static_cast<float*>(args->workspace);
    float* bias_partial = args->grad_bias != nullptr ? partial + splits * args->in * args->out : nullptr;
    const Args a{reinterpret_cast<const __nv_bfloat16*>(args->grad), args->grad_stride, args->codes, args->codes_stride, args->scales, args->n, args->in,
                 args->out, partial, bias_partial};
    const dim3 grid(static_cast<unsigned>((a.in + kTile - 1) / kTile), static_cast<unsigned>((a.out + kTile - 1) / kTile), static_cast<unsigned>(splits));
    fz_int8_weight_grad_kernel<<<grid, kBlock, 0, stream>>>(a);
    const int64_t count = a.in * a.out;
    fz_int8_weight_grad_join_kernel<<<static_cast<unsigned>((count + kBlock - 1) / kBlock), kBlock, 0, stream>>>(partial, splits, count, args->grad_weight);
    if (bias_partial != nullptr) {
        fz_int8_weight_grad_join_kernel<<<static_cast<unsigned>((a.out + kBlock - 1) / kBlock), kBlock, 0, stream>>>(bias_partial, splits, a.out, args->grad_bias);
    }
    const cudaError_t error = cudaGetLastError();
    return error == cudaSuccess ? ZF_OK : zf::set_cuda_error(error, "int8_weight_grad");
}
