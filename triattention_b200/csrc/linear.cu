// Product of INT8 code rows with one scale per token and one per channel:
//   out[t][n] = round( (sum_k c[t][k] d[n][k]) * sd[n] * sc[t] + bias[n] + residual[t][n] )
// The sum over k is an exact 32-bit integer: |c d| <= 128 * 128, so width <= 131071 cannot overflow, and its value does not
// depend on the order of the additions.  The rest is fp32, rounded once.
#include "common.cuh"
#include "abi_internal.h"

namespace tri {

constexpr int LinTile = 64, LinDepth = 64, LinThreads = 256;   // 64 tokens x 64 channels per CTA, 64 bytes of width per step

template <typename T> __device__ __forceinline__ T lin_out(float x);
template <> __device__ __forceinline__ __nv_bfloat16 lin_out(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half lin_out(float x) { return __float2half(x); }
template <> __device__ __forceinline__ float lin_out(float x) { return x; }
__device__ __forceinline__ float lin_in(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float lin_in(__half x) { return __half2float(x); }
__device__ __forceinline__ float lin_in(float x) { return x; }

struct LinearArgs {
  const int8_t *codes, *weight;
  int64_t codes_stride, weight_stride, residual_stride, out_stride;
  const float *scales, *weight_scales;
  const void *bias, *residual;
  void* out;
  int tokens, outputs, width;
};

// CUDA-core product (dp4a), one 4 x 4 block of outputs per thread.
template <typename T> __global__ void __launch_bounds__(LinThreads) linear_kernel(const LinearArgs p) {
  __shared__ int a[LinDepth / 4][LinTile + 1], b[LinDepth / 4][LinTile + 1];
  const int t0 = blockIdx.y * LinTile, n0 = blockIdx.x * LinTile, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.width; k0 += LinDepth) {
    __syncthreads();
    for (int i = threadIdx.x; i < LinTile * LinDepth / 4; i += LinThreads) {
      const int r = i / (LinDepth / 4), w = i % (LinDepth / 4), k = k0 + 4 * w;
      uint32_t va = 0, vb = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (k + j < p.width && t0 + r < p.tokens) va |= (uint32_t)(uint8_t)p.codes[(int64_t)(t0 + r) * p.codes_stride + k + j] << (8 * j);
        if (k + j < p.width && n0 + r < p.outputs) vb |= (uint32_t)(uint8_t)p.weight[(int64_t)(n0 + r) * p.weight_stride + k + j] << (8 * j);
      }
      a[w][r] = (int)va; b[w][r] = (int)vb;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LinDepth / 4; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[w][ty + 16 * i], b[w][tx + 16 * j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (t >= p.tokens || n >= p.outputs) continue;
      float y = (float)acc[i][j] * p.weight_scales[n] * p.scales[t];
      if (p.bias != nullptr) y += lin_in(static_cast<const T*>(p.bias)[n]);
      if (p.residual != nullptr) y += lin_in(static_cast<const T*>(p.residual)[(int64_t)t * p.residual_stride + n]);
      static_cast<T*>(p.out)[(int64_t)t * p.out_stride + n] = lin_out<T>(y);
    }
}

}  // namespace tri

using namespace tri;

extern "C" int tri_int8_linear(const void* codes, int64_t codes_stride, const float* scales, const void* weight,
    int64_t weight_stride, const float* weight_scales, const void* bias, const void* residual, int64_t residual_stride, void* out,
    int64_t out_stride, int type, int64_t tokens, int outputs, int width, int* device_error, void* stream) {
  TRI_CHECK(tokens >= 0 && tokens <= 0x7fffff00 && outputs > 0 && outputs <= 0x7fffff00 && width > 0 && width <= TRI_MAX_WIDTH &&
                type >= TRI_BF16 && type <= TRI_FP32,
            "int8_linear: tokens, outputs, width 1..131071, type");
  if (tokens == 0) return TRI_OK;
  TRI_CHECK(codes && scales && weight && weight_scales && out && device_error, "int8_linear: null buffers");
  TRI_CHECK(aligned16(codes) && aligned16(weight) && codes_stride % 16 == 0 && weight_stride % 16 == 0 && weight_stride >= width &&
                codes_stride >= width,
            "int8_linear: code rows start on 16-byte boundaries");
  const uintptr_t cell = type == TRI_FP32 ? 4 : 2;
  TRI_CHECK(reinterpret_cast<uintptr_t>(out) % cell == 0 && reinterpret_cast<uintptr_t>(bias) % cell == 0 &&
                reinterpret_cast<uintptr_t>(residual) % cell == 0,
            "int8_linear: output, bias and residual alignment");
  TRI_CHECK(out_stride >= outputs && (residual == nullptr || residual_stride >= 0), "int8_linear: output and residual rows");
  const LinearArgs p{static_cast<const int8_t*>(codes), static_cast<const int8_t*>(weight), codes_stride, weight_stride, residual_stride,
                     out_stride, scales, weight_scales, bias, residual, out, (int)tokens, outputs, width};
  const dim3 grid((outputs + LinTile - 1) / LinTile, ((unsigned)tokens + LinTile - 1) / LinTile);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == TRI_BF16) linear_kernel<__nv_bfloat16><<<grid, LinThreads, 0, s>>>(p);
  else if (type == TRI_FP16) linear_kernel<__half><<<grid, LinThreads, 0, s>>>(p);
  else linear_kernel<float><<<grid, LinThreads, 0, s>>>(p);
  return tri_launch_status("int8_linear");
}
