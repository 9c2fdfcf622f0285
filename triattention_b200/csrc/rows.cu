// Rows as INT8 codes: the operands of tri_int8_linear, made from activations (or weights).
//
//   rows    y = x
//   gated   y = g / (1 + e^-g) * u
//   norm    h = round(x + r),  y = h * rsqrt(mean h^2 + eps) * w
//   codes   s = max|y| / 127,  c = rint(y / s)      symmetric, one scale per row
//
// A row of zeros has scale 0 and codes 0; so has one whose largest magnitude is below 2^-119, where max/127 would leave the
// range of normal floats.  A row that holds a NaN or an infinity, or whose y overflows, has scale NaN and codes 0: every product
// that reads it is NaN, and no other row is touched by it.
// All arithmetic is IEEE fp32 (this file is compiled without --use_fast_math): the codes of plain and gated rows are, bit for
// bit, rint(y / s) of the formulas above with s = max|y| * fl(1/127) and CUDA's expf.  A row's largest element can be eighty
// times its root mean square, so a code that is off by one step where y / s is next to a tie would be off by more than half
// of that.  h is rounded to the stream's type before it is normed, because that is what later layers read.
#include "common.cuh"
#include "abi_internal.h"

namespace tri {

enum RowMode : int { RowPlain = 0, RowGated = 1, RowNorm = 2 };
constexpr int RowThreads = 256;
constexpr float RowTiny = 1.504632769052528e-36f;   // 2^-119
constexpr float RowLargestScale = 0x1.0204060000000p+121f;   // the largest float of which 127 times is no infinity

template <typename T> __device__ __forceinline__ float row_to_float(T x);
template <> __device__ __forceinline__ float row_to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float row_to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float row_to_float(float x) { return x; }
template <typename T> __device__ __forceinline__ T row_from_float(float x);
template <> __device__ __forceinline__ __nv_bfloat16 row_from_float(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half row_from_float(float x) { return __float2half(x); }
template <> __device__ __forceinline__ float row_from_float(float x) { return x; }

struct RowArgs {
  const void *a, *b, *weight;         // x | gate, residual | up (or null), norm weight
  int64_t a_stride, b_stride;         // elements
  void* sum;                          // norm: the new residual stream (or null)
  int64_t sum_stride;
  int8_t* codes;
  int64_t codes_stride;               // bytes
  float* scales;
  int width;
  float eps;
};

// Largest magnitude as the bits of |y|: an integer maximum, so that a NaN (whose bits lie above every number's) survives.
__device__ __forceinline__ uint32_t magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// Sum and maximum over the CTA; every thread gets both.
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& peak, float* sums, uint32_t* peaks) {
#pragma unroll
  for (int bit = 16; bit > 0; bit >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, bit);
    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, bit));
  }
  const int warps = blockDim.x / 32, warp = threadIdx.x / 32;
  __syncthreads();                    // the arrays may still be read from the call before
  if (threadIdx.x % 32 == 0) { sums[warp] = sum; peaks[warp] = peak; }
  __syncthreads();
  sum = 0.f; peak = 0;
  for (int i = 0; i < warps; ++i) { sum += sums[i]; peak = max(peak, peaks[i]); }
}

// y of element e up to the norm's common factor; adds the element's square to `squares` (norm only).
template <typename T, int Mode>
__device__ __forceinline__ float row_element(const RowArgs& p, const T* a, const T* b, T* sum, int e, float shift, float& squares) {
  if constexpr (Mode == RowPlain) return row_to_float(a[e]);
  if constexpr (Mode == RowGated) {
    const float g = row_to_float(a[e]);
    return g / (1.f + expf(-g)) * row_to_float(b[e]);
  }
  float h = row_to_float(a[e]);
  if (b != nullptr) {
    const T rounded = row_from_float<T>(h + row_to_float(b[e]));
    if (sum != nullptr) sum[e] = rounded;
    h = row_to_float(rounded);
  }
  h *= shift;
  squares = fmaf(h, h, squares);
  return h * row_to_float(static_cast<const T*>(p.weight)[e]);
}

// One CTA per row, two passes over it (the second from cache).
template <typename T, int Mode> __global__ void __launch_bounds__(RowThreads) rows_kernel(const RowArgs p) {
  __shared__ float sums[RowThreads / 32];
  __shared__ uint32_t peaks[RowThreads / 32];
  const int64_t row = blockIdx.x;
  const T* a = static_cast<const T*>(p.a) + row * p.a_stride;
  const T* b = p.b == nullptr ? nullptr : static_cast<const T*>(p.b) + row * p.b_stride;
  T* sum = p.sum == nullptr ? nullptr : static_cast<T*>(p.sum) + row * p.sum_stride;
  float shift = 1.f, squares;
  uint32_t peak;
  // A norm whose squares leave fp32's range (|h| above 1e19 or so, or so small that they flush to zero) is done again with
  // h scaled by a power of two, which rsqrt and eps undo exactly.
  for (int attempt = 0; attempt < 2; ++attempt) {
    squares = 0.f; peak = 0;
    for (int e = threadIdx.x; e < p.width; e += RowThreads)
      peak = max(peak, magnitude(row_element<T, Mode>(p, a, b, sum, e, shift, squares)));
    row_reduce(squares, peak, sums, peaks);
    if (Mode == RowNorm && sum != nullptr) { a = sum; b = nullptr; sum = nullptr; }   // from here on h is read (a thread reads
                                                                                      // what it wrote; residual may be gone)
    if (Mode != RowNorm || (squares < 3e38f && squares > 1e-24f) || (squares == 0.f && peak == 0)) break;
    shift = squares > 1.f || squares != squares ? 8.271806125530277e-25f : 1.152921504606847e18f;   // 2^-80, 2^60
  }
  const float largest = __uint_as_float(peak);
  float factor = 1.f;
  if (Mode == RowNorm) factor = __frsqrt_rn(__fdiv_rn(squares, (float)p.width) + p.eps * shift * shift);
  const bool finite = peak < 0x7f800000u && (Mode != RowNorm || squares < 3e38f);
  const bool zero = largest < RowTiny || (Mode == RowNorm && squares == 0.f && p.eps == 0.f);
  const float scale = !finite ? CUDART_NAN_F : zero ? 0.f : fminf(largest * (1.f / 127.f) * factor, RowLargestScale);
  const float inverse = !finite || zero ? 0.f : __fdiv_rn(127.f, largest);
  if (threadIdx.x == 0) p.scales[row] = scale;
  int8_t* codes = p.codes + row * p.codes_stride;
  for (int e = threadIdx.x; e < p.width; e += RowThreads) {
    const float y = row_element<T, Mode>(p, a, b, sum, e, shift, squares);
    codes[e] = finite && !zero ? (int8_t)__float2int_rn(Mode == RowNorm ? y * inverse : y / scale) : (int8_t)0;
  }
}

template <typename T> __global__ void __launch_bounds__(RowThreads) dequantize_rows_kernel(const int8_t* codes, int64_t codes_stride,
    const float* scales, T* out, int64_t out_stride, int width) {
  const int64_t row = blockIdx.x;
  const float scale = scales[row];
  for (int e = threadIdx.x; e < width; e += RowThreads)
    out[row * out_stride + e] = row_from_float<T>((float)codes[row * codes_stride + e] * scale);
}

static int launch_rows(int mode, int type, int64_t rows, const RowArgs& p, cudaStream_t s) {
  const unsigned grid = (unsigned)rows;
#define TRI_ROWS(T, M) rows_kernel<T, M><<<grid, RowThreads, 0, s>>>(p)
#define TRI_ROWS_TYPE(M)                                                                      \
  do {                                                                                        \
    if (type == TRI_BF16) TRI_ROWS(__nv_bfloat16, M);                                         \
    else if (type == TRI_FP16) TRI_ROWS(__half, M);                                           \
    else TRI_ROWS(float, M);                                                                  \
  } while (0)
  if (mode == RowPlain) TRI_ROWS_TYPE(RowPlain);
  else if (mode == RowGated) TRI_ROWS_TYPE(RowGated);
  else TRI_ROWS_TYPE(RowNorm);
#undef TRI_ROWS_TYPE
#undef TRI_ROWS
  return tri_launch_status("rows");
}

}  // namespace tri

using namespace tri;

static bool row_shape(int64_t rows, int width) { return rows >= 0 && rows <= 0x7fffffff && width > 0 && width <= TRI_MAX_WIDTH; }
static bool code_rows(const void* codes, int64_t stride, int width) { return aligned16(codes) && stride % 16 == 0 && stride >= width; }
static bool row_type(int type) { return type >= TRI_BF16 && type <= TRI_FP32; }
static bool row_pointer(const void* p, int type) { return reinterpret_cast<uintptr_t>(p) % (type == TRI_FP32 ? 4 : 2) == 0; }

extern "C" int tri_quantize_rows(const void* x, int type, int64_t rows, int width, int64_t x_stride, void* codes,
    int64_t codes_stride, float* scales, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "quantize_rows: rows, width 1..131071, type");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(x && codes && scales, "quantize_rows: null buffers");
  TRI_CHECK(row_pointer(x, type) && x_stride >= 0, "quantize_rows: input rows");
  TRI_CHECK(code_rows(codes, codes_stride, width), "quantize_rows: code rows start on 16-byte boundaries");
  RowArgs p{};
  p.a = x; p.a_stride = x_stride; p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width;
  return launch_rows(RowPlain, type, rows, p, static_cast<cudaStream_t>(stream));
}

extern "C" int tri_silu_mul_rows(const void* gate, const void* up, int type, int64_t rows, int width, int64_t gate_stride,
    int64_t up_stride, void* codes, int64_t codes_stride, float* scales, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "silu_mul_rows: rows, width 1..131071, type");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(gate && up && codes && scales, "silu_mul_rows: null buffers");
  TRI_CHECK(row_pointer(gate, type) && row_pointer(up, type) && gate_stride >= 0 && up_stride >= 0, "silu_mul_rows: input rows");
  TRI_CHECK(code_rows(codes, codes_stride, width), "silu_mul_rows: code rows start on 16-byte boundaries");
  RowArgs p{};
  p.a = gate; p.b = up; p.a_stride = gate_stride; p.b_stride = up_stride;
  p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width;
  return launch_rows(RowGated, type, rows, p, static_cast<cudaStream_t>(stream));
}

extern "C" int tri_rms_norm_rows(const void* x, const void* residual, const void* weight, int type, int64_t rows, int width,
    int64_t x_stride, int64_t residual_stride, double eps, void* residual_out, int64_t residual_out_stride, void* codes,
    int64_t codes_stride, float* scales, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "rms_norm_rows: rows, width 1..131071, type");
  TRI_CHECK(eps >= 0. && eps <= 1., "rms_norm_rows: eps 0..1");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(x && weight && codes && scales, "rms_norm_rows: null buffers");
  TRI_CHECK((residual == nullptr) == (residual_out == nullptr), "rms_norm_rows: the residual and where its sum goes (both or none)");
  TRI_CHECK(row_pointer(x, type) && row_pointer(residual, type) && row_pointer(weight, type) && row_pointer(residual_out, type) &&
                x_stride >= 0 && residual_stride >= 0,
            "rms_norm_rows: input rows");
  TRI_CHECK(residual == nullptr || residual_out_stride >= width, "rms_norm_rows: rows of the new residual overlap");
  TRI_CHECK(code_rows(codes, codes_stride, width), "rms_norm_rows: code rows start on 16-byte boundaries");
  RowArgs p{};
  p.a = x; p.b = residual; p.weight = weight; p.a_stride = x_stride; p.b_stride = residual_stride;
  p.sum = residual_out; p.sum_stride = residual_out_stride;
  p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width; p.eps = (float)eps;
  return launch_rows(RowNorm, type, rows, p, static_cast<cudaStream_t>(stream));
}

extern "C" int tri_dequantize_rows(const void* codes, int64_t codes_stride, const float* scales, int type, int64_t rows, int width,
    void* out, int64_t out_stride, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "dequantize_rows: rows, width 1..131071, type");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(codes && scales && out, "dequantize_rows: null buffers");
  TRI_CHECK(code_rows(codes, codes_stride, width), "dequantize_rows: code rows start on 16-byte boundaries");
  TRI_CHECK(row_pointer(out, type) && out_stride >= width, "dequantize_rows: output rows");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = (unsigned)rows;
  const int8_t* c = static_cast<const int8_t*>(codes);
  if (type == TRI_BF16) dequantize_rows_kernel<<<grid, RowThreads, 0, s>>>(c, codes_stride, scales, static_cast<__nv_bfloat16*>(out), out_stride, width);
  else if (type == TRI_FP16) dequantize_rows_kernel<<<grid, RowThreads, 0, s>>>(c, codes_stride, scales, static_cast<__half*>(out), out_stride, width);
  else dequantize_rows_kernel<<<grid, RowThreads, 0, s>>>(c, codes_stride, scales, static_cast<float*>(out), out_stride, width);
  return tri_launch_status("dequantize_rows");
}
