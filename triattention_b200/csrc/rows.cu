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
#include <type_traits>

namespace tri {

enum RowMode : int { RowPlain = 0, RowGated = 1, RowNorm = 2 };
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
  int64_t rows;
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

// silu(g) * u in IEEE arithmetic.  Below a gate of -87.3 the sum passes 2^126 and the product counts as zero (silu(g) is within
// 1e-36 of it): that is where the fast reciprocal of the kernel below ends.
__device__ __forceinline__ float gated(float g, float u) {
  const float d = 1.f + expf(-g);
  return d > 8.507059173023462e37f ? 0.f * g * u : g / d * u;      // (0 * g * u: an infinite gate or NaN stays one)
}

// Whether a sum of squares came out in fp32's range (false for NaN too).
__device__ __forceinline__ bool squares_fit(float squares) { return squares < 3e38f && squares > 1e-24f; }

struct RowScale {
  float scale, inverse;                 // inverse: 127 / max|y| before the norm's common factor
  bool live;                            // codes are not all zero
};
template <int Mode> __device__ __forceinline__ RowScale row_scale(uint32_t peak, float squares, float factor, float eps) {
  const float largest = __uint_as_float(peak);
  const bool finite = peak < 0x7f800000u && (Mode != RowNorm || squares < 3e38f);
  const bool zero = largest < RowTiny || (Mode == RowNorm && squares == 0.f && eps == 0.f);
  RowScale r;
  r.live = finite && !zero;
  r.scale = !finite ? CUDART_NAN_F : zero ? 0.f : fminf(largest * (1.f / 127.f) * factor, RowLargestScale);
  r.inverse = r.live ? __fdiv_rn(127.f, largest) : 0.f;
  return r;
}

// y of element e up to the norm's common factor; adds the element's square to `squares` (norm only).
template <typename T, int Mode>
__device__ __forceinline__ float row_element(const RowArgs& p, const T* a, const T* b, T* sum, int e, float shift, float& squares) {
  if constexpr (Mode == RowPlain) return row_to_float(a[e]);
  if constexpr (Mode == RowGated) return gated(row_to_float(a[e]), row_to_float(b[e]));
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

// ---- general form: one CTA per row, two passes over it (the second from cache), any width and alignment ------------------
template <typename T, int Mode> __device__ __noinline__ void row_general(const RowArgs& p, int64_t row, bool summed, float* sums,
                                                                         uint32_t* peaks) {
  const int threads = blockDim.x;
  const T* a = static_cast<const T*>(p.a) + row * p.a_stride;
  const T* b = p.b == nullptr ? nullptr : static_cast<const T*>(p.b) + row * p.b_stride;
  T* sum = p.sum == nullptr ? nullptr : static_cast<T*>(p.sum) + row * p.sum_stride;
  if (Mode == RowNorm && sum != nullptr && summed) { a = sum; b = nullptr; sum = nullptr; }
  float shift = 1.f, squares;
  uint32_t peak;
  // A norm whose squares leave fp32's range (|h| above 1e19 or so, or so small that they flush to zero) is done again with
  // h scaled by a power of two, which rsqrt and eps undo exactly.
  for (int attempt = 0; attempt < 2; ++attempt) {
    squares = 0.f; peak = 0;
    for (int e = threadIdx.x; e < p.width; e += threads)
      peak = max(peak, magnitude(row_element<T, Mode>(p, a, b, sum, e, shift, squares)));
    row_reduce(squares, peak, sums, peaks);
    if (Mode == RowNorm && sum != nullptr) { a = sum; b = nullptr; sum = nullptr; }   // from here on h is read (a thread reads
                                                                                      // what it wrote; residual may be gone)
    if (Mode != RowNorm || squares_fit(squares) || (squares == 0.f && peak == 0)) break;
    shift = squares > 1.f || squares != squares ? 8.271806125530277e-25f : 1.152921504606847e18f;   // 2^-80, 2^60
  }
  float factor = 1.f;
  if (Mode == RowNorm) factor = __frsqrt_rn(__fdiv_rn(squares, (float)p.width) + p.eps * shift * shift);
  const RowScale r = row_scale<Mode>(peak, squares, factor, p.eps);
  if (threadIdx.x == 0) p.scales[row] = r.scale;
  int8_t* codes = p.codes + row * p.codes_stride;
  for (int e = threadIdx.x; e < p.width; e += threads) {
    const float y = row_element<T, Mode>(p, a, b, sum, e, shift, squares);
    codes[e] = !r.live ? (int8_t)0 : (int8_t)__float2int_rn(Mode == RowNorm ? y * r.inverse : y / r.scale);
  }
}

template <typename T, int Mode> __global__ void __launch_bounds__(1024) rows_general_kernel(const RowArgs p) {
  __shared__ float sums[32];
  __shared__ uint32_t peaks[32];
  row_general<T, Mode>(p, blockIdx.x, false, sums, peaks);
}

// ---- rows held in registers ---------------------------------------------------------------------------------------------
// A thread holds V vectors of 16 bytes of the row (vector j of thread i is number j * threads + i), loaded at once, so the row
// is read from memory once whatever the mode.  Rows * width decides nothing here; the work is bound by HBM for long batches
// and by one round trip to memory plus one reduction for short ones.
// Gated: the y that a thread keeps are computed with the fast exponential and reciprocal (12 instead of 30 instructions per
// element, which would bound the kernel); they are within GatedError of the IEEE values.  Where that could show, at elements
// that may be the row's largest and at quotients next to a tie, the element is computed again in IEEE arithmetic.
constexpr float GatedError = 2e-5f;     // relative: __expf 2 + 1.17 |g| steps of 2^-23 with |g| < 88, reciprocal 2, rest 3: 1.3e-5
constexpr float PlainError = 3e-7f;     // y * (1/s) against y / s: three roundings of 2^-24
constexpr float Round = 12582912.f;     // 1.5 * 2^23: x + Round has rint(x) in its low bits

template <typename T> struct RowVector {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void unpack(float (&x)[N]) const {
    if constexpr (sizeof(T) == 4) {
      x[0] = __uint_as_float(raw.x); x[1] = __uint_as_float(raw.y); x[2] = __uint_as_float(raw.z); x[3] = __uint_as_float(raw.w);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
      }
    }
  }
  __device__ __forceinline__ void pack(const float (&x)[N]) {
    if constexpr (sizeof(T) == 4) {
      raw = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// One gated element in IEEE arithmetic, for the few that need it.
template <typename T> __device__ __noinline__ float gated_exact(const T* gate, const T* up, int e) {
  return gated(row_to_float(gate[e]), row_to_float(up[e]));
}

// Rows that start on 16-byte boundaries (all inputs) with a width of whole vectors.  Warp = true: a warp per row, several rows
// per CTA; otherwise a CTA per row.
template <typename T, int Mode, int V, bool Warp> __global__ void __launch_bounds__(Warp ? 128 : 1024) rows_kernel(const RowArgs p) {
  constexpr int N = RowVector<T>::N;
  __shared__ float sums[32];
  __shared__ uint32_t peaks[32];
  __shared__ uint32_t exact_peak;
  const int threads = Warp ? 32 : blockDim.x, me = Warp ? threadIdx.x % 32 : threadIdx.x;
  const int64_t row = Warp ? (int64_t)blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x;
  if (Warp && row >= p.rows) return;
  const int vectors = p.width / N;
  const T* a = static_cast<const T*>(p.a) + row * p.a_stride;
  const T* b = p.b == nullptr ? nullptr : static_cast<const T*>(p.b) + row * p.b_stride;
  RowVector<T> va[V], vb[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = j * threads + me;
    va[j].raw = v < vectors ? __ldcs(reinterpret_cast<const uint4*>(a) + v) : make_uint4(0, 0, 0, 0);
    if (Mode != RowPlain && b != nullptr) vb[j].raw = v < vectors ? __ldcs(reinterpret_cast<const uint4*>(b) + v) : make_uint4(0, 0, 0, 0);
  }
  if (!Warp && Mode == RowGated && threadIdx.x == 0) exact_peak = 0;
  float y[V][N], squares = 0.f;
  float largest = 0.f, odd = 0.f;      // odd turns NaN with any y that is not finite
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = j * threads + me;
    va[j].unpack(y[j]);
    if constexpr (Mode == RowGated) {
      float u[N];
      vb[j].unpack(u);
#pragma unroll
      for (int i = 0; i < N; ++i) y[j][i] = __fdividef(y[j][i], 1.f + __expf(-y[j][i])) * u[i];
    }
    if constexpr (Mode == RowNorm) {
      if (b != nullptr) {
        float r[N];
        vb[j].unpack(r);
#pragma unroll
        for (int i = 0; i < N; ++i) y[j][i] += r[i];
        RowVector<T> h;
        h.pack(y[j]);
        h.unpack(y[j]);
        if (v < vectors) reinterpret_cast<uint4*>(static_cast<T*>(p.sum) + row * p.sum_stride)[v] = h.raw;
      }
      RowVector<T> vw;
      vw.raw = v < vectors ? __ldg(reinterpret_cast<const uint4*>(p.weight) + v) : make_uint4(0, 0, 0, 0);
      float w[N];
      vw.unpack(w);
#pragma unroll
      for (int i = 0; i < N; ++i) { squares = fmaf(y[j][i], y[j][i], squares); y[j][i] *= w[i]; }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) { largest = fmaxf(largest, fabsf(y[j][i])); odd = fmaf(y[j][i], 0.f, odd); }
  }
  uint32_t peak = odd == 0.f ? __float_as_uint(largest) : 0x7fc00000u;
  if constexpr (Warp) {
#pragma unroll
    for (int bit = 16; bit > 0; bit >>= 1) {
      squares += __shfl_xor_sync(0xffffffffu, squares, bit);
      peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, bit));
    }
  } else {
    row_reduce(squares, peak, sums, peaks);
  }
  if constexpr (Mode == RowNorm && !Warp) {
    if (!squares_fit(squares) && !(squares == 0.f && peak == 0)) {      // (the same for the whole CTA)
      row_general<T, Mode>(p, row, b != nullptr, sums, peaks);
      return;
    }
  }
  if constexpr (Mode == RowGated) {
    if (peak != 0 && peak < 0x7f800000u) {
      const float bar = __uint_as_float(peak) * (1.f - 2.f * GatedError);
      uint32_t exact = 0;
      if (largest >= bar) {
        for (int j = 0; j < V; ++j) {
          const int v = j * threads + me;
          for (int i = 0; i < N; ++i)
            if (v < vectors && fabsf(reinterpret_cast<float(&)[V][N]>(y)[j][i]) >= bar) exact = max(exact, magnitude(gated_exact(a, b, v * N + i)));
        }
      }
      if constexpr (Warp) {
        peak = __reduce_max_sync(0xffffffffu, exact);
      } else {
        if (exact != 0) atomicMax(&exact_peak, exact);
        __syncthreads();
        peak = exact_peak;
      }
    }
  }
  const float factor = Mode == RowNorm ? __frsqrt_rn(__fdiv_rn(squares, (float)p.width) + p.eps) : 1.f;
  const RowScale r = row_scale<Mode>(peak, squares, factor, p.eps);
  if (me == 0) p.scales[row] = r.scale;
  const float inverse = Mode == RowNorm ? r.inverse : r.live ? __frcp_rn(r.scale) : 0.f;
  int8_t* codes = p.codes + row * p.codes_stride;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int v = j * threads + me;
    uint32_t c[N];
    float off = 0.f;                    // above 0.5: some quotient may lie on the other side of a tie
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float q = y[j][i] * inverse, up = q + Round;
      c[i] = __float_as_uint(up);
      if (Mode != RowNorm) off = fmaxf(off, fmaf(fabsf(q), Mode == RowGated ? GatedError : PlainError, fabsf(q - (up - Round))));
    }
    if (Mode != RowNorm && off >= 0.5f && r.live && v < vectors) {
      for (int i = 0; i < N; ++i) {
        const float exact = Mode == RowGated ? gated_exact(a, b, v * N + i) : row_to_float(a[v * N + i]);
        const uint32_t code = (uint32_t)__float2int_rn(exact / r.scale);
#pragma unroll
        for (int k = 0; k < N; ++k) if (k == i) c[k] = code;
      }
    }
    if (v < vectors) {
      uint32_t w[N / 4];
#pragma unroll
      for (int k = 0; k < N / 4; ++k)
        w[k] = r.live ? __byte_perm(__byte_perm(c[4 * k], c[4 * k + 1], 0x0040), __byte_perm(c[4 * k + 2], c[4 * k + 3], 0x0040), 0x5410) : 0u;
      if constexpr (N == 8) reinterpret_cast<uint2*>(codes)[v] = make_uint2(w[0], w[1]);
      else reinterpret_cast<uint32_t*>(codes)[v] = w[0];
    }
  }
}

// out = scale * code.  One thread per 8 codes where the output rows allow 16-byte stores, else per element.
template <typename T, bool Vector> __global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* codes, int64_t codes_stride,
    const float* scales, T* out, int64_t out_stride, int64_t rows, int width) {
  constexpr int N = Vector ? 8 : 1;
  const int per_row = width / N;
  const int64_t total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = total <= 0x7fffffff ? (uint32_t)i / (uint32_t)per_row : i / per_row;
    const int e = (int)(i - row * per_row) * N;
    const float scale = scales[row];
    if constexpr (!Vector) {
      out[row * out_stride + e] = row_from_float<T>((float)codes[row * codes_stride + e] * scale);
    } else {
      const uint2 c = *reinterpret_cast<const uint2*>(codes + row * codes_stride + e);
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = (float)(int8_t)((k < 4 ? c.x : c.y) >> (8 * (k & 3))) * scale;
      uint4* to = reinterpret_cast<uint4*>(out + row * out_stride + e);
      if constexpr (sizeof(T) == 4) {
        to[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        to[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
      } else {
        RowVector<T> v;
        v.pack(x);
        to[0] = v.raw;
      }
    }
  }
}

template <typename T, int Mode> static void launch_rows_type(int64_t rows, const RowArgs& p, cudaStream_t s) {
  constexpr int N = RowVector<T>::N;
  const auto vector_rows = [](const void* base, int64_t stride) { return aligned16(base) && stride % N == 0; };
  const int vectors = p.width / N;
  const bool fast = p.width % N == 0 && vectors <= 4096 && vector_rows(p.a, p.a_stride) && vector_rows(p.b, p.b_stride) &&
                    vector_rows(p.weight, 0) && vector_rows(p.sum, p.sum_stride);
  if (!fast) {
    const int threads = p.width <= 256 ? 128 : p.width <= 2048 ? 256 : 512;
    rows_general_kernel<T, Mode><<<(unsigned)rows, threads, 0, s>>>(p);
    return;
  }
  if constexpr (Mode != RowNorm) {
    if (vectors <= 64) {
      const unsigned grid = (unsigned)((rows + 3) / 4);
      if (vectors <= 32) rows_kernel<T, Mode, 1, true><<<grid, 128, 0, s>>>(p);
      else rows_kernel<T, Mode, 2, true><<<grid, 128, 0, s>>>(p);
      return;
    }
  }
  // one vector per thread while that gives every SM little to do (one round trip bounds the call), four otherwise
  const int want = rows <= 592 ? 1 : 4, least = (vectors + 1023) / 1024;
  const int v = want < least ? (least <= 2 ? 2 : 4) : want;
  int threads = ((vectors + v - 1) / v + 31) / 32 * 32;
  if (v == 1) rows_kernel<T, Mode, 1, false><<<(unsigned)rows, threads, 0, s>>>(p);
  else if (v == 2) rows_kernel<T, Mode, 2, false><<<(unsigned)rows, threads, 0, s>>>(p);
  else rows_kernel<T, Mode, 4, false><<<(unsigned)rows, threads, 0, s>>>(p);
}

template <int Mode> static int launch_rows(int type, int64_t rows, const RowArgs& p, cudaStream_t s) {
  if (type == TRI_BF16) launch_rows_type<__nv_bfloat16, Mode>(rows, p, s);
  else if (type == TRI_FP16) launch_rows_type<__half, Mode>(rows, p, s);
  else launch_rows_type<float, Mode>(rows, p, s);
  return tri_launch_status("rows");
}

template <typename T> static void launch_values(const void* codes, int64_t codes_stride, const float* scales, int64_t rows, int width,
                                                void* out, int64_t out_stride, cudaStream_t s) {
  const bool vector = width % 8 == 0 && aligned16(out) && out_stride * sizeof(T) % 16 == 0;
  const int64_t blocks = (rows * (vector ? width / 8 : width) + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 148 * 64 ? blocks : 148 * 64);
  if (vector) dequantize_rows_kernel<T, true><<<grid, 256, 0, s>>>(static_cast<const int8_t*>(codes), codes_stride, scales, static_cast<T*>(out), out_stride, rows, width);
  else dequantize_rows_kernel<T, false><<<grid, 256, 0, s>>>(static_cast<const int8_t*>(codes), codes_stride, scales, static_cast<T*>(out), out_stride, rows, width);
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
  p.rows = rows;
  p.a = x; p.a_stride = x_stride; p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width;
  return launch_rows<RowPlain>(type, rows, p, static_cast<cudaStream_t>(stream));
}

extern "C" int tri_silu_mul_rows(const void* gate, const void* up, int type, int64_t rows, int width, int64_t gate_stride,
    int64_t up_stride, void* codes, int64_t codes_stride, float* scales, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "silu_mul_rows: rows, width 1..131071, type");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(gate && up && codes && scales, "silu_mul_rows: null buffers");
  TRI_CHECK(row_pointer(gate, type) && row_pointer(up, type) && gate_stride >= 0 && up_stride >= 0, "silu_mul_rows: input rows");
  TRI_CHECK(code_rows(codes, codes_stride, width), "silu_mul_rows: code rows start on 16-byte boundaries");
  RowArgs p{};
  p.rows = rows;
  p.a = gate; p.b = up; p.a_stride = gate_stride; p.b_stride = up_stride;
  p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width;
  return launch_rows<RowGated>(type, rows, p, static_cast<cudaStream_t>(stream));
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
  p.rows = rows;
  p.a = x; p.b = residual; p.weight = weight; p.a_stride = x_stride; p.b_stride = residual_stride;
  p.sum = residual_out; p.sum_stride = residual_out_stride;
  p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width; p.eps = (float)eps;
  return launch_rows<RowNorm>(type, rows, p, static_cast<cudaStream_t>(stream));
}

extern "C" int tri_dequantize_rows(const void* codes, int64_t codes_stride, const float* scales, int type, int64_t rows, int width,
    void* out, int64_t out_stride, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "dequantize_rows: rows, width 1..131071, type");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(codes && scales && out, "dequantize_rows: null buffers");
  TRI_CHECK(code_rows(codes, codes_stride, width), "dequantize_rows: code rows start on 16-byte boundaries");
  TRI_CHECK(row_pointer(out, type) && out_stride >= width, "dequantize_rows: output rows");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == TRI_BF16) launch_values<__nv_bfloat16>(codes, codes_stride, scales, rows, width, out, out_stride, s);
  else if (type == TRI_FP16) launch_values<__half>(codes, codes_stride, scales, rows, width, out, out_stride, s);
  else launch_values<float>(codes, codes_stride, scales, rows, width, out, out_stride, s);
  return tri_launch_status("dequantize_rows");
}
