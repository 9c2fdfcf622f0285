// Rows as INT8 codes: the operands of tri_int8_linear, made from activations (or weights).
//
//   rows    y = x
//   gated   y = g / (1 + e^-g) * u
//   norm    h = round(x + r),  y = h * rsqrt(mean h^2 + eps) * w
//   codes   s = max|y| / 127,  c = rint(y / s)      symmetric, one scale per row
//
// A row of zeros has scale 0 and codes 0; so has one whose largest magnitude is below 2^-119, where max/127 would leave the
// range of normal floats.  A row that holds a NaN or an infinity, or whose y overflows, has scale NaN and codes 0: every product
// that reads it is NaN, and no other row is touched by it.  (Of a norm, |y| here is |h * w|, before the root divides it.)
// Plain and gated rows: codes and scales are, bit for bit, rint(y / s) and s = max|y| * fl(1/127) of the formulas above in IEEE fp32
// with CUDA's expf (the file is compiled without --use_fast_math).  Approximate instructions are used on the way, but every
// element whose code they might change is worked out again.  A row's largest element can be eighty times its root mean square, so a
// code that is off by one step where y / s is next to a tie would be off by more than half of that.
// Normed rows: the code is rint(127 y / max|y|) of y = h * w in fp32 (exact for 16-bit types), the quotient rounded to fp32 once: on
// a tie, which products of 16-bit numbers do meet, the even code as exact arithmetic has it.  (The quotient comes from the reciprocal
// in two terms.  With one, 1273 of 58.7 million codes of 16384 x 3584 in bf16 fell on a tie's other side.  Times of that size: 54 us
// without a residual, 57 like this; with one 73 and 68 in a replayed graph, 71 and 73 called one by one; deciding near ties by a
// branch took 71 and 80.)  The scale's root is approximate (2^-22.9).  h is rounded to the stream's type before it is normed,
// because that is what later layers read.
#include "common.cuh"
#include "abi_internal.h"
#include <type_traits>

namespace tri {

enum RowMode : int { RowPlain = 0, RowGated = 1, RowNorm = 2 };
constexpr int RowShared = 200 * 1024;                // per SM, for the rows ahead
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
  float eps, inverse_width;
};

// Largest magnitude as the bits of |y|: an integer maximum, so that a NaN (whose bits lie above every number's) survives.
__device__ __forceinline__ uint32_t magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// Maximum (and, for the norm, sum) over the CTA; every thread gets both.  One barrier: consecutive calls use the two halves of the
// arrays in turn, and a warp that writes a half again has passed the barrier of the call between.
struct RowShare {
  float sums[2][32];
  uint32_t peaks[2][32];
};
template <bool Sum> __device__ __forceinline__ void row_reduce(float& sum, uint32_t& peak, RowShare& share, uint32_t turn) {
  peak = __reduce_max_sync(0xffffffffu, peak);
  if (Sum)
#pragma unroll
    for (int bit = 16; bit > 0; bit >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, bit);
  const int warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (warps == 1) return;
  if (lane == 0) { if (Sum) share.sums[turn][warp] = sum; share.peaks[turn][warp] = peak; }
  __syncthreads();
  peak = __reduce_max_sync(0xffffffffu, lane < warps ? share.peaks[turn][lane] : 0u);
  if (Sum) {
    sum = lane < warps ? share.sums[turn][lane] : 0.f;
#pragma unroll
    for (int bit = 16; bit > 0; bit >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, bit);
  }
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
  float scale, inverse;                 // inverse: of max|y| / 127, before the norm's common factor
  float rest;                           // norm: what `inverse` lacks of 127 / max|y| (inverse + rest: to 2^-45)
  bool live;                            // codes are not all zero
};
// (Every thread of a row works this out, and it weighs as much as eight elements: approximate reciprocal and root, 2^-22.9.)
template <int Mode> __device__ __forceinline__ RowScale row_scale(uint32_t peak, float squares, float eps, float inverse_width, float shift) {
  const float step = __uint_as_float(peak) * (1.f / 127.f);
  bool finite = peak < 0x7f800000u, zero = __uint_as_float(peak) < RowTiny;
  RowScale r;
  r.scale = step;
  if (Mode == RowNorm) {
    const float power = fmaf(squares, inverse_width, eps * shift * shift);
    finite = finite && squares < 3e38f;
    zero = zero || power == 0.f;
    float factor;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(factor) : "f"(power));
    r.scale *= factor;
  }
  r.live = finite && !zero;
  r.scale = !finite ? CUDART_NAN_F : zero ? 0.f : fminf(r.scale, RowLargestScale);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.inverse) : "f"(r.live ? step : 1.f));
  if (Mode == RowNorm) r.rest = fmaf(-r.inverse, __uint_as_float(peak), 127.f) * (r.inverse * (1.f / 127.f));
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
template <typename T, int Mode> __device__ __noinline__ void row_general(const RowArgs& p, int64_t row, bool summed, RowShare& share) {
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
    __syncthreads();                  // (a call before this one may have used the same half)
    row_reduce<Mode == RowNorm>(squares, peak, share, attempt);
    if (Mode == RowNorm && sum != nullptr) { a = sum; b = nullptr; sum = nullptr; }   // from here on h is read (a thread reads
                                                                                      // what it wrote; residual may be gone)
    if (Mode != RowNorm || squares_fit(squares) || (squares == 0.f && peak == 0)) break;
    shift = squares > 1.f || squares != squares ? 8.271806125530277e-25f : 1.152921504606847e18f;   // 2^-80, 2^60
  }
  const RowScale r = row_scale<Mode>(peak, squares, p.eps, p.inverse_width, shift);
  if (threadIdx.x == 0) p.scales[row] = r.scale;
  int8_t* codes = p.codes + row * p.codes_stride;
  for (int e = threadIdx.x; e < p.width; e += threads) {
    const float y = row_element<T, Mode>(p, a, b, sum, e, shift, squares);
    codes[e] = !r.live ? (int8_t)0 : (int8_t)__float2int_rn(Mode == RowNorm ? fmaf(y, r.inverse, y * r.rest) : y / r.scale);
  }
}

template <typename T, int Mode> __global__ void __launch_bounds__(1024) rows_general_kernel(const RowArgs p) {
  __shared__ RowShare share;
  grid_launch_dependents();
  grid_dependency_wait();
  row_general<T, Mode>(p, blockIdx.x, false, share);
}

// ---- rows held in registers ---------------------------------------------------------------------------------------------
// A thread holds V vectors of 16 bytes (or V * N single elements) of a row, so the row is read from memory once whatever the
// mode.  Long batches are bound by HBM: a CTA takes rows in turn and copies the rows after the current one into shared memory
// meanwhile (cp.async, every thread its own vectors, so no barrier is involved): without that the loads of a row wait for the
// reduction of the row before.  Short batches are bound by one trip to memory and one reduction.
// Gated: the y that a thread keeps are computed with the fast exponential and reciprocal (8 instead of 30 instructions per
// element, which would bound the kernel).  Where that could show, at elements
// that may be the row's largest and at quotients next to a tie, the element is computed again in IEEE arithmetic.
// Relative error of the fast y and of y / s worked out from it, in steps of 2^-24: 1.5 |g| for the exponent's argument, 4 for the
// exponential, 5 for sum, reciprocal and products, 5 for the IEEE evaluation itself, 4 for the quotient: 42 for |g| <= 16 (which
// gates hardly ever leave), 150 for the |g| < 88 that give a y at all.
constexpr float GatedNear = 3e-6f, GatedFar = 1.2e-5f, GateNear = -16.f;
constexpr float PlainError = 5e-7f;     // y * (1/s) against y / s: 2^-23 for the reciprocal, 2^-24 for product and quotient each, 2^-22
constexpr float Round = 12582912.f;     // 1.5 * 2^23: x + Round has rint(x) in its low bits

enum RowLayout : int { RowCta = 0, RowFull = 1, RowWarp = 2, RowAnywhere = 3 };

// max(|a|, |b|, |c|); NaN where any is.
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 operations in one instruction; the kernels are bound by the instructions they issue as much as by HBM.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 gated_fast2(float2 g, float2 u) {
  const float2 x = mul2(g, both(-1.4426950408889634f));
  float2 e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
  e = add2(e, both(1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
  return mul2(mul2(g, r), u);
}
__device__ __forceinline__ void copy_async(uint32_t to, const char* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return v;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait(int pending) {      // until at most `pending` of this thread's groups are under way
  if (pending >= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (pending == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

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

// ---- rows that start anywhere ---------------------------------------------------------------------------------------------
// Memory is read and written in aligned blocks of 16 bytes, and vectors are shifted out of two neighbouring ones.  Blocks that reach
// over an end of the tensor (of the row, where something is written) are taken element by element.  8192 x 4095 in single
// elements, 2 bytes an access, and like this: plain 62 and 35 us, gated 91 and 59, norm with residual 140 and 85, values 65 and 30.
// 16 bytes from byte `shift` (0..15) on of lo, hi.  (Four branches, one of which a whole row takes: 59 us for the gated rows above,
// 65 with selects.)
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, uint32_t shift) {
  const uint32_t bits = 8 * (shift & 3);
  const auto join = [bits](uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e) {
    return make_uint4(__funnelshift_r(a, b, bits), __funnelshift_r(b, c, bits), __funnelshift_r(c, d, bits), __funnelshift_r(d, e, bits));
  };
  switch (shift >> 2) {
    case 0: return join(lo.x, lo.y, lo.z, lo.w, hi.x);
    case 1: return join(lo.y, lo.z, lo.w, hi.x, hi.y);
    case 2: return join(lo.z, lo.w, hi.x, hi.y, hi.z);
    default: return join(lo.w, hi.x, hi.y, hi.z, hi.w);
  }
}
template <typename T> __device__ __forceinline__ uint32_t element_bits(const T* from) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t*>(from);
  else return *reinterpret_cast<const unsigned short*>(from);
}
// The vector-th vector of a row of `width` elements; zero past its end.
template <typename T> __device__ __forceinline__ uint4 load_anywhere(const T* row, int vector, int width) {
  constexpr int N = 16 / sizeof(T), S = sizeof(T);
  const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
  const int before = shift / S, e = vector * N;             // elements of the block in front of the vector's first
  const uint4* block = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row) + (int64_t)vector * 16 - shift);
  if (shift == 0 ? e + N <= width : e >= before && e - before + 2 * N <= width) {
    const uint4 lo = block[0];
    return shift == 0 ? lo : shifted(lo, block[1], shift);
  }
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (e + i < width) w[i * S / 4] |= element_bits(row + e + i) << (8 * (i * S % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The vector that begins `shift` bytes into the block at `from`, in shared memory; zero from its live-th element on.
template <typename T> __device__ __forceinline__ uint4 shared_vector(uint32_t from, uint32_t shift, int live) {
  constexpr int N = 16 / sizeof(T), S = sizeof(T);
  if (live <= 0) return make_uint4(0, 0, 0, 0);
  uint4 v = load_shared(from);
  if (shift != 0) v = shifted(v, load_shared(from + 16), shift);
  if (live < N) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i >= live) w[i * S / 4] &= S == 4 ? 0u : i % 2 ? 0x0000ffffu : 0xffff0000u;
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
// A block's elements that lie in [low, high).
template <typename T> __device__ __noinline__ void copy_elements(uint32_t to, const char* block, const char* low, const char* high) {
  if (block >= low && block + 16 <= high) { copy_async(to, block); return; }
#pragma unroll 1
  for (int i = 0; i < 16; i += sizeof(T))
    if (block + i >= low && block + i < high) {
      if constexpr (sizeof(T) == 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + i), "r"(element_bits(reinterpret_cast<const T*>(block + i))) : "memory");
      else asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + i), "h"((unsigned short)element_bits(reinterpret_cast<const T*>(block + i))) : "memory");
    }
}
// Stores the vectors that a whole warp holds, lane l the one after lane l - 1's.  A lane writes the block that its vector begins in.
template <typename T> __device__ __forceinline__ void store_anywhere(T* row, int vector, int width, const uint4& v) {
  constexpr int N = 16 / sizeof(T), S = sizeof(T);
  const uint32_t shift = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
  const int lane = threadIdx.x % 32, before = shift / S, e = vector * N;
  const uint4 last = make_uint4(__shfl_up_sync(0xffffffffu, v.x, 1), __shfl_up_sync(0xffffffffu, v.y, 1),
                                __shfl_up_sync(0xffffffffu, v.z, 1), __shfl_up_sync(0xffffffffu, v.w, 1));
  const uint4 block = shift == 0 ? v : shifted(last, v, 16 - shift);
  const auto put = [&](const uint4& from, int i, int at) {   // element i of a block
    const uint32_t w[4] = {from.x, from.y, from.z, from.w}, bits = w[i * S / 4] >> (8 * (i * S % 4));
    if constexpr (S == 4) reinterpret_cast<uint32_t*>(row)[at] = bits;
    else reinterpret_cast<unsigned short*>(row)[at] = (unsigned short)bits;
  };
  if ((before == 0 || lane > 0) && e - before + N <= width) {
    *reinterpret_cast<uint4*>(reinterpret_cast<char*>(row) + (int64_t)vector * 16 - shift) = block;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i >= before || lane > 0) && e - before + i < width) put(block, i, e - before + i);
  }
  if (lane == 31) {                                          // the next lane is another warp's
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i >= N - before && e + i < width) put(v, i, e + i);
  }
}

// gated() out of line, for the few elements that need it.
__device__ __noinline__ float gated_exact(float gate, float up) { return gated(gate, up); }
template <typename T> __device__ __forceinline__ float load_shared_element(uint32_t from) {
  if constexpr (sizeof(T) == 4) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
    return v;
  } else {
    unsigned short v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
    return row_to_float(*reinterpret_cast<const T*>(&v));
  }
}

// RowCta: inputs start on 16-byte boundaries and hold whole vectors; a CTA per row, gridDim.x rows at a time, `depth` rows in
// shared memory.  RowFull: the same where every thread has all of its vectors.  RowWarp: for short rows, a warp per row, four
// per CTA.  RowAnywhere: any alignment and width, a CTA per row.
template <typename T, int Mode, int V, int Layout> __global__ void __launch_bounds__(Layout == RowWarp ? 128 : 1024)
    rows_kernel(const RowArgs p, int depth) {
  constexpr int N = RowVector<T>::N;
  constexpr bool Ring = Layout != RowWarp, Full = Layout == RowFull, Anywhere = Layout == RowAnywhere;
  extern __shared__ uint4 ring[];       // [depth][a, b][V][thread]; RowAnywhere: [depth][a, b][V][warp][33 blocks]
  __shared__ RowShare share;
  grid_launch_dependents();
  grid_dependency_wait();
  const int threads = Layout == RowWarp ? 32 : blockDim.x, me = Layout == RowWarp ? threadIdx.x % 32 : threadIdx.x;
  const int64_t first = Layout == RowWarp ? (int64_t)blockIdx.x * 4 + threadIdx.x / 32 : blockIdx.x;
  const int64_t stride = Layout == RowWarp ? (int64_t)gridDim.x * 4 : gridDim.x;
  const int vectors = (p.width + N - 1) / N;
  const bool two = Mode == RowGated || (Mode == RowNorm && p.b != nullptr);
  const auto element = [&](int j, int i) { return (j * threads + me) * N + i; };
  const auto mine = [&](int j) { return Full || j * threads + me < vectors; };     // whether this thread has a j-th vector
  const auto row_a = [&](int64_t row) { return static_cast<const T*>(p.a) + row * p.a_stride; };
  const auto row_b = [&](int64_t row) { return static_cast<const T*>(p.b) + row * p.b_stride; };

  // Every address below is a start that advances by row plus j * `step` bytes, on both sides of the copies: with products worked
  // out per vector the address arithmetic was a third of all instructions.
  const int step = threads * 16, ring_step = Anywhere ? threads / 32 * 33 * 16 : step, slot_bytes = (two ? 2 : 1) * V * ring_step;
  const uint32_t ring_start = smem_u32(ring) + (me + (Anywhere ? me / 32 : 0)) * 16, ring_end = ring_start + depth * slot_bytes;
  const char *next_a = reinterpret_cast<const char*>(row_a(first)) + me * 16, *next_b = two ? reinterpret_cast<const char*>(row_b(first)) + me * 16 : nullptr;
  const int64_t advance_a = stride * p.a_stride * (int64_t)sizeof(T), advance_b = stride * p.b_stride * (int64_t)sizeof(T);
  int64_t next_row = first;
  // RowAnywhere: the blocks that a warp's 32 vectors begin in, and the one after them (lane 31's).  A block may reach over the
  // row's ends into the rows beside it, but not out of the tensor: the first and the last row are copied with care.
  const auto copy_anywhere = [&](uint32_t to, const char* from, int vector, const void* base, int64_t row_stride) {
    const int shift = (int)reinterpret_cast<uintptr_t>(from) & 15, past = vector * 16 - p.width * (int)sizeof(T);    // (of the row's end)
    const char* block = from - shift;
    const bool first_block = past < shift, extra_block = me % 32 == 31 && past + 16 < shift;
    // Between two other rows neither block leaves the tensor.
    if (next_row > 0 && next_row + 1 < p.rows && row_stride >= N) {
      if (first_block) copy_async(to, block);
      if (extra_block) copy_async(to + 16, block + 16);
    } else {
      const char *low = static_cast<const char*>(base), *high = low + ((p.rows - 1) * row_stride + p.width) * (int64_t)sizeof(T);
      if (first_block) copy_elements<T>(to, block, low, high);
      if (extra_block) copy_elements<T>(to + 16, block + 16, low, high);
    }
  };
  const auto prefetch = [&](uint32_t slot) {     // the next row that has not been asked for
    if (next_row < p.rows) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if constexpr (Anywhere) {
          copy_anywhere(slot + j * ring_step, next_a + j * step, j * threads + me, p.a, p.a_stride);
          if (two) copy_anywhere(slot + (V + j) * ring_step, next_b + j * step, j * threads + me, p.b, p.b_stride);
        } else if (mine(j)) {
          copy_async(slot + j * step, next_a + j * step);
          if (two) copy_async(slot + (V + j) * step, next_b + j * step);
        }
    }
    copy_commit();
    next_row += stride; next_a += advance_a; next_b += advance_b;
  };
  if constexpr (Ring)
    for (uint32_t slot = ring_start; slot < ring_end; slot += slot_bytes) prefetch(slot);
  RowVector<T> vw[V];                   // norm: this thread's part of the weight, which every row needs
  if constexpr (Mode == RowNorm && Ring && V <= 2) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (Anywhere) vw[j].raw = load_anywhere(static_cast<const T*>(p.weight), j * threads + me, p.width);
      else vw[j].raw = mine(j) ? __ldg(reinterpret_cast<const uint4*>(p.weight) + j * threads + me) : make_uint4(0, 0, 0, 0);
    }
  }

  uint32_t slot = ring_start, parity = 0;
  int8_t* codes = p.codes + first * p.codes_stride + me * N;
  char* sum = Mode == RowNorm && two ? reinterpret_cast<char*>(static_cast<T*>(p.sum) + first * p.sum_stride) + (Layout == RowAnywhere ? 0 : me * 16) : nullptr;
  const int64_t advance_codes = stride * p.codes_stride, advance_sum = stride * p.sum_stride * (int64_t)sizeof(T);
  for (int64_t row = first; row < p.rows; row += stride, codes += advance_codes, sum += advance_sum, parity ^= 1) {
    float y[V][N], squares = 0.f, largest = 0.f, lowest = 0.f;   // lowest: of the gates
    if constexpr (Ring) copy_wait(depth - 1);
    uint32_t shift_a = 0, shift_b = 0;  // RowAnywhere: from a block's start to the vector's
    if constexpr (Anywhere) {
      __syncwarp();                     // a vector reaches into the next lane's block
      shift_a = (uint32_t)reinterpret_cast<uintptr_t>(row_a(row)) & 15u;
      if (two) shift_b = (uint32_t)reinterpret_cast<uintptr_t>(row_b(row)) & 15u;
    }
    RowVector<T> held[Layout == RowAnywhere && Mode == RowNorm ? V : 1];      // h, until the whole row has been read (h may replace it)
    {
      RowVector<T> va[V], vb[V];
      float2 squares2 = both(0.f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (Anywhere) {
          va[j].raw = shared_vector<T>(slot + j * ring_step, shift_a, p.width - element(j, 0));
          if (two) vb[j].raw = shared_vector<T>(slot + (V + j) * ring_step, shift_b, p.width - element(j, 0));
        } else if constexpr (Ring) {
          va[j].raw = mine(j) ? load_shared(slot + j * step) : make_uint4(0, 0, 0, 0);
          if (two) vb[j].raw = mine(j) ? load_shared(slot + (V + j) * step) : make_uint4(0, 0, 0, 0);
        } else {
          va[j].raw = mine(j) ? __ldcs(reinterpret_cast<const uint4*>(row_a(row)) + j * threads + me) : make_uint4(0, 0, 0, 0);
          if (two) vb[j].raw = mine(j) ? __ldcs(reinterpret_cast<const uint4*>(row_b(row)) + j * threads + me) : make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        va[j].unpack(y[j]);
        if (two) {
          float r[N];
          vb[j].unpack(r);
          if constexpr (Mode == RowGated) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
              lowest = fminf(lowest, fminf(y[j][i], y[j][i + 1]));
              const float2 t = gated_fast2(make_float2(y[j][i], y[j][i + 1]), make_float2(r[i], r[i + 1]));
              y[j][i] = t.x; y[j][i + 1] = t.y;
            }
          } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
              const float2 t = add2(make_float2(y[j][i], y[j][i + 1]), make_float2(r[i], r[i + 1]));
              y[j][i] = t.x; y[j][i + 1] = t.y;
            }
            RowVector<T> h;
            h.pack(y[j]);
            h.unpack(y[j]);
            if constexpr (Layout == RowAnywhere) held[j] = h;
            else if (mine(j)) *reinterpret_cast<uint4*>(sum + j * step) = h.raw;
          }
        }
        if constexpr (Mode == RowNorm) {
          if constexpr (Anywhere && V > 2) vw[j].raw = load_anywhere(static_cast<const T*>(p.weight), j * threads + me, p.width);
          else if constexpr (!Ring || V > 2) vw[j].raw = mine(j) ? __ldg(reinterpret_cast<const uint4*>(p.weight) + j * threads + me) : make_uint4(0, 0, 0, 0);
          float w[N];
          vw[j].unpack(w);
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            const float2 h = make_float2(y[j][i], y[j][i + 1]), t = mul2(h, make_float2(w[i], w[i + 1]));
            squares2 = fma2(h, h, squares2);
            y[j][i] = t.x; y[j][i + 1] = t.y;
          }
        }
      }
      squares = squares2.x + squares2.y;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < N; i += 2) largest = max_magnitude(largest, y[j][i], y[j][i + 1]);
    const float error = Mode == RowPlain ? PlainError : lowest < GateNear ? GatedFar : GatedNear;
    uint32_t peak = __float_as_uint(largest);
    if constexpr (Mode == RowGated) {
      // This warp's largest y in IEEE arithmetic: of the few elements (one, nearly always) that may be it.
      const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, peak)), bar = top * (1.f - 2.f * GatedFar);
      if (top > 0.f && top < CUDART_INF_F) {
        uint32_t exact = 0;
        if (largest >= bar) {
#pragma unroll
          for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i)
              if (fabsf(y[j][i]) >= bar) {
                float g, u;
                if constexpr (Ring) {
                  g = load_shared_element<T>(slot + j * ring_step + shift_a + i * (int)sizeof(T));
                  u = load_shared_element<T>(slot + (V + j) * ring_step + shift_b + i * (int)sizeof(T));
                } else {
                  g = row_to_float(row_a(row)[element(j, i)]);
                  u = row_to_float(row_b(row)[element(j, i)]);
                }
                exact = max(exact, magnitude(gated_exact(g, u)));
              }
        }
        peak = exact;
      }
    }
    if constexpr (Anywhere) __syncwarp();
    if constexpr (Ring) {               // the row's inputs are in registers: its slot takes the row `depth` turns ahead
      prefetch(slot);
      slot += slot_bytes;
      if (slot == ring_end) slot = ring_start;
    }
    if constexpr (Layout == RowWarp) peak = __reduce_max_sync(0xffffffffu, peak);
    else row_reduce<Mode == RowNorm>(squares, peak, share, parity);
    if constexpr (Layout == RowAnywhere && Mode == RowNorm) {
      if (two)
#pragma unroll
        for (int j = 0; j < V; ++j) store_anywhere(reinterpret_cast<T*>(sum), j * threads + me, p.width, held[j].raw);
    }
    if constexpr (Mode == RowNorm) {
      if (!squares_fit(squares) && !(squares == 0.f && peak == 0)) {      // (the same for the whole CTA)
        __syncthreads();                // other threads' h has just been written; the reduction's own barrier comes before it
                                        // (RowAnywhere) or is left out (a row of one warp: shuffles order no memory)
        row_general<T, Mode>(p, row, two, share);
        __syncthreads();                // (it leaves either half in use)
        continue;
      }
    }
    const RowScale r = row_scale<Mode>(peak, squares, p.eps, p.inverse_width, 1.f);
    if (me == 0) p.scales[row] = r.scale;
    const float inverse = r.inverse;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      uint32_t c[N];
      float off = 0.f, size = 0.f;      // largest distance from the next code, largest quotient
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 two_y = make_float2(y[j][i], y[j][i + 1]);
        const float2 q = Mode == RowNorm ? fma2(two_y, both(inverse), mul2(two_y, both(r.rest))) : mul2(two_y, both(inverse)), up = add2(q, both(Round));
        c[i] = __float_as_uint(up.x); c[i + 1] = __float_as_uint(up.y);
        if (Mode != RowNorm) {
          const float2 back = add2(up, both(-Round)), from = fma2(back, both(-1.f), q);
          off = max_magnitude(off, from.x, from.y);
          size = max_magnitude(size, q.x, q.y);
        }
      }
      if (Mode != RowNorm && fmaf(size, error, off) >= 0.5f && r.live) {
        // some quotient of these may lie on the other side of a tie
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float q = y[j][i] * inverse, from = fabsf(q - (q + Round - Round));
          if (fmaf(fabsf(q), error, from) >= 0.5f) {
            const float exact = Mode == RowGated ? gated_exact(row_to_float(row_a(row)[element(j, i)]), row_to_float(row_b(row)[element(j, i)])) : y[j][i];
            c[i] = (uint32_t)__float2int_rn(exact / r.scale);
          }
        }
      }
      if (Layout == RowAnywhere && element(j, N) > p.width) {
#pragma unroll
        for (int i = 0; i < N; ++i) if (element(j, i) < p.width) codes[j * threads * N + i] = r.live ? (int8_t)c[i] : (int8_t)0;
      } else if (mine(j)) {
        uint32_t w[N / 4];
#pragma unroll
        for (int k = 0; k < N / 4; ++k)
          w[k] = r.live ? __byte_perm(__byte_perm(c[4 * k], c[4 * k + 1], 0x0040), __byte_perm(c[4 * k + 2], c[4 * k + 3], 0x0040), 0x5410) : 0u;
        if constexpr (N == 8) *reinterpret_cast<uint2*>(codes + j * threads * N) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(codes + j * threads * N) = w[0];
      }
    }
  }
}

// out = scale * code.  blockDim.x threads per row, blockDim.y rows per CTA at a time; a thread takes the codes of 16 bytes of
// output (neighbouring threads then write neighbouring 16 bytes; 32 bytes a thread were 7 % slower), shifted into place where the
// output rows start anywhere.  Bound by HBM (the writes): no index is divided, a row's scale is read once.
template <typename T, bool Vector> __global__ void __launch_bounds__(256) dequantize_rows_kernel(const int8_t* codes, int64_t codes_stride,
    const float* scales, T* out, int64_t out_stride, int64_t rows, int width) {
  grid_launch_dependents();
  grid_dependency_wait();
  for (int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; row < rows; row += (int64_t)gridDim.x * blockDim.y) {
    const float scale = scales[row];
    const int8_t* from = codes + row * codes_stride;
    T* to = out + row * out_stride;
    constexpr int N = RowVector<T>::N;
    if constexpr (!Vector) {
      for (int base = threadIdx.x & ~31; N * base < width; base += blockDim.x) {      // (the same turns for a whole warp)
        const int vector = base + threadIdx.x % 32, e = N * vector;
        float x[N];
        if (e + N <= width) {
          uint32_t w[N / 4];
          if constexpr (N == 8) {
            const uint2 c = __ldcs(reinterpret_cast<const uint2*>(from + e));
            w[0] = c.x; w[1] = c.y;
          } else {
            w[0] = __ldcs(reinterpret_cast<const uint32_t*>(from + e));
          }
#pragma unroll
          for (int i = 0; i < N; ++i) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) x[i] = e + i < width ? (float)from[e + i] * scale : 0.f;
        }
        RowVector<T> v;
        v.pack(x);
        store_anywhere(to, vector, width, v.raw);
      }
    } else {
#pragma unroll 4
      for (int e = N * threadIdx.x; e < width; e += N * blockDim.x) {
        uint32_t w[N / 4];
        if constexpr (N == 8) {
          const uint2 c = __ldcs(reinterpret_cast<const uint2*>(from + e));
          w[0] = c.x; w[1] = c.y;
        } else {
          w[0] = __ldcs(reinterpret_cast<const uint32_t*>(from + e));
        }
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
        RowVector<T> v;
        v.pack(x);
        *reinterpret_cast<uint4*>(to + e) = v.raw;
      }
    }
  }
}

// One call of rows_kernel with as many CTAs as are resident at once (RowCta, RowFull) or as the rows need.
template <typename T, int Mode, int V, int Layout> static int launch_rows_kernel(const RowArgs& p, int sms, cudaStream_t s) {
  constexpr int N = RowVector<T>::N;
  const auto kernel = rows_kernel<T, Mode, V, Layout>;
  if (Layout == RowWarp) {
    TRI_CUDA(launch_chained(kernel, dim3((unsigned)((p.rows + 3) / 4)), dim3(128), 0, s, p, 1), "rows");
    return tri_launch_status("rows");
  }
  const int vectors = (p.width + N - 1) / N, threads = ((vectors + V - 1) / V + 31) / 32 * 32;
  static TriPerDevice configured;
  static std::atomic<int> registers{0};
  const int device = configured.pending();
  TRI_CHECK(device != -2, "rows: no current CUDA device");
  if (device >= 0) {
    cudaFuncAttributes attributes;
    TRI_CUDA(cudaFuncGetAttributes(&attributes, kernel), "rows");
    TRI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RowShared), "rows");
    registers.store(attributes.numRegs, std::memory_order_relaxed);
    configured.mark(device);
  }
  // resident CTAs per SM by threads, registers and shared memory, then the depth that the rest of the shared memory gives
  const int row_bytes = (Mode != RowPlain && p.b != nullptr ? 2 : 1) * V * (Layout == RowAnywhere ? threads / 32 * 33 : threads) * 16;
  int resident = 2048 / threads < 32 ? 2048 / threads : 32;
  const int by_registers = 65536 / ((registers.load(std::memory_order_relaxed) + 7) / 8 * 8 * threads);
  if (by_registers < resident) resident = by_registers;
  if (RowShared / row_bytes < resident) resident = RowShared / row_bytes;
  if (resident < 1) resident = 1;
  int depth = RowShared / (resident * row_bytes);
  if (depth > 4) depth = 4;
  if (p.rows <= (int64_t)resident * sms) depth = 1;
  const int64_t slots = (int64_t)resident * sms, grid = p.rows < slots ? p.rows : slots;
  TRI_CUDA(launch_chained(kernel, dim3((unsigned)grid), dim3(threads), (size_t)depth * row_bytes, s, p, depth), "rows");
  return tri_launch_status("rows");
}

template <typename T, int Mode, int V> static int launch_rows_ring(const RowArgs& p, int sms, cudaStream_t s) {
  if (p.width / RowVector<T>::N % (32 * V) == 0) return launch_rows_kernel<T, Mode, V, RowFull>(p, sms, s);
  return launch_rows_kernel<T, Mode, V, RowCta>(p, sms, s);
}

template <typename T, int Mode> static int launch_rows_type(const RowArgs& p, int sms, cudaStream_t s) {
  constexpr int N = RowVector<T>::N;
  const auto vector_rows = [](const void* base, int64_t stride) { return aligned16(base) && stride % N == 0; };
  const int vectors = p.width / N;
  // Vectors per thread.  One while there are few rows (a trip to memory and a reduction bound the call); for long batches as
  // many as pay for what a thread does once a row, as few as keep warps on the SM.  Measured (us, 1 / 2 / 4 vectors): norm
  // 16384 x 3584 with residual 69 / 78 / 82, without 57 / 54 / 67, 16384 x 8192 146 / 172 / 162 and 122 / 115 / 120; gated
  // 8192 x 4096 51 / 43 / 39, 8192 x 8192 97 / 83 / 72, 8192 x 14336 146 / 146 / 129; plain 16384 x 4096 58 / 43 / 44, 16384 x 8192
  // 117 / 83 / 80.  (A norm keeps one without a residual too: the sum of squares takes another order with two, and a row's scale has
  // the same bits whatever batch it is in.)
  const int want = p.rows <= 2 * sms || Mode == RowNorm ? 1 : Mode == RowGated || vectors > 512 ? 4 : 2;
  if (p.width % N == 0 && vector_rows(p.a, p.a_stride) && vector_rows(p.b, p.b_stride) && vector_rows(p.weight, 0) &&
      vector_rows(p.sum, p.sum_stride) && vectors <= 4096) {
    if constexpr (Mode != RowNorm) {
      if (vectors <= 32) return launch_rows_kernel<T, Mode, 1, RowWarp>(p, sms, s);
      if (vectors <= 64) return launch_rows_kernel<T, Mode, 2, RowWarp>(p, sms, s);
    }
    if (want == 1 && vectors <= 1024) return launch_rows_ring<T, Mode, 1>(p, sms, s);
    if (want <= 2 && vectors <= 2048) return launch_rows_ring<T, Mode, 2>(p, sms, s);
    return launch_rows_ring<T, Mode, 4>(p, sms, s);
  }
  // Rows that start anywhere: four vectors do not fit into the registers beside the shifts.  1 / 2 / 4 vectors: plain 8192 x 4095
  // 38 / 35 / 36, 16384 x 101 8.1 / 9.8 / 16; gated 8192 x 4095 68 / 59 / 78, 16384 x 101 12 / 19 / 39; norm with residual
  // 8192 x 4095 85 / 111 / 142, without 52 / 54 / 66.
  if ((want == 1 || vectors <= 32) && vectors < 1024) return launch_rows_kernel<T, Mode, 1, RowAnywhere>(p, sms, s);
  if (vectors < 2048) return launch_rows_kernel<T, Mode, 2, RowAnywhere>(p, sms, s);
  if (vectors < 4096) return launch_rows_kernel<T, Mode, 4, RowAnywhere>(p, sms, s);
  TRI_CUDA(launch_chained(rows_general_kernel<T, Mode>, dim3((unsigned)p.rows), dim3(1024), 0, s, p), "rows");
  return tri_launch_status("rows");
}

// SMs of the current GPU, asked for once; -1 after an error.
static int row_sms() {
  static std::atomic<int> counts[TriPerDevice::MaxDevices];
  int device = -1, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= TriPerDevice::MaxDevices) { tri_set_error("rows: no current CUDA device"); return -1; }
  n = counts[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { tri_set_error("rows: no current CUDA device"); return -1; }
    counts[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int Mode> static int launch_rows(int type, const RowArgs& p, cudaStream_t s) {
  const int sms = row_sms();
  if (sms < 0) return TRI_ERR_CUDA;
  if (type == TRI_BF16) return launch_rows_type<__nv_bfloat16, Mode>(p, sms, s);
  if (type == TRI_FP16) return launch_rows_type<__half, Mode>(p, sms, s);
  return launch_rows_type<float, Mode>(p, sms, s);
}

template <typename T> static int launch_values(const void* codes, int64_t codes_stride, const float* scales, int64_t rows, int width,
                                               void* out, int64_t out_stride, cudaStream_t s) {
  const bool vector = width % RowVector<T>::N == 0 && aligned16(out) && out_stride * sizeof(T) % 16 == 0;
  const int items = (width + RowVector<T>::N - 1) / RowVector<T>::N;
  // Threads of a row: 256, but 128 for long batches of rows that they walk in a few turns (16384 x 2560 28.8 and 25.7 us, x 3584
  // 35.8 and 34.4, x 4096 38.9 and 37.8; 8192 x 14336 63.1 and 65.0; 32 x 3584 1.7 and 2.2).
  const int most = rows >= 4096 && items <= 1024 ? 128 : 256;
  int across = 32;
  while (across < most && across < items) across *= 2;
  const dim3 block((unsigned)across, (unsigned)(256 / across));
  const int64_t blocks = (rows + block.y - 1) / block.y;
  const int sms = row_sms();
  if (sms < 0) return TRI_ERR_CUDA;
  const int64_t most_blocks = (int64_t)sms * 32;            // (8 are resident; the rest evens out the last turn)
  const dim3 grid((unsigned)(blocks < most_blocks ? blocks : most_blocks));
  const int8_t* c = static_cast<const int8_t*>(codes);
  if (vector) TRI_CUDA(launch_chained(dequantize_rows_kernel<T, true>, grid, block, 0, s, c, codes_stride, scales, static_cast<T*>(out), out_stride, rows, width), "values");
  else TRI_CUDA(launch_chained(dequantize_rows_kernel<T, false>, grid, block, 0, s, c, codes_stride, scales, static_cast<T*>(out), out_stride, rows, width), "values");
  return tri_launch_status("dequantize_rows");
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
  return launch_rows<RowPlain>(type, p, static_cast<cudaStream_t>(stream));
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
  return launch_rows<RowGated>(type, p, static_cast<cudaStream_t>(stream));
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
  p.codes = static_cast<int8_t*>(codes); p.codes_stride = codes_stride; p.scales = scales; p.width = width; p.eps = (float)eps; p.inverse_width = 1.f / (float)width;
  return launch_rows<RowNorm>(type, p, static_cast<cudaStream_t>(stream));
}

extern "C" int tri_dequantize_rows(const void* codes, int64_t codes_stride, const float* scales, int type, int64_t rows, int width,
    void* out, int64_t out_stride, void* stream) {
  TRI_CHECK(row_shape(rows, width) && row_type(type), "dequantize_rows: rows, width 1..131071, type");
  if (rows == 0) return TRI_OK;
  TRI_CHECK(codes && scales && out, "dequantize_rows: null buffers");
  TRI_CHECK(code_rows(codes, codes_stride, width), "dequantize_rows: code rows start on 16-byte boundaries");
  TRI_CHECK(row_pointer(out, type) && out_stride >= width, "dequantize_rows: output rows");
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == TRI_BF16) return launch_values<__nv_bfloat16>(codes, codes_stride, scales, rows, width, out, out_stride, s);
  if (type == TRI_FP16) return launch_values<__half>(codes, codes_stride, scales, rows, width, out, out_stride, s);
  return launch_values<float>(codes, codes_stride, scales, rows, width, out, out_stride, s);
}
