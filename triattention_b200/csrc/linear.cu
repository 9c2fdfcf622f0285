// Product of INT8 code rows with one scale per token and one per channel:
//   out[t][n] = round( (sum_k c[t][k] d[n][k]) * sd[n] * sc[t] + bias[n] + residual[t][n] )
// The sum over k is an exact 32-bit integer: |c d| <= 128 * 128, so width <= 131071 cannot overflow, and its value does not
// depend on the order of the additions (nor on how the width is split).  The rest is fp32, rounded once.
//
// One kernel for every size, tcgen05 kind::i8 with the WEIGHTS as the 128-row operand and the tokens as the N of the MMA:
// N goes from 16 to 256 in steps of 16, so a decode step of one to 256 tokens is one tile of tokens that fits it, and the
// weights (what such a step is bound by) are read once.  TMEM lane = channel, TMEM column = token; a warp's 32 lanes write
// 32 neighbouring channels of one token, which needs no alignment of the output rows.
//   warp 0      producer: TMA copies of the weights' and tokens' 128-byte columns (128-byte swizzle, edges zero-filled)
//   warp 1      issues the MMAs (one elected thread), accumulators alternate between two TMEM buffers
//   warps 2-5   epilogue: TMEM -> scales, bias, residual -> global, while the next tile's MMAs run
// A CTA takes tiles in turn (persistent).  Where there are fewer tiles than SMs the width is split over a cluster of 2, 4 or 8
// CTAs; their integer partial sums are joined through distributed shared memory, so no workspace and no atomics are involved.
// Every wait on a barrier is bounded; after one has run out the CTA runs through, reports it and its output is void.
#include "tcgen05.cuh"
#include "abi_internal.h"

namespace tri {

constexpr int LinChannels = 128, LinDepth = 128;             // channels of a tile; bytes of width per stage
constexpr int LinThreads = 192, LinEpilogue = 128;
constexpr int LinWeightBytes = LinChannels * LinDepth;
constexpr int LinShared = 216 * 1024;                        // stages (and, after a split tile, its partial sums); also keeps
                                                             // a second CTA that allocates TMEM off the SM
constexpr int LinMaxStages = 12;

struct LinearArgs {
  int64_t residual_stride, out_stride;
  const float *scales, *weight_scales;
  const void *bias, *residual;
  void* out;
  int tokens, outputs, width;
  int token_tile, stages, columns;                           // columns: TMEM columns allocated
  int channel_tiles, tiles, group;                           // group: token tiles that share a sweep over the channels
  int* error;
};

template <typename T> __device__ __forceinline__ T lin_out(float x);
template <> __device__ __forceinline__ __nv_bfloat16 lin_out(float x) { return __float2bfloat16(x); }
template <> __device__ __forceinline__ __half lin_out(float x) { return __float2half(x); }
template <> __device__ __forceinline__ float lin_out(float x) { return x; }
__device__ __forceinline__ float lin_in(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float lin_in(__half x) { return __half2float(x); }
__device__ __forceinline__ float lin_in(float x) { return x; }

__device__ __forceinline__ void lin_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_load(uint32_t address, uint32_t rank) {   // the word at `address` of the cluster's CTA `rank`
  int v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.s32 %0, [a];\n\t}"
               : "=r"(v) : "r"(address), "r"(rank) : "memory");
  return v;
}

struct LinearBarriers {
  uint64_t full[LinMaxStages], empty[LinMaxStages], done[2], free[2];
};

// grid = CTAs (persistent) when cluster size is 1, otherwise tiles * cluster size with one tile per cluster.
template <typename T> __global__ void __launch_bounds__(LinThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap map_w,
    const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearArgs p, int splits) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) LinearBarriers bars;
  __shared__ float token_scales[2][256];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  uint8_t* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int bt = p.token_tile, stage_bytes = LinWeightBytes + bt * LinDepth;
  const int rank = blockIdx.x % splits, first = blockIdx.x / splits, step = gridDim.x / splits;
  const int all_steps = (p.width + LinDepth - 1) / LinDepth;
  const int k0 = (int)((int64_t)all_steps * rank / splits), k1 = (int)((int64_t)all_steps * (rank + 1) / splits);
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&bars.full[s], 1); mbar_init(&bars.empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&bars.done[b], 1); mbar_init(&bars.free[b], LinEpilogue / 32); }
    mbar_fence_init();
    abort_flag = 0;
  }
  if (warp == 0) { tmem_alloc(&tmem_slot, p.columns); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  volatile int* abortp = &abort_flag;
  const uint32_t tmem = tmem_slot, buffer = p.columns / 2;    // columns of an accumulator buffer
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait_parked(bar, parity & 1u, abortp); };
  // tile -> first channel and first token: sweeps of `group` token tiles over all channels, so that the tiles that run at the
  // same time share both operands in L2
  auto origin = [&](int tile, int& n0, int& t0) {
    const int sweep = tile / (p.group * p.channel_tiles), within = tile % (p.group * p.channel_tiles);
    const int token_tiles = p.tiles / p.channel_tiles, wide = min(p.group, token_tiles - sweep * p.group);
    n0 = within / wide * LinChannels;
    t0 = (sweep * p.group + within % wide) * bt;
  };

  if (warp == 0) {
    if (lane == 0) {
      int i = 0;                                              // stages filled so far
      bool ok = true;
      for (int tile = first; ok && tile < p.tiles; tile += step) {
        int n0, t0;
        origin(tile, n0, t0);
        for (int k = k0; k < k1; ++k, ++i) {
          const int s = i % p.stages, round = i / p.stages;
          if (round > 0 && !(ok = wait(&bars.empty[s], round - 1))) break;
          uint8_t* stage = smem + s * stage_bytes;
          mbar_expect_tx(&bars.full[s], stage_bytes);
          tma_load_2d(stage, &map_w, k * LinDepth, n0, &bars.full[s]);
          tma_load_2d(stage + LinWeightBytes, &map_x, k * LinDepth, t0, &bars.full[s]);
        }
      }
      if (*abortp)                                            // the copies in flight land before the CTA may leave
        for (int j = max(0, i - p.stages); j < i; ++j) mbar_wait(&bars.full[j % p.stages], (j / p.stages) & 1u, 100000000ull);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc(2, 1, 1, LinChannels, bt);
      const uint32_t base = smem_u32(smem);
      int i = 0, n = 0;
      bool ok = true;
      for (int tile = first; ok && tile < p.tiles; tile += step, ++n) {
        const int b = n & 1;
        if (n >= 2 && !(ok = wait(&bars.free[b], (n >> 1) - 1))) break;
        tc_fence_after();
        for (int k = k0; k < k1; ++k, ++i) {
          const int s = i % p.stages;
          if (!(ok = wait(&bars.full[s], i / p.stages))) break;
          tc_fence_after();
          const uint64_t dw = smem_desc(base + s * stage_bytes, 0, 1024, Layout128B);
          const uint64_t dx = smem_desc(base + s * stage_bytes + LinWeightBytes, 0, 1024, Layout128B);
#pragma unroll
          for (int kk = 0; kk < LinDepth / 32; ++kk)          // 32 codes per MMA: 2 units of 16 bytes along the row
            umma_i8(tmem + b * buffer, dw + 2 * kk, dx + 2 * kk, idesc, (k > k0 || kk > 0) ? 1u : 0u);
          tc_commit(&bars.empty[s]);
        }
        tc_commit(&bars.done[b]);
      }
    }
  } else {
    const int quad = warp % 4, channel = quad * 32 + lane, et = tid - 64;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    int n = 0;
    for (int tile = first; tile < p.tiles; tile += step, ++n) {
      const int b = n & 1;
      int n0, t0;
      origin(tile, n0, t0);
      const int valid = min(bt, p.tokens - t0), out_n = n0 + channel;
      const bool live = out_n < p.outputs;
      for (int t = et; t < valid; t += LinEpilogue) token_scales[b][t] = p.scales[t0 + t];
      const float sw = live ? p.weight_scales[out_n] : 0.f;
      const float bias = live && p.bias != nullptr ? lin_in(static_cast<const T*>(p.bias)[out_n]) : 0.f;
      asm volatile("bar.sync 1, 128;" ::: "memory");          // token_scales of this tile; the other buffer's readers are a tile behind
      wait(&bars.done[b], n >> 1);                            // (no early exit: the other epilogue warps count on this one's bar.sync)
      tc_fence_after();
      if (splits > 1) {                                       // one tile per cluster: this CTA's partial sums, [token][channel]
        int* partial = reinterpret_cast<int*>(smem);
        for (int c = 0; c < valid; c += 16) {
          uint32_t a[16];
          tmem_ld16(lanes + b * buffer + c, a);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) partial[(c + j) * LinChannels + channel] = (int)a[j];
        }
        break;
      }
      T* out = static_cast<T*>(p.out) + (int64_t)t0 * p.out_stride + out_n;
      const T* residual = p.residual == nullptr ? nullptr : static_cast<const T*>(p.residual) + (int64_t)t0 * p.residual_stride + out_n;
      for (int c = 0; c < valid; c += 16) {
        uint32_t a[16];
        tmem_ld16(lanes + b * buffer + c, a);
        float r[16];
        if (residual != nullptr)
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = live && c + j < valid ? lin_in(residual[(c + j) * p.residual_stride]) : 0.f;
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float y = __fmul_rn(__fmul_rn((float)(int)a[j], sw), token_scales[b][c + j]);
          if (p.bias != nullptr) y += bias;
          if (residual != nullptr) y += r[j];
          if (live && c + j < valid) out[(c + j) * p.out_stride] = lin_out<T>(y);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) lin_arrive(&bars.free[b]);
    }
  }
  if (splits > 1) {
    // every rank finishes its share of the tokens from all ranks' partial sums
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2) {
      int n0, t0;
      origin(first, n0, t0);
      const int valid = min(bt, p.tokens - t0), channel = tid - 64, out_n = n0 + channel;
      if (out_n < p.outputs) {
        const uint32_t partial = smem_u32(smem) + channel * 4;
        const float sw = p.weight_scales[out_n], bias = p.bias != nullptr ? lin_in(static_cast<const T*>(p.bias)[out_n]) : 0.f;
        for (int t = rank; t < valid; t += splits) {
          int sum = 0;
#pragma unroll 8
          for (int r = 0; r < splits; ++r) sum += cluster_load(partial + t * LinChannels * 4, r);
          float y = __fmul_rn(__fmul_rn((float)sum, sw), p.scales[t0 + t]);
          if (p.bias != nullptr) y += bias;
          if (p.residual != nullptr) y += lin_in(static_cast<const T*>(p.residual)[(int64_t)(t0 + t) * p.residual_stride + out_n]);
          static_cast<T*>(p.out)[(int64_t)(t0 + t) * p.out_stride + out_n] = lin_out<T>(y);
        }
      }
      __syncwarp();
    }
    cluster_sync_all();                                       // nobody's shared memory goes away while it is read
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_flag) atomicExch(p.error, ErrBarrierTimeout);
  if (warp == 0) tmem_dealloc(tmem, p.columns);
}

// int8 rows: box = `box` rows x 128 bytes, 128-byte swizzle; what lies past the last row or the width reads as zero.
static int make_code_map(CUtensorMap* map, const void* base, int64_t rows, int width, int64_t stride, unsigned box) {
  EncodeTiled enc = encode_fn();
  TRI_CHECK(enc != nullptr, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride};
  const cuuint32_t boxes[2] = {(cuuint32_t)LinDepth, box}, estr[2] = {1u, 1u};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TRI_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed for code rows");
  return TRI_OK;
}

template <typename T> static int launch_linear(const CUtensorMap& map_w, const CUtensorMap& map_x, const LinearArgs& p, int ctas,
                                               int splits, cudaStream_t s) {
  static TriPerDevice configured;
  const int device = configured.pending();
  TRI_CHECK(device != -2, "int8_linear: no current CUDA device");
  if (device >= 0) {
    TRI_CUDA(cudaFuncSetAttribute(linear_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, LinShared), "int8_linear");
    configured.mark(device);
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)splits; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(LinThreads); cfg.dynamicSmemBytes = LinShared; cfg.stream = s;
  cfg.attrs = &attr; cfg.numAttrs = splits > 1 ? 1 : 0;
  TRI_CUDA(cudaLaunchKernelEx(&cfg, linear_kernel<T>, map_w, map_x, p, splits), "int8_linear");
  return tri_launch_status("int8_linear");
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
  static std::atomic<int> sm_count[TriPerDevice::MaxDevices];
  int device = -1;
  TRI_CUDA(cudaGetDevice(&device), "int8_linear");
  TRI_CHECK(device >= 0 && device < TriPerDevice::MaxDevices, "int8_linear: device");
  int sms = sm_count[device].load(std::memory_order_relaxed);
  if (sms == 0) {
    TRI_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "int8_linear");
    sm_count[device].store(sms, std::memory_order_relaxed);
  }

  LinearArgs p{};
  p.residual_stride = residual_stride; p.out_stride = out_stride; p.scales = scales; p.weight_scales = weight_scales;
  p.bias = bias; p.residual = residual; p.out = out; p.tokens = (int)tokens; p.outputs = outputs; p.width = width; p.error = device_error;
  p.token_tile = (int)(tokens >= 256 ? 256 : (tokens + 15) / 16 * 16);
  p.channel_tiles = (outputs + LinChannels - 1) / LinChannels;
  const int64_t tiles = (tokens + p.token_tile - 1) / p.token_tile * (int64_t)p.channel_tiles;
  TRI_CHECK(tiles <= 0x7fffffff / 8, "int8_linear: tokens * outputs");
  p.tiles = (int)tiles;
  p.group = 8;
  p.stages = (LinShared - 1024) / (LinWeightBytes + p.token_tile * LinDepth);
  if (p.stages > LinMaxStages) p.stages = LinMaxStages;
  p.columns = 32;
  while (p.columns < 2 * p.token_tile) p.columns *= 2;
  const int steps = (width + LinDepth - 1) / LinDepth;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 * 2 <= steps) splits *= 2;
  const int ctas = splits > 1 ? p.tiles * splits : (p.tiles < sms ? p.tiles : sms);
  CUtensorMap map_w, map_x;
  if (make_code_map(&map_w, weight, outputs, width, weight_stride, LinChannels) != TRI_OK) return TRI_ERR_CUDA;
  if (make_code_map(&map_x, codes, tokens, width, codes_stride, (unsigned)p.token_tile) != TRI_OK) return TRI_ERR_CUDA;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (type == TRI_BF16) return launch_linear<__nv_bfloat16>(map_w, map_x, p, ctas, splits, s);
  if (type == TRI_FP16) return launch_linear<__half>(map_w, map_x, p, ctas, splits, s);
  return launch_linear<float>(map_w, map_x, p, ctas, splits, s);
}
