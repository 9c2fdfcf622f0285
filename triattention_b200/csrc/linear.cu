// Product of INT8 code rows with one scale per token and one per channel:
//   out[t][n] = round( (sum_k c[t][k] d[n][k]) * sd[n] * sc[t] + bias[n] + residual[t][n] )
// The sum over k is an exact 32-bit integer: |c d| <= 128 * 128, so width <= 131071 cannot overflow, and its value does not
// depend on the order of the additions (nor on how the width is split).  The rest is IEEE fp32 (subnormal numbers too: this file is
// compiled without --use_fast_math), rounded once.
//
// tcgen05 kind::i8 with the WEIGHTS as the 128-row operand and the tokens as the N of the MMA: N goes from 16 to 256 in steps of
// 16, so a decode step of two to 256 tokens is one tile of tokens that fits it, and the weights (what such a step is bound by)
// are read once (a single token has a kernel of its own, linear_row_kernel).  TMEM lane = channel, TMEM column = token.
//   warp 0      producer: TMA copies of the weights' and tokens' 128-byte columns (128-byte swizzle, edges zero-filled)
//   warp 1      issues the MMAs (one elected thread), accumulators alternate between two TMEM buffers
//   warps 2-    epilogue: TMEM -> scales, bias, residual -> global, while the next tiles' MMAs run
// A CTA takes tiles in turn (persistent).  Where there are fewer tiles than SMs the width is split over a cluster of up to 8 CTAs;
// their integer partial sums are joined through distributed shared memory, so no workspace and no atomics are involved.  A row of
// the result has the same bits whatever else is in the batch: only the exact sums depend on tile and split.
// Every wait on a barrier is bounded; after one has run out the CTA runs through, reports it and its output is void.
//
// Measured on one B200 (device time; DRAM-cold weights): 16 x 4096 -> 128256 fp32 84 us = 6.3 TB/s, bound by HBM; 32 x 3584 -> 4608
// 8.2-9.0 us depending on the GPU, bound by latencies (launch, first bytes, cluster exchange: of width 128 3.0, of 1024 5.1, the
// smallest product 2.7); 16384 x 14336 -> 4096 with residual 602-632 us = 3.0-3.2 POP/s in bursts, bound by the 1000 W limit when it
// runs for seconds.
#include "tcgen05.cuh"
#include "abi_internal.h"
#include <mutex>
#include <type_traits>

namespace tri {

constexpr int LinChannels = 128, LinDepth = 128;             // channels of a CTA's tile; bytes of width per step
constexpr int LinWarps = 8, LinSmallWarps = 4;               // epilogue warps of a group, where a CTA has the SM to itself and where two
                                                             // share it; two groups take a CTA's tiles in turn
__host__ __device__ constexpr int lin_threads(int warps) { return 64 + 2 * 32 * warps; }
constexpr int LinWeightBytes = LinChannels * LinDepth;
constexpr int LinShared = 193 * 1024;                        // stages (and, after a split tile, its partial sums); also keeps
                                                             // a second CTA that allocates TMEM off the SM
constexpr int LinSmallTile = 64, LinSharedSmall = 97 * 1024;  // up to this token tile two CTAs fit on an SM (and in TMEM)
constexpr int LinMaxStages = 12;

struct LinearArgs {
  int64_t residual_stride, out_stride;
  const float *scales, *weight_scales;
  const void *bias, *residual;
  void* out;
  int tokens, outputs, width;
  int token_tile, stages, columns;                           // columns: TMEM columns allocated
  int channel_tiles, tiles, group;                           // group: token tiles that share a sweep over the channels
  int splits;                                                // CTAs of a cluster that share a tile's width
  int shared;                                                // dynamic shared memory
  int ahead;                                                 // steps whose weights are asked for before the kernel before this one has ended
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
__device__ __forceinline__ int4 cluster_load(uint32_t address, uint32_t rank) {   // 16 bytes at `address` of the cluster's CTA `rank`
  int4 v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [a];\n\t}"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address), "r"(rank) : "memory");
  return v;
}

// The same operations as in common.cuh on 32-bit shared-memory addresses.
__device__ __forceinline__ bool lin_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool lin_wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  const uint64_t t0 = globaltimer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (lin_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (globaltimer_ns() - t0 > 2000000000ull) { *abort_flag = 1; return false; }
  }
}
__device__ __forceinline__ bool lin_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (lin_try_wait(bar, parity)) return true;
  return lin_wait_long(bar, parity, abort_flag);
}
__device__ __forceinline__ void lin_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void lin_copy(uint32_t to, const CUtensorMap* map, int column, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(column), "r"(row), "r"(bar) : "memory");
}
__device__ __forceinline__ void lin_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void lin_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void lin_prefetch_box(const CUtensorMap* map, int column, int row) {      // into L2
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(column), "r"(row) : "memory");
}

// The forms for a pair of CTAs.  In a shared::cluster address of a pair bit 24 tells the two CTAs apart: barrier addresses with it
// cleared name the even CTA's barrier at the same place.
constexpr uint32_t PairEven = 0xfeffffffu;
__device__ __forceinline__ void pair_alloc(uint32_t* slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_dealloc(uint32_t tmem, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ void pair_copy(uint32_t to, const CUtensorMap* map, int column, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(column), "r"(row), "r"(bar & PairEven) : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void pair_commit(uint32_t bar) {        // arrives at this barrier of both CTAs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void pair_arrive(uint32_t bar) {        // arrives at the even CTA's barrier
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\tmbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(bar) : "memory");
}

struct LinearBarriers {
  uint64_t full[LinMaxStages], empty[LinMaxStages], done[2], free[2];
};

// tile -> first channel and first token: sweeps of `group` token tiles over all channels, so that the tiles that run at the
// same time share both operands in L2.
__device__ __forceinline__ void lin_origin(const LinearArgs& p, int tile, int channels, int& n0, int& t0) {
  const int sweep = tile / (p.group * p.channel_tiles), within = tile % (p.group * p.channel_tiles);
  const int token_tiles = p.tiles / p.channel_tiles, wide = min(p.group, token_tiles - sweep * p.group);
  n0 = within / wide * channels;
  t0 = (sweep * p.group + within % wide) * p.token_tile;
}

// C neighbouring channels of one token as one access.
template <typename T, int C> struct LinVector {
  alignas(C * sizeof(T)) T v[C];
};
// The same as it is read ahead: 32-bit words, taken apart only where they are used.  (With elements of 16 bits the compiler takes
// them apart right behind the load, which waits for it: 16384 x 4096 outputs of width 128 with a residual took 120 us, now 74; of width 4096 210 and 190.)
template <typename T, int C> struct LinWords {
  alignas(C * sizeof(T) < 4 ? 4 : C * sizeof(T)) uint32_t w[(C * sizeof(T) + 3) / 4];
  __device__ __forceinline__ void load(const T* from) {
    constexpr int B = C * sizeof(T);
    if constexpr (B == 16) *reinterpret_cast<uint4*>(w) = __ldcs(reinterpret_cast<const uint4*>(from));
    else if constexpr (B == 8) *reinterpret_cast<uint2*>(w) = __ldcs(reinterpret_cast<const uint2*>(from));
    else if constexpr (B == 4) w[0] = __ldcs(reinterpret_cast<const uint32_t*>(from));
    else w[0] = *reinterpret_cast<const unsigned short*>(from);
  }
  __device__ __forceinline__ void load_some(const T* from, int count) {
#pragma unroll
    for (int k = 0; k < C; ++k) {
      uint32_t bits = 0;
      if (k < count) {
        if constexpr (sizeof(T) == 4) bits = *reinterpret_cast<const uint32_t*>(from + k);
        else bits = *reinterpret_cast<const unsigned short*>(from + k);
      }
      if constexpr (sizeof(T) == 4) w[k] = bits;
      else w[k / 2] = k % 2 ? w[k / 2] | bits << 16 : bits;
    }
  }
  __device__ __forceinline__ float value(int k) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[k]);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(k % 2 ? w[k / 2] & 0xffff0000u : w[k / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(w[k / 2] >> (16 * (k % 2)))));
  }
};
template <typename T, int C> __device__ __forceinline__ void lin_store(T* to, const LinVector<T, C>& x) {
  constexpr int B = C * sizeof(T);
  if constexpr (B == 16) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(x.v);
  else if constexpr (B == 8) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(x.v);
  else if constexpr (B == 4) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(x.v);
  else *to = x.v[0];
}

// Epilogue of one tile by a group of Warps warps: 128 channels from n0 on (TMEM lanes), `valid` tokens from t0 on (columns).
// The group's warps of a lane quadrant take blocks of 16 tokens x 32 channels in turn.  A lane holds one channel of 16 tokens; the scaled
// block goes, 8 tokens at a time, through the warp's own shared memory, out of which a lane takes C neighbouring channels of a
// token (C: what the rows of output and residual allow, 16 bytes at most), so that the residual is read and the result written in
// wide accesses.  Two groups, because most of a tile's epilogue is latency (scales, the accumulators' barrier, TMEM, the residual):
// they overlap those of two tiles (with a residual, 16384 x 4096 outputs of width 4096: 249 us with one group of all warps, 210 with two).
// `ready` is called once, when everything that does not depend on the sums is under way.
constexpr int LinPitch = 36, LinBlockTokens = 8, LinBlockFloats = LinBlockTokens * LinPitch;   // pitch: no two lanes on one bank either way
template <typename T, int C, int Warps, bool Residual, typename Ready>
__device__ __forceinline__ void lin_epilogue_as(const LinearArgs& p, uint32_t column, int n0, int t0, int valid, float* token_scales,
                                                float* block, Ready ready) {
  constexpr int Passes = 16 / C, Across = 32 / C;             // passes over a block's 16 tokens; lanes per token
  constexpr int Step = 4 * Warps;                             // tokens from one block of a warp to its next
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = warp % 4, member = (warp - 2) % Warps, c0 = member / 4 * 16;
  const int first_n = n0 + quad * 32, safe_n = min(first_n + lane, p.outputs - 1);       // (what a lane past the last channel may read)
  column += (uint32_t)(quad * 32) << 16;
  const int my_token = lane / Across, my_n = first_n + lane % Across * C, count = min(C, p.outputs - my_n);
  const bool all = count >= C;
  const int64_t out_step = C * p.out_stride, residual_step = C * p.residual_stride;      // from pass to pass
  // the residual is asked for two blocks ahead (the first two under the MMAs): one trip to HBM outlasts a block by far
  using Ahead = LinWords<T, C>[Residual ? Passes : 1];
  Ahead even, odd;
  auto fetch = [&](Ahead& ahead, int c) {
    const T* from = static_cast<const T*>(p.residual) + (int64_t)(t0 + c + my_token) * p.residual_stride + my_n;
#pragma unroll
    for (int i = 0; i < (Residual ? Passes : 0); ++i, from += residual_step) {
      if (c + i * C + my_token < valid) {
        if (all) ahead[i].load(from);
        else ahead[i].load_some(from, count);
      }
    }
  };
  if (Residual && c0 < valid) fetch(even, c0);
  if (Residual && c0 + Step < valid) fetch(odd, c0 + Step);
  for (int t = 32 * member + lane; t < valid; t += 32 * Warps) token_scales[t] = p.scales[t0 + t];
  const float sw = p.weight_scales[safe_n], bias = p.bias != nullptr ? lin_in(static_cast<const T*>(p.bias)[safe_n]) : 0.f;
  // token_scales of this tile are complete (and the other buffer's readers a tile behind); waits have no early exit, because
  // the group's other warps count on this one at the barrier
  asm volatile("bar.sync %0, %1;" ::"r"(1 + (warp - 2) / Warps), "n"(32 * Warps) : "memory");
  ready();
  tc_fence_after();
  T* out = static_cast<T*>(p.out) + (int64_t)(t0 + c0 + my_token) * p.out_stride + my_n;
  const int64_t block_step = Step * p.out_stride;
  float* const mine = block + lane;
  const float* const from = block + my_token * LinPitch + lane % Across * C;
  uint32_t a[16];
  if (c0 < valid) tmem_ld16(column + c0, a);
  auto work = [&](Ahead& ahead, int c) {
    tmem_ld_wait();
    T* to = out;
#pragma unroll
    for (int part = 0; part < 16; part += LinBlockTokens) {
#pragma unroll
      for (int j = 0; j < LinBlockTokens; j += 4) {
        const float4 st = *reinterpret_cast<const float4*>(&token_scales[c + part + j]);
        mine[j * LinPitch] = fmaf(__fmul_rn((float)(int)a[part + j], sw), st.x, bias);
        mine[(j + 1) * LinPitch] = fmaf(__fmul_rn((float)(int)a[part + j + 1], sw), st.y, bias);
        mine[(j + 2) * LinPitch] = fmaf(__fmul_rn((float)(int)a[part + j + 2], sw), st.z, bias);
        mine[(j + 3) * LinPitch] = fmaf(__fmul_rn((float)(int)a[part + j + 3], sw), st.w, bias);
      }
      if (part + LinBlockTokens == 16 && c + Step < valid) tmem_ld16(column + c + Step, a);    // on its way while this block is written out
      __syncwarp();
#pragma unroll
      for (int i = 0; i < LinBlockTokens / C; ++i, to += out_step) {
        constexpr int Skip = C * LinPitch;
        const int pass = part / C + i;
        alignas(16) float y[C];
        if constexpr (C >= 4) {
#pragma unroll
          for (int k = 0; k < C; k += 4) *reinterpret_cast<float4*>(y + k) = *reinterpret_cast<const float4*>(from + i * Skip + k);
        } else if constexpr (C == 2) {
          *reinterpret_cast<float2*>(y) = *reinterpret_cast<const float2*>(from + i * Skip);
        } else {
          y[0] = from[i * Skip];
        }
        LinVector<T, C> x;
#pragma unroll
        for (int k = 0; k < C; ++k) x.v[k] = lin_out<T>(Residual ? y[k] + ahead[Residual ? pass : 0].value(k) : y[k]);
        if (c + pass * C + my_token < valid) {
          if (all) {
            lin_store<T, C>(to, x);
          } else {
#pragma unroll
            for (int k = 0; k < C; ++k) if (k < count) to[k] = x.v[k];
          }
        }
      }
      __syncwarp();                                           // the block has been read
    }
    if (Residual && c + 2 * Step < valid) fetch(ahead, c + 2 * Step);
    out += block_step;
  };
  for (int c = c0; c < valid; c += 2 * Step) {
    work(even, c);
    if (c + Step < valid) work(odd, c + Step);
  }
  tc_fence_before();
  __syncwarp();
}
template <typename T, int C, int Warps, typename Ready>
__device__ __forceinline__ void lin_epilogue(const LinearArgs& p, uint32_t column, int n0, int t0, int valid, float* token_scales,
                                             float* blocks, Ready ready) {
  float* block = blocks + (threadIdx.x / 32 - 2) * LinBlockFloats;
  if (p.residual != nullptr) lin_epilogue_as<T, C, Warps, true>(p, column, n0, t0, valid, token_scales, block, ready);
  else lin_epilogue_as<T, C, Warps, false>(p, column, n0, t0, valid, token_scales, block, ready);
}

// One CTA per tile of 128 channels; Small: two of them per SM; Deep: steps of 128 bytes of width that a stage holds.
// grid = CTAs (persistent) when splits is 1, otherwise tiles * splits with one tile per cluster.
template <typename T, int C, bool Small, int Deep>
__global__ void __launch_bounds__(lin_threads(Small ? LinSmallWarps : LinWarps), Small ? 2 : 1)
    linear_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearArgs p) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) LinearBarriers bars;
  __shared__ __align__(16) float token_scales[2][2][256];      // [group][the group's turn]
  constexpr int Warps = Small ? LinSmallWarps : LinWarps;
  __shared__ __align__(16) float blocks[2 * Warps * LinBlockFloats];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  uint8_t* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int bt = p.token_tile, step_bytes = LinWeightBytes + bt * LinDepth, stage_bytes = Deep * step_bytes, splits = p.splits;
  const int rank = blockIdx.x % splits, first = blockIdx.x / splits, step = gridDim.x / splits;
  const int all_steps = (p.width + LinDepth - 1) / LinDepth;
  const int k0 = (int)((int64_t)all_steps * rank / splits), k1 = (int)((int64_t)all_steps * (rank + 1) / splits);
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) { mbar_init(&bars.full[s], 1); mbar_init(&bars.empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&bars.done[b], 1); mbar_init(&bars.free[b], Warps); }
    mbar_fence_init();
    abort_flag = 0;
  }
  if (tid == 32) {
    lin_prefetch(&map_w); lin_prefetch(&map_x);
    if (p.ahead > 0 && first < p.tiles) {
      int n0, t0;
      lin_origin(p, first, LinChannels, n0, t0);
      for (int k = k0; k < min(k1, k0 + p.ahead); ++k) lin_prefetch_box(&map_w, k * LinDepth, n0);
    }
  }
  if (warp == 0) { tmem_alloc(&tmem_slot, p.columns); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();
  grid_dependency_wait();            // the set-up above overlaps the tail of the kernel before this one in the stream
  volatile int* abortp = &abort_flag;
  const uint32_t tmem = tmem_slot, buffer = p.columns / 2;    // columns of an accumulator buffer
  // (The loops of the two issuing threads are serial code that the whole CTA waits for: shared-memory addresses as 32-bit numbers
  // that only advance, no divisions.  With indexes and remainders a stage took 640 cycles, however little it held.)
  const uint32_t smem_base = smem_u32(smem), full_base = smem_u32(&bars.full[0]), empty_base = smem_u32(&bars.empty[0]);
  const int stages = p.stages;
  if (warp == 0) {
    if (lane == 0) {
      uint32_t at = smem_base, full = full_base, empty = empty_base, phase = 1;
      int stage = 0, filled = 0;
      bool ok = true;
      for (int tile = first; ok && tile < p.tiles; tile += step) {
        int n0, t0;
        lin_origin(p, tile, LinChannels, n0, t0);
        for (int k = k0; k < k1; k += Deep) {
          if (filled >= stages && !(ok = lin_wait(empty, phase, abortp))) break;
          const bool both = Deep > 1 && k + 1 < k1;
          lin_expect(full, both ? stage_bytes : step_bytes);
          lin_copy(at, &map_w, k * LinDepth, n0, full);
          lin_copy(at + LinWeightBytes, &map_x, k * LinDepth, t0, full);
          if (both) {
            lin_copy(at + step_bytes, &map_w, (k + 1) * LinDepth, n0, full);
            lin_copy(at + step_bytes + LinWeightBytes, &map_x, (k + 1) * LinDepth, t0, full);
          }
          ++filled;
          at += stage_bytes; full += 8; empty += 8;
          if (++stage == stages) { stage = 0; at = smem_base; full = full_base; empty = empty_base; phase ^= 1u; }
        }
      }
      if (*abortp)                                            // the copies in flight land before the CTA may leave
        for (int j = max(0, filled - stages); j < filled; ++j) mbar_wait(&bars.full[j % stages], (j / stages) & 1u, 100000000ull);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc(2, 1, 1, LinChannels, bt);
      const uint64_t desc = smem_desc(smem_base, 0, 1024, Layout128B);
      const uint32_t stage_units = stage_bytes >> 4, step_units = step_bytes >> 4;   // descriptors address 16-byte units, all below 2^14
      uint32_t full = full_base, empty = empty_base, phase = 0;
      int stage = 0, n = 0;
      uint64_t dw = desc;
      bool ok = true;
      for (int tile = first; ok && tile < p.tiles; tile += step, ++n) {
        const int b = n & 1;
        if (n >= 2 && !(ok = lin_wait(smem_u32(&bars.free[b]), ((n >> 1) - 1) & 1, abortp))) break;
        tc_fence_after();
        const uint32_t acc = tmem + b * buffer;
        uint32_t accumulate = 0;
        for (int k = k0; k < k1; k += Deep) {
          if (!(ok = lin_wait(full, phase, abortp))) break;
          tc_fence_after();
          const uint64_t dx = dw + (LinWeightBytes >> 4);
          umma_i8(acc, dw, dx, idesc, accumulate);            // 32 codes per MMA: 2 units of 16 bytes along the row
#pragma unroll
          for (int kk = 1; kk < LinDepth / 32; ++kk) umma_i8(acc, dw + 2 * kk, dx + 2 * kk, idesc, 1u);
          if (Deep > 1 && k + 1 < k1) {
#pragma unroll
            for (int kk = 0; kk < LinDepth / 32; ++kk) umma_i8(acc, dw + step_units + 2 * kk, dx + step_units + 2 * kk, idesc, 1u);
          }
          lin_commit(empty);
          accumulate = 1;
          dw += stage_units; full += 8; empty += 8;
          if (++stage == stages) { stage = 0; phase ^= 1u; dw = desc; full = full_base; empty = empty_base; }
        }
        tc_commit(&bars.done[b]);
      }
    }
  } else if (splits == 1) {
    if (p.tiles <= step) {                                    // one tile per CTA: all warps share it
      if (first < p.tiles) {
        int n0, t0;
        lin_origin(p, first, LinChannels, n0, t0);
        lin_epilogue<T, C, 2 * Warps>(p, tmem, n0, t0, min(bt, p.tokens - t0), token_scales[0][0], blocks,
                                      [&] { lin_wait(smem_u32(&bars.done[0]), 0, abortp); });
      }
    }
    const int b = (warp - 2) / Warps;                         // group, and the accumulator buffer that it empties
    uint32_t turn = 0;
    for (int tile = first + b * step; p.tiles > step && tile < p.tiles; tile += 2 * step, turn ^= 1) {
      int n0, t0;
      lin_origin(p, tile, LinChannels, n0, t0);
      lin_epilogue<T, C, Warps>(p, tmem + b * buffer, n0, t0, min(bt, p.tokens - t0), token_scales[b][turn], blocks,
                      [&] { lin_wait(smem_u32(&bars.done[b]), turn, abortp); });
      if (lane == 0) lin_arrive(&bars.free[b]);
    }
  } else {                                                    // one tile per cluster: this CTA's partial sums, [token][channel]
    const int quad = warp % 4, channel = quad * 32 + lane;
    int n0, t0;
    lin_origin(p, first, LinChannels, n0, t0);
    const int valid = min(bt, p.tokens - t0);
    lin_wait(smem_u32(&bars.done[0]), 0, abortp);
    tc_fence_after();
    int* partial = reinterpret_cast<int*>(smem);
    for (int c = (warp - 2) / 4 * 16; c < valid; c += 8 * Warps) {
      uint32_t a[16];
      tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + c, a);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) partial[(c + j) * LinChannels + channel] = (int)a[j];
    }
  }
  if (splits > 1) {
    // Every rank finishes its share of the tokens from all ranks' partial sums: a warp takes a token, a lane four channels.
    int n0, t0;
    lin_origin(p, first, LinChannels, n0, t0);
    const int valid = min(bt, p.tokens - t0), n = n0 + 4 * lane, count = min(4, p.outputs - n);
    float sw[4], bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int safe = min(n + i, p.outputs - 1);
      sw[i] = p.weight_scales[safe];
      bias[i] = p.bias != nullptr ? lin_in(static_cast<const T*>(p.bias)[safe]) : 0.f;
    }
    __syncwarp();
    cluster_sync_all();
    const uint32_t partial = smem_base + lane * 16;
    for (int t = rank + warp * splits; t < valid; t += splits * (lin_threads(Warps) / 32)) {
      const float st = p.scales[t0 + t];
      float r[4] = {};
      if (p.residual != nullptr) {
        const T* from = static_cast<const T*>(p.residual) + (int64_t)(t0 + t) * p.residual_stride;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = lin_in(from[min(n + i, p.outputs - 1)]);
      }
      int4 v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = q < splits ? cluster_load(partial + t * LinChannels * 4, q) : make_int4(0, 0, 0, 0);
      int sum[4] = {};
#pragma unroll
      for (int q = 0; q < 8; ++q) { sum[0] += v[q].x; sum[1] += v[q].y; sum[2] += v[q].z; sum[3] += v[q].w; }
      T* to = static_cast<T*>(p.out) + (int64_t)(t0 + t) * p.out_stride + n;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y = fmaf(__fmul_rn((float)sum[i], sw[i]), st, bias[i]);    // (the epilogue's arithmetic)
        if (p.residual != nullptr) y += r[i];
        if (i < count) to[i] = lin_out<T>(y);
      }
    }
    __syncwarp();
    cluster_sync_all();                                       // nobody's shared memory goes away while it is read
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && abort_flag) atomicExch(p.error, ErrBarrierTimeout);
  if (warp == 0) tmem_dealloc(tmem, p.columns);
}

// Two CTAs (a cluster of 2) per tile of 256 channels x token_tile tokens: MMAs of M = 256 that run on both SMs' tensor cores
// (cta_group::2).  Each CTA holds its own 128 channels and half of the tokens, so an SM fetches 32 KB per 128 bytes of width
// where a CTA alone fetches 48 KB for the same work, and the SM's port to L2 is what bounds the product of two large operands.
// The even CTA issues the MMAs of both; copies of both report to its `full` barriers, commits arrive at both CTAs' barriers.
template <typename T, int C>
__global__ void __launch_bounds__(lin_threads(LinWarps), 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ LinearArgs p) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ __align__(8) LinearBarriers bars;
  __shared__ __align__(16) float token_scales[2][2][256];      // [group][the group's turn]
  __shared__ __align__(16) float blocks[2 * LinWarps * LinBlockFloats];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  uint8_t* smem = raw_smem + ((1024u - (smem_u32(raw_smem) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  constexpr int Deep = 2;
  const int bt = p.token_tile, step_bytes = LinWeightBytes + bt / 2 * LinDepth, stage_bytes = Deep * step_bytes;
  const int rank = blockIdx.x & 1, first = blockIdx.x / 2, step = gridDim.x / 2;
  const int steps = (p.width + LinDepth - 1) / LinDepth, stages = p.stages;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(&bars.full[s], 1); mbar_init(&bars.empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&bars.done[b], 1); mbar_init(&bars.free[b], 2 * LinWarps); }
    mbar_fence_init();
    abort_flag = 0;
  }
  if (tid == 32) { lin_prefetch(&map_w); lin_prefetch(&map_x); }
  if (warp == 0) pair_alloc(&tmem_slot, p.columns);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                         // both CTAs' barriers exist before anything arrives at them
  tc_fence_after();
  grid_launch_dependents();
  grid_dependency_wait();
  volatile int* abortp = &abort_flag;
  const uint32_t tmem = tmem_slot, buffer = p.columns / 2;
  const uint32_t smem_base = smem_u32(smem), full_base = smem_u32(&bars.full[0]), empty_base = smem_u32(&bars.empty[0]);
  if (warp == 0) {
    if (lane == 0) {
      uint32_t at = smem_base, full = full_base, empty = empty_base, phase = 1;
      int stage = 0, filled = 0;
      bool ok = true;
      for (int tile = first; ok && tile < p.tiles; tile += step) {
        int n0, t0;
        lin_origin(p, tile, 2 * LinChannels, n0, t0);
        n0 += rank * LinChannels; t0 += rank * (bt / 2);
        for (int k = 0; k < steps; k += Deep) {
          if (filled >= stages && !(ok = lin_wait(empty, phase, abortp))) break;
          const bool both = Deep > 1 && k + 1 < steps;
          if (rank == 0) lin_expect(full, 2 * (both ? stage_bytes : step_bytes));   // what both CTAs' copies bring
          pair_copy(at, &map_w, k * LinDepth, n0, full);
          pair_copy(at + LinWeightBytes, &map_x, k * LinDepth, t0, full);
          if (both) {
            pair_copy(at + step_bytes, &map_w, (k + 1) * LinDepth, n0, full);
            pair_copy(at + step_bytes + LinWeightBytes, &map_x, (k + 1) * LinDepth, t0, full);
          }
          ++filled;
          at += stage_bytes; full += 8; empty += 8;
          if (++stage == stages) { stage = 0; at = smem_base; full = full_base; empty = empty_base; phase ^= 1u; }
        }
      }
      if (*abortp && rank == 0)                               // the copies in flight land before the CTAs may leave
        for (int j = max(0, filled - stages); j < filled; ++j) mbar_wait(&bars.full[j % stages], (j / stages) & 1u, 100000000ull);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = instr_desc(2, 1, 1, 2 * LinChannels, bt);
      const uint64_t desc = smem_desc(smem_base, 0, 1024, Layout128B);
      const uint32_t stage_units = stage_bytes >> 4, step_units = step_bytes >> 4;
      uint32_t full = full_base, empty = empty_base, phase = 0;
      int stage = 0, n = 0;
      uint64_t dw = desc;
      bool ok = true;
      for (int tile = first; ok && tile < p.tiles; tile += step, ++n) {
        const int b = n & 1;
        if (n >= 2 && !(ok = lin_wait(smem_u32(&bars.free[b]), ((n >> 1) - 1) & 1, abortp))) break;
        tc_fence_after();
        const uint32_t acc = tmem + b * buffer;
        uint32_t accumulate = 0;
        for (int k = 0; k < steps; k += Deep) {
          if (!(ok = lin_wait(full, phase, abortp))) break;
          tc_fence_after();
          const uint64_t dx = dw + (LinWeightBytes >> 4);
          pair_umma(acc, dw, dx, idesc, accumulate);
#pragma unroll
          for (int kk = 1; kk < LinDepth / 32; ++kk) pair_umma(acc, dw + 2 * kk, dx + 2 * kk, idesc, 1u);
          if (Deep > 1 && k + 1 < steps) {
#pragma unroll
            for (int kk = 0; kk < LinDepth / 32; ++kk) pair_umma(acc, dw + step_units + 2 * kk, dx + step_units + 2 * kk, idesc, 1u);
          }
          pair_commit(empty);
          accumulate = 1;
          dw += stage_units; full += 8; empty += 8;
          if (++stage == stages) { stage = 0; phase ^= 1u; dw = desc; full = full_base; empty = empty_base; }
        }
        pair_commit(smem_u32(&bars.done[b]));
      }
    }
  } else {
    if (p.tiles <= step && first < p.tiles) {
      int n0, t0;
      lin_origin(p, first, 2 * LinChannels, n0, t0);
      lin_epilogue<T, C, 2 * LinWarps>(p, tmem, n0 + rank * LinChannels, t0, min(bt, p.tokens - t0), token_scales[0][0], blocks,
                                       [&] { lin_wait(smem_u32(&bars.done[0]), 0, abortp); });
    }
    const int b = (warp - 2) / LinWarps;
    uint32_t turn = 0;
    for (int tile = first + b * step; p.tiles > step && tile < p.tiles; tile += 2 * step, turn ^= 1) {
      int n0, t0;
      lin_origin(p, tile, 2 * LinChannels, n0, t0);
      lin_epilogue<T, C, LinWarps>(p, tmem + b * buffer, n0 + rank * LinChannels, t0, min(bt, p.tokens - t0), token_scales[b][turn], blocks,
                      [&] { lin_wait(smem_u32(&bars.done[b]), turn, abortp); });
      if (lane == 0) pair_arrive(smem_u32(&bars.free[b]));
    }
  }
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_sync_all();                                         // the partner's MMAs and arrivals reach into this CTA until here
  if (tid == 0 && abort_flag) atomicExch(p.error, ErrBarrierTimeout);
  if (warp == 0) pair_dealloc(tmem, p.columns);
}

// One token: a warp per channel, whose codes it reads once, 16 bytes a lane, four products an instruction.  No tensor core, no TMEM,
// no cluster: a call is the trip to memory and one reduction across the warp.  `Ahead` loads of a lane are under way at a time, twice
// as many in the Deep form, which takes registers that more than 32 warps an SM do not have.  Measured (us, DRAM-cold weights, with
// the quantisation before it; tensor cores / this / this, Deep): 4096 -> 6144 11.3 / 7.7 / 8.0, 4096 -> 4096 8.5 / 6.1 / 5.9,
// 14336 -> 4096 17.4 / 15.3 / 13.7, 14336 -> 256 10.2 / 11.9 / 9.9, 4096 -> 28672 24.0 / 22.3 / 23.0, 4096 -> 128256 84 / 79 / 90.
// Alone 4096 -> 6144 takes 4.6 us (5.4 TB/s), 9.6 on the tensor cores.  Two tokens are faster there already (4096 -> 28672: 24.0 us,
// 28.6 like this).
constexpr int LinRowWarps = 4, LinRowDeep = 32;               // LinRowDeep: warps an SM up to which the Deep form is taken
__device__ __forceinline__ uint4 row_end_codes(const int8_t* from, int count) {     // the last 1..15 codes of a row, then zeros
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < 15; ++i) if (i < count) w[i / 4] |= (uint32_t)(uint8_t)from[i] << (8 * (i % 4));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int sum) {
  sum = __dp4a((int)a.x, (int)b.x, sum);
  sum = __dp4a((int)a.y, (int)b.y, sum);
  sum = __dp4a((int)a.z, (int)b.z, sum);
  return __dp4a((int)a.w, (int)b.w, sum);
}
template <typename T, bool Deep> __global__ void __launch_bounds__(32 * LinRowWarps)
    linear_row_kernel(const int8_t* codes, const int8_t* weight, int64_t weight_stride, const __grid_constant__ LinearArgs p) {
  constexpr int Ahead = 4, Step = 512, Chunk = Ahead * Step;  // Step: bytes that a warp reads at a time
  const int lane = threadIdx.x % 32, whole = p.width & ~15;
  const int64_t step = (int64_t)gridDim.x * LinRowWarps;
  int64_t n = (int64_t)blockIdx.x * LinRowWarps + threadIdx.x / 32;
  grid_launch_dependents();
  if (n < p.outputs)                                          // into L2 only, under the kernel that makes the codes
    for (int e = lane * 128; e < min(p.width, 4096); e += 4096)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(weight + n * weight_stride + e));
  grid_dependency_wait();
  const float st = p.scales[0];
  for (; n < p.outputs; n += step) {
    const int8_t* row = weight + n * weight_stride;
    const auto fetch = [&](uint4 (&w)[Ahead], int e) {
#pragma unroll
      for (int a = 0; a < Ahead; ++a) {
        w[a] = make_uint4(0, 0, 0, 0);
        if (e + a * Step < whole) w[a] = __ldcs(reinterpret_cast<const uint4*>(row + e + a * Step));
      }
    };
    int sum = 0;
    const auto work = [&](const uint4 (&w)[Ahead], int e) {
      uint4 c[Ahead];
#pragma unroll
      for (int a = 0; a < Ahead; ++a) {
        c[a] = make_uint4(0, 0, 0, 0);
        if (e + a * Step < whole) c[a] = *reinterpret_cast<const uint4*>(codes + e + a * Step);
      }
#pragma unroll
      for (int a = 0; a < Ahead; ++a) sum = dot16(c[a], w[a], sum);
    };
    const float sw = p.weight_scales[n], bias = p.bias != nullptr ? lin_in(static_cast<const T*>(p.bias)[n]) : 0.f;
    const float r = p.residual != nullptr ? lin_in(static_cast<const T*>(p.residual)[n]) : 0.f;
    uint4 even[Ahead], odd[Ahead];
    if constexpr (Deep) {
      fetch(even, lane * 16);
      for (int e = lane * 16; e < whole; e += 2 * Chunk) {
        fetch(odd, e + Chunk);
        work(even, e);
        fetch(even, e + 2 * Chunk);
        work(odd, e + Chunk);
      }
    } else {
      for (int e = lane * 16; e < whole; e += Chunk) {
        fetch(even, e);
        work(even, e);
      }
    }
    if (whole < p.width && lane == 31) sum = dot16(row_end_codes(codes + whole, p.width - whole), row_end_codes(row + whole, p.width - whole), sum);
    sum = __reduce_add_sync(0xffffffffu, sum);
    float y = fmaf(__fmul_rn((float)sum, sw), st, bias);      // (the other kernels' arithmetic)
    if (p.residual != nullptr) y += r;
    if (lane == 0) static_cast<T*>(p.out)[n] = lin_out<T>(y);
  }
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

template <typename T, int C> static int launch_linear_as(const CUtensorMap& map_w, const CUtensorMap& map_x, const LinearArgs& p, int ctas,
                                                         bool pair, int deep, cudaStream_t s) {
  const bool small = !pair && p.shared == LinSharedSmall;
  const auto kernel = pair ? linear_pair_kernel<T, C> : small ? linear_kernel<T, C, true, 1>
                      : deep == 1 ? linear_kernel<T, C, false, 1> : linear_kernel<T, C, false, 2>;
  static TriPerDevice configured[4];
  TriPerDevice& known = configured[pair ? 0 : small ? 1 : 1 + deep];
  const int device = known.pending();
  TRI_CHECK(device != -2, "int8_linear: no current CUDA device");
  if (device >= 0) {
    TRI_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, small ? LinSharedSmall : LinShared), "int8_linear");
    known.mark(device);
  }
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pair ? 2u : (unsigned)p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(lin_threads(small ? LinSmallWarps : LinWarps)); cfg.dynamicSmemBytes = (size_t)p.shared; cfg.stream = s;
  cfg.attrs = attr; cfg.numAttrs = attr[1].val.clusterDim.x > 1 ? 2 : 1;
  TRI_CUDA(cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p), "int8_linear");
  return tri_launch_status("int8_linear");
}
template <typename T> static int launch_linear(const CUtensorMap& map_w, const CUtensorMap& map_x, const LinearArgs& p, int ctas,
                                               int channels, bool pair, int deep, cudaStream_t s) {
  constexpr int Widest = 16 / (int)sizeof(T);
  if (channels == Widest) return launch_linear_as<T, Widest>(map_w, map_x, p, ctas, pair, deep, s);
  if (channels == 2) return launch_linear_as<T, 2>(map_w, map_x, p, ctas, pair, deep, s);
  return launch_linear_as<T, 1>(map_w, map_x, p, ctas, pair, deep, s);
}

template <typename T> static int launch_row(const void* codes, const void* weight, int64_t weight_stride, const LinearArgs& p, int sms, cudaStream_t s) {
  const bool deep = p.outputs <= LinRowDeep * sms;
  const int ctas = (p.outputs + LinRowWarps - 1) / LinRowWarps, most = sms * (48 / LinRowWarps);
  TRI_CUDA(launch_chained(deep ? linear_row_kernel<T, true> : linear_row_kernel<T, false>, dim3((unsigned)(ctas < most ? ctas : most)),
                          dim3(32 * LinRowWarps), 0, s, static_cast<const int8_t*>(codes), static_cast<const int8_t*>(weight), weight_stride, p),
           "int8_linear");
  return tri_launch_status("int8_linear");
}

// ---- which tile, how many CTAs per tile --------------------------------------------------------------------------------
struct LinearPlan {
  int token_tile, splits;
  bool pair;
};
struct LinearDevice {                  // of one GPU, asked for once
  int sms;
  int clusters[2][9];                  // clusters of n CTAs that are resident at once, by shared memory (0: LinShared, 1: LinSharedSmall)
};

// Estimated time (us) of a plan, less what every plan takes.  The constants are a fit to measured times of 346 shapes (1 to 16384
// tokens, 96 to 32768 channels, widths 96 to 16384) under every tile and split: the plan that the estimate picks takes 1 % more
// than the best one on average, 16 % at worst.  A step of 128 bytes of width costs what the issuing threads need for it (0.3 us)
// or what the SM's port to L2 does (0.1 MB/us); tiles run in rounds of as many as are resident, each no shorter than its epilogue;
// a split adds a cluster barrier and the exchange of the partial sums; and part of it overlaps with the traffic to HBM.
static float plan_time(const LinearPlan& plan, int64_t tokens, int outputs, int width, const LinearDevice& d) {
  const int steps = (width + LinDepth - 1) / LinDepth, bt = plan.token_tile;
  const int channels = plan.pair ? 2 * LinChannels : LinChannels;
  const int64_t tiles = (tokens + bt - 1) / bt * (int64_t)((outputs + channels - 1) / channels);
  float t;
  if (plan.pair) {
    const float rounds = (float)((tiles + d.sms / 2 - 1) / (d.sms / 2)), epilogue = 0.0054f + 0.009f * bt;
    const float step = fmaxf(0.279f, (LinWeightBytes + bt / 2 * LinDepth) * (1.f / 98080.f));
    t = rounds * fmaxf(step * steps, epilogue) + epilogue;
  } else {
    const bool small = bt <= LinSmallTile;
    const int64_t ctas = tiles * plan.splits, slots = (int64_t)d.clusters[small][plan.splits] * plan.splits;
    const float rounds = (float)((ctas + slots - 1) / slots), live = (float)(tokens < bt ? tokens : bt);
    float step = fmaxf(!small && bt <= 128 ? 0.297f : 0.31f, (LinWeightBytes + bt * LinDepth) * (1.f / 98080.f));
    if (small && ctas > d.sms) step *= 1.96f;                // two CTAs per SM share its port and its tensor core
    const float mine = (float)((steps + plan.splits - 1) / plan.splits) * step, epilogue = 0.091f + 0.0017f * live;
    if (plan.splits > 1) t = rounds * (mine + 2.19f + 0.0061f * live);
    else t = rounds * fmaxf(mine, epilogue) + epilogue;
  }
  const float memory = (((float)outputs + (float)tokens) * (float)width + 2.f * (float)outputs * (float)tokens) * (1.f / 6.2e6f);
  return fmaxf(t, memory) + 0.58f * fminf(t, memory);
}

// The current GPU's figures; null after an error.
static const LinearDevice* linear_device() {
  static LinearDevice devices[TriPerDevice::MaxDevices];
  static TriPerDevice known;
  static std::mutex guard;
  const int pending = known.pending();
  int device = -1;
  if (pending == -2 || cudaGetDevice(&device) != cudaSuccess) { tri_set_error("int8_linear: no current CUDA device"); return nullptr; }
  if (pending >= 0) {
    std::lock_guard<std::mutex> lock(guard);
    if (known.pending() < 0) return &devices[device];         // another thread was first
    LinearDevice d{};
    cudaError_t e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device);
    const auto large_tiles = linear_kernel<__nv_bfloat16, 8, false, 2>, small_tiles = linear_kernel<__nv_bfloat16, 8, true, 1>;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(large_tiles, cudaFuncAttributeMaxDynamicSharedMemorySize, LinShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(small_tiles, cudaFuncAttributeMaxDynamicSharedMemorySize, LinSharedSmall);
    for (int small = 0; small < 2; ++small)
      for (int n = 1; n <= 8 && e == cudaSuccess; ++n) {
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = (unsigned)n; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(n * 64)); cfg.blockDim = dim3(lin_threads(small ? LinSmallWarps : LinWarps)); cfg.dynamicSmemBytes = small ? LinSharedSmall : LinShared;
        cfg.attrs = &attr; cfg.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&d.clusters[small][n], small ? small_tiles : large_tiles, &cfg);
        if (e == cudaSuccess && d.clusters[small][n] < 1) d.clusters[small][n] = 1;
      }
    if (e != cudaSuccess) { tri_set_error(cudaGetErrorString(e)); return nullptr; }
    devices[device] = d;
    known.mark(device);
  }
  return &devices[device];
}

static LinearPlan choose_plan(int64_t tokens, int outputs, int width, const LinearDevice& d) {
  const int steps = (width + LinDepth - 1) / LinDepth;
  LinearPlan best{16, 1, false};
  float best_time = 1e30f;
  int tried = 0;
  const auto consider = [&](int64_t bt) {                     // a token tile, in steps of 16 (a pair's: 32)
    bt = bt < 16 ? 16 : bt > 256 ? 256 : (bt + 15) / 16 * 16;
    const int bit = 1 << (bt / 16 - 1);
    if (tried & bit) return;
    tried |= bit;
    const int64_t tiles = (tokens + bt - 1) / bt * (int64_t)((outputs + LinChannels - 1) / LinChannels);
    for (int splits = 1; splits <= 8 && splits <= steps && (splits == 1 || tiles * splits <= 2 * (int64_t)d.sms); ++splits) {
      const LinearPlan plan{(int)bt, splits, false};
      const float time = plan_time(plan, tokens, outputs, width, d);
      if (time < best_time) { best_time = time; best = plan; }
    }
    if (bt >= 128 && bt % 32 == 0) {
      const LinearPlan plan{(int)bt, 1, true};
      const float time = plan_time(plan, tokens, outputs, width, d);
      if (time < best_time) { best_time = time; best = plan; }
    }
  };
  const int64_t least = (tokens + 255) / 256;                 // token tiles at their largest; then evenly cut into a few more
  for (int64_t more = 0; more < 4; ++more) consider((tokens + least + more - 1) / (least + more));
  for (int bt : {256, 192, 128, 96, 64, 32}) if (bt < tokens + 16) consider(bt);
  return best;
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
  const LinearDevice* gpu = linear_device();
  if (gpu == nullptr) return TRI_ERR_CUDA;
  LinearArgs p{};
  p.residual_stride = residual_stride; p.out_stride = out_stride; p.scales = scales; p.weight_scales = weight_scales;
  p.bias = bias; p.residual = residual; p.out = out; p.tokens = (int)tokens; p.outputs = outputs; p.width = width; p.error = device_error;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tokens == 1) {
    if (type == TRI_BF16) return launch_row<__nv_bfloat16>(codes, weight, weight_stride, p, gpu->sms, s);
    if (type == TRI_FP16) return launch_row<__half>(codes, weight, weight_stride, p, gpu->sms, s);
    return launch_row<float>(codes, weight, weight_stride, p, gpu->sms, s);
  }
  const LinearPlan plan = choose_plan(tokens, outputs, width, *gpu);
  p.token_tile = plan.token_tile; p.splits = plan.splits;
  const auto rows_allow = [&](int channels) {                // accesses of so many channels to the rows of output and residual
    const int64_t bytes = channels * (int64_t)cell;
    return reinterpret_cast<uintptr_t>(out) % bytes == 0 && reinterpret_cast<uintptr_t>(residual) % bytes == 0 && out_stride % channels == 0 &&
           (residual == nullptr || residual_stride % channels == 0);
  };
  const int each = rows_allow(16 / (int)cell) ? 16 / (int)cell : rows_allow(2) ? 2 : 1;
  const int channels = plan.pair ? 2 * LinChannels : LinChannels, box = plan.pair ? p.token_tile / 2 : p.token_tile;
  p.channel_tiles = (outputs + channels - 1) / channels;
  const int64_t tiles = (tokens + p.token_tile - 1) / p.token_tile * (int64_t)p.channel_tiles;
  TRI_CHECK(tiles <= 0x7fffffff / 8, "int8_linear: tokens * outputs");
  p.tiles = (int)tiles;
  p.group = 8;
  // Where a CTA's share of the weights is short, its first stages start on their way into L2 while the kernel that makes the
  // tokens' codes still runs (L2 only, so whatever that kernel writes is what is read afterwards).
  // quantize_rows and product, DRAM-cold weights: 1 x 4096 -> 4096 9.3 us, 8.5 like this; 64 tokens 12.0, 11.3.  With longer
  // shares it is no gain (16 x 14336 -> 4096 17.4, 18.2).
  const int share = ((width + LinDepth - 1) / LinDepth + plan.splits - 1) / plan.splits;
  p.ahead = !plan.pair && tokens <= p.token_tile && share <= 8 ? (share < 5 ? share : 5) : 0;
  p.shared = !plan.pair && p.token_tile <= LinSmallTile ? LinSharedSmall : LinShared;
  // Two steps per stage where three stages of them fit: the issuing threads' work per stage is 0.1 us dearer than the MMAs of a
  // narrow tile (128 steps of 16 tokens: 38 us, 29 with two per stage; 16384 x 14336 -> 4096 in pairs: 649 us, 602).
  const int step_bytes = LinWeightBytes + box * LinDepth;
  const int deep = plan.pair || (p.shared == LinShared && (p.shared - 1024) / (2 * step_bytes) >= 3) ? 2 : 1;
  p.stages = (p.shared - 1024) / (deep * step_bytes);
  if (p.stages > LinMaxStages) p.stages = LinMaxStages;
  p.columns = 32;
  while (p.columns < 2 * p.token_tile) p.columns *= 2;
  const int resident = plan.pair ? gpu->sms / 2 : p.shared == LinShared ? gpu->sms : 2 * gpu->sms;
  const int ctas = plan.pair ? 2 * (p.tiles < resident ? p.tiles : resident)
                             : p.splits > 1 ? p.tiles * p.splits : (p.tiles < resident ? p.tiles : resident);
  CUtensorMap map_w, map_x;
  if (make_code_map(&map_w, weight, outputs, width, weight_stride, LinChannels) != TRI_OK) return TRI_ERR_CUDA;
  if (make_code_map(&map_x, codes, tokens, width, codes_stride, (unsigned)box) != TRI_OK) return TRI_ERR_CUDA;
  if (type == TRI_BF16) return launch_linear<__nv_bfloat16>(map_w, map_x, p, ctas, each, plan.pair, deep, s);
  if (type == TRI_FP16) return launch_linear<__half>(map_w, map_x, p, ctas, each, plan.pair, deep, s);
  return launch_linear<float>(map_w, map_x, p, ctas, each, plan.pair, deep, s);
}
