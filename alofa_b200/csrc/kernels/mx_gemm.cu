// Product of rows in 8 bits and a weight in 4 (mx.cuh) on the 5th-generation tensor cores:
//   y[t, f] = sum_b 2^(sx[t, b] + sw[f, b] - 254) sum_{k in block b} x[t, k] w[f, k]
// and out = y (+ bias[f]) (+ add[t, f]) in bf16 or fp32, or, for a gated weight, rows in 8 bits of
// silu(y of the gate) * (y of the up projection)  (src/alofa/kernels/cpu/scalar.mojo:132-231).
// One tcgen05.mma.kind::mxf8f6f4.block_scale takes one block of 32 numbers of its rows; the scales are its
// operands too, in tensor memory, so sums are of the numbers themselves and in fp32.  The tensor cores' additions cut off towards zero
// where scalar ones round; sums go in runs so that this stays small (RUN_SLICES).  At depth 3,584 with scales over a range of 2^14, 1,999 x
// 18,944 gated numbers are then 0.6e-4 to 1.3e-4 of the rows' norm off, and from sums of scalar additions 0.5e-4 to 1.1e-4: some hundred of
// 37.9 million that fall on the other side of a tie of two codes (one rounding to 8 bits is up to 2^-4).
//
// A k-slice is 128 numbers: four blocks.  A weight's tile of a slice is 8,704 contiguous bytes of memory
// (8,192 of codes, 512 of scales), fetched by one thread with two copies: TMA, which unpacks 4-bit numbers on
// the way (shared memory holds them as 16 in 8 bytes and 8 bytes of room, rows of 128 bytes with 128-byte
// swizzle), and a plain bulk copy.  Spreading them with cp.async, 8 bytes at a time, was bound by the copies'
// instructions: 7B's gate and up projections, one token, 21.9 us and 2,048 tokens 419 us.  Tokens come by TMA,
// their scales 4 bytes a row.  The weights depend on no earlier kernel of the stream: the first ring of them is
// asked for before the dependency wait.
//
// Two kernels: mx_few_kernel, the weight's rows on the M side, for a few tokens or few tiles, whose time is
// the weight's bytes or a launch's latency; mx_pair_kernel, the tokens on the M side and a pair of CTAs to a
// tile, for prompts, whose time is the tensor cores'.
//
// Every wait on an mbarrier is bounded: after the limit the CTA raises the status word, lets its copies
// and products end, frees its tensor memory and returns; what it should have written is NaN.
#include "mx.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

#include <string.h>

#include <atomic>

struct MxArgs {
  const uint8_t* tiles;     // the weight: [ceil(N / 128), slices, MX_TILE_BYTES]
  const uint8_t* x_scales;  // [T, 4 * slices]
  void* out;                // [T, N] bf16 or fp32; gated: codes [T, padded(F)]
  uint8_t* out_scales;      // gated: [T, padded(F) / 32]
  const float* bias;        // [N] or null
  const float* add;         // [T, N] or null
  int T, N, slices;         // tokens, rows of the weight, k-slices
  int F;                    // gated: features
  int out_bf16, wide;       // wide: four numbers of a row are stored (and bias and add read) at once
  float gate_alpha, gate_limit;
  int* status;
};

__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
// The barrier counts one arrival of this thread when all its copies so far have landed.
__device__ __forceinline__ void arrive_when_landed(uint64_t* bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void fence_to_tensor_core() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y) : "memory");
}
// The same by either CTA of a pair; bar: the first CTA's barrier.  (A weight's tile is 136 rows of 64 bytes, 128 of codes and eight of
// scales; of codes the barrier counts the 8,192 bytes that they have in memory, not the 16,384 that they fill.)
__device__ __forceinline__ void load_tile_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void load_bytes(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// The warps that copy and issue run their loops whole, every lane through the same waits and counters, and only the
// instructions themselves are one lane's: what those take (addresses, descriptors, barriers) then stands in uniform
// registers.  With the whole loop inside `if (lane == 0)` each tcgen05 instruction took 65 to 100 clocks to issue, and a
// slice of the pair kernel 1,060 where its products take 512.
__device__ __forceinline__ bool elect_lane() {
  uint32_t chosen;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(chosen));
  return chosen != 0;
}
__device__ __forceinline__ bool all_lanes(bool v) { return __all_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }  // a value that every lane has

// After a wait that ran out: what is still in flight ends in a bounded time.
constexpr uint32_t DRAIN_LIMIT = 1u << 14;
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity, uint32_t limit = DRAIN_LIMIT) {
  for (uint32_t w = 0; w < limit && !mbar_try_wait(bar, parity); ++w) {
  }
}
// `count` arrivals at once, in the place of those who gave up before they made theirs.
__device__ __forceinline__ void arrive_for(uint64_t* bar, uint32_t count) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory"); }

// Shared memory seen as rows of 16 bytes, groups of 8 rows 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t scales_desc(uint32_t smem) { return (uint64_t)((smem & 0x3FFFFu) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46); }
// 512 bytes of scales (32 rows of 16) to four columns of tensor memory, the same in all four quarters of its lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(scales_desc(smem)) : "memory");
}
__device__ __forceinline__ void umma_mx(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
      : "memory");
}
// The same for a pair of CTAs: each CTA's own shared memory to its own tensor memory.
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t tmem, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(scales_desc(smem)) : "memory");
}
__device__ __forceinline__ void umma_mx_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
      : "memory");
}
// The tensor cores' additions cut off towards zero some bits below the accumulator's last one, which takes 3.9e-9 off every sum for
// each slice that went into it: 1.1e-7 over 28 slices, 7.7e-7 over 148.  The depth therefore goes in runs of slices, each with an accumulator
// of its own, added up by additions that round.  With 14 slices a run 1,999 x 37,888 sums of depth 3,584 are 0.9e-7 of their norm
// off, with 28 1.55e-7, and 0.7e-7 by scalar additions; of depth 18,944 (2.0e-7 with 37, 9.4e-7 with 148) 1.8e-7.
// Runs cost next to nothing for a few tokens, whose accumulators are small enough to stand beside one another.  For prompts each
// takes the accumulator from the products for 1,100 clocks: gate and up of 7B, 1,999 tokens, 227 us in one run and 237 in two.  What is
// stored takes twice the slices a run there, as its rounding to bfloat16 is 10^4 times as much, and fp32 sums of any depth are within 2e-7:
// q, k and v of 7B, 2,048 tokens, 33.5 us in one run and 35.6 in two.
constexpr int RUN_SLICES = 16, RUN_SLICES_STORED = 32;
constexpr uint32_t E4M3 = 0, E2M1 = 5;
// The instruction: types of A and B, scales E8M0, M and N, the scales' byte `block` of their column.
constexpr uint32_t mx_idesc(uint32_t a, uint32_t b, int m, int n, int block) {
  return (a << 7) | (b << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)block << 29) | ((uint32_t)block << 4);
}

// An arrival on another CTA's barrier that says only that this warp's reads of tensor memory are over (they are complete, and
// tcgen05.fence::before_thread_sync stands between): nothing of ordinary memory goes with it.  As a release for the cluster it
// took 1,200 to 1,500 clocks, and the next tile's products wait for it.
__device__ __forceinline__ void tell_in_cluster(uint32_t bar_in_cluster) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_in_cluster) : "memory");
}
__device__ __forceinline__ uint32_t cta_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {  // every thread of every CTA of the cluster
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Its two halves: every warp once each.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ---------------------------------------------------------------------------
// A few tokens.  A CTA has 128 of the weight's rows, BN tokens and a part of the depth; the CTAs of a tile's
// parts are a cluster.  Each leaves its sums in its shared memory as [token][row]; the cluster's CTAs share
// out the tokens, add the parts in order out of one another's shared memory and write whole rows: no sums go
// through memory, nothing is launched to add them, and the last step is spread over as many SMs as the first.
//
// In a graph, weights from memory: 0.5B's q, k and v 3.2 us for one token; 7B's 5.5 for one and 8.8 for 128; 7B's
// down projection for eight 10.6 (its 36 MB take 5.6), gate and up for one 13.9 (72 MB, 11.0).  Small products are a
// launch, a cluster's start and two trips to memory one after the other; large ones two CTAs an SM whose rings hold 200 KB.
// ---------------------------------------------------------------------------
constexpr int FEW_THREADS = 192;  // warp 0 weights, 4 tokens, 5 products; then warps 0-3 read the sums and all write rows
constexpr int FEW_PARTS = 8;      // of a depth, at most: a portable cluster
constexpr int SUM_PITCH = MX_TILE_ROWS + 4;

template <int BN>
struct FewTile {
  static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : 3;  // two CTAs an SM
  static constexpr uint32_t A_BYTES = MX_TILE_ROWS * MX_GROUP, B_BYTES = BN * MX_GROUP;
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES + 1024;  // tiles, 512 bytes of the weight's scales, 512 of the tokens'
  static constexpr uint32_t SMEM = STAGES * STAGE_BYTES + 1024;
  static constexpr int SCALE_COLS = STAGES * 8;  // the scales have as many places as the ring has stages: those of a slice are written when the products of the slice before them there are complete
  static constexpr int MOST_RUNS = (256 - SCALE_COLS) / BN;  // two CTAs an SM: 256 columns each at most
  static_assert(BN * SUM_PITCH * 4 <= STAGES * STAGE_BYTES, "the sums take the ring's room");
};

// Four neighbouring rows' sums of one token, as a gated weight has them (16 rows of the gate, the same 16 of the up
// projection): the warp's 64 features as codes and two scales.  f0: the first of the tile's features.
template <bool CLAMPED>
__device__ __forceinline__ void few_gated_token(const MxArgs& args, float4 v, int t, int f0, int lane) {
  const int f = f0 + (lane >> 3) * 16 + (lane & 3) * 4;  // lanes with bit 2 clear have the gate's rows, those with it set the up projection's
  float g[4] = {v.x, v.y, v.z, v.w}, u[4];
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = __shfl_xor_sync(0xffffffffu, g[j], 4);
  // told apart once for the four: for every number it took 64 tokens of 8,960 features 12.2 us instead of 11.1
  if (__builtin_expect(!mx_gate_far<CLAMPED>(fminf(fminf(g[0], g[1]), fminf(g[2], g[3])), args.gate_alpha), 1)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = mx_gate_times<CLAMPED, false>(g[j], u[j], args.gate_alpha, args.gate_limit);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = mx_gate_times<CLAMPED, true>(g[j], u[j], args.gate_alpha, args.gate_limit);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = f + j < args.F ? g[j] : 0.f;
  if ((lane & 4) == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j) largest = max(largest, mx_size(g[j]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));  // a block: half the warp
  const uint32_t s = mx_row_scale(largest);
  const float over = mx_over(s);
  const int fp = (args.F + MX_GROUP - 1) / MX_GROUP * MX_GROUP;
  uint8_t* codes = reinterpret_cast<uint8_t*>(args.out) + (size_t)t * fp;
  uint8_t* scales = args.out_scales + (size_t)t * (fp / MX_BLOCK);
  if ((lane & 4) == 0) *reinterpret_cast<uint32_t*>(codes + f) = s == 255u ? 0u : mx_e4m3(g[0] * over, g[1] * over, g[2] * over, g[3] * over);
  if ((lane & 15) == 0) scales[f / MX_BLOCK] = (uint8_t)s;
  if (f0 + 64 < fp && f0 + 64 >= (args.N + 1) / 2) {  // the last tile fills half a group: the other half is zeros
    if (lane < 16) *reinterpret_cast<uint32_t*>(codes + f0 + 64 + lane * 4) = 0u;
    if (lane < 2) scales[(f0 + 64) / MX_BLOCK + lane] = 0;
  }
}

// The same four rows of a product that is stored.
__device__ __forceinline__ void few_stored_token(const MxArgs& args, float4 v, int t, int f) {
  const size_t at = (size_t)t * args.N + f;
  if (args.wide && f + 4 <= args.N) {
    if (args.bias) {
      const float4 b = *reinterpret_cast<const float4*>(args.bias + f);
      v.x += b.x, v.y += b.y, v.z += b.z, v.w += b.w;
    }
    if (args.add) {
      const float4 a = *reinterpret_cast<const float4*>(args.add + at);
      v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
    }
    if (args.out_bf16) {
      __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
      *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(args.out) + at) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
    } else {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(args.out) + at) = v;
    }
    return;
  }
  const float y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (f + j >= args.N) break;
    float z = y[j] + (args.bias ? args.bias[f + j] : 0.f);
    if (args.add) z += args.add[at + j];
    if (args.out_bf16) reinterpret_cast<bf16*>(args.out)[at + j] = __float2bfloat16_rn(z);
    else reinterpret_cast<float*>(args.out)[at + j] = z;
  }
}

template <int BN>
__global__ void __launch_bounds__(FEW_THREADS, 2) mx_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const MxArgs args, const int parts) {
  using Tile = FewTile<BN>;
  constexpr int STAGES = Tile::STAGES;
  constexpr uint32_t BY_WEIGHTS = 1, BY_TOKENS = 1 + 32;  // arrivals a slice: the weight's bytes; the tokens', and the copies of their scales
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  // asked_all: both copying warps have said in `asked` how many slices they asked for; quiet: no copy writes the ring any more
  __shared__ uint64_t landed[STAGES], stage_free[STAGES], sums_done, asked_all, quiet;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag, asked[2];

  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int f_tile = blockIdx.x / (unsigned)parts, part = blockIdx.x - f_tile * parts;  // a cluster: the parts of one tile's depth
  const int f0 = f_tile * MX_TILE_ROWS, t0 = blockIdx.y * BN;
  // parts that differ by one slice at most
  const int first = (unsigned)(args.slices * part) / (unsigned)parts, n = (unsigned)(args.slices * (part + 1)) / (unsigned)parts - first;  // at most 2^23 slices in 8 parts
  const int runs = min((n + RUN_SLICES - 1) / RUN_SLICES, Tile::MOST_RUNS);  // of slices, each with sums of its own
  const uint32_t need = (uint32_t)(runs * BN + Tile::SCALE_COLS), tmem_cols = need <= 64 ? 64 : need <= 128 ? 128 : 256;
  if (threadIdx.x == 0) {
    abort_flag = asked[0] = asked[1] = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&landed[s], BY_WEIGHTS + BY_TOKENS);
      mbar_init(&stage_free[s], 1);
    }
    mbar_init(&sums_done, 1);
    mbar_init(&asked_all, 2);
    mbar_init(&quiet, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc(&tmem_base_smem, tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_smem;

  if (warp == 0) {
    const bool chosen = elect_lane();
    int i = 0, s = 0;
    uint32_t round = 1;  // parity of the phase in which this stage was last freed; the first round waits for nothing
    bool free = true;
    for (; i < n; ++i) {
      if (!all_lanes(free) && !all_lanes(mbar_wait(&stage_free[s], round, &abort_flag))) break;
      const uint32_t stage = tiles + s * Tile::STAGE_BYTES;
      const int tile = f_tile * args.slices + first + i;
      uint64_t* bar = &landed[s];
      s = s + 1 == STAGES ? 0 : s + 1;
      round ^= s == 0 ? 1u : 0u;
      free = i + 1 < STAGES || mbar_complete(&stage_free[s], round);
      if (chosen) {
        mbar_expect_tx(bar, MX_TILE_BYTES);
        load_tile(stage, &map_w, bar, 0, tile * MX_TILE_MAP_ROWS);
        load_bytes(stage + Tile::A_BYTES + Tile::B_BYTES, args.tiles + (size_t)tile * MX_TILE_BYTES + MX_TILE_CODES, MX_TILE_BYTES - MX_TILE_CODES, bar);
      }
    }
    if (lane == 0) asked[0] = i, mbar_arrive(&asked_all);
  } else if (warp == 4) {
    pdl_wait();
    pdl_launch();
    const bool chosen = elect_lane();
    const int row_bytes = 4 * args.slices;
    int i = 0, s = 0;
    uint32_t round = 1;
    bool free = true;
    for (; i < n; ++i) {
      if (!all_lanes(free) && !all_lanes(mbar_wait(&stage_free[s], round, &abort_flag))) break;
      const uint32_t stage = tiles + s * Tile::STAGE_BYTES, scales = stage + Tile::A_BYTES + Tile::B_BYTES + 512;
      uint64_t* bar = &landed[s];
      s = s + 1 == STAGES ? 0 : s + 1;
      round ^= s == 0 ? 1u : 0u;
      free = i + 1 < STAGES || mbar_complete(&stage_free[s], round);
      if (chosen) {
        mbar_expect_tx(bar, Tile::B_BYTES);
        load_tile(stage + Tile::A_BYTES, &map_x, bar, (first + i) * MX_GROUP, t0);
      }
#pragma unroll
      for (int r = 0; r < BN; r += 32) {
        const int t = r + lane;
        if (t < BN && t0 + t < args.T) copy4(scales + (uint32_t)mx_scale_at(t, 0), args.x_scales + (size_t)(t0 + t) * row_bytes + 4 * (first + i));
      }
      arrive_when_landed(bar);
    }
    if (lane == 0) asked[1] = i, mbar_arrive(&asked_all);
  } else if (warp == 5) {
    const bool chosen = elect_lane();
    const uint32_t place = uniform(tmem) + (uint32_t)(runs * BN);
    uint32_t sums = uniform(tmem), add = 0;  // a run's first products begin its sums
    const int run_slices = runs > 1 ? (unsigned)n / (unsigned)runs : n, longer = n - runs * run_slices;  // the first `longer` runs have one slice more
    int s = 0, run = 0, left = run_slices + (longer > 0 ? 1 : 0);
    uint32_t round = 0;
    bool ok = true, ready = false;
    for (int i = 0; i < n; ++i) {
      if (!all_lanes(ready)) ok = all_lanes(mbar_wait(&landed[s], round, &abort_flag));
      if (!ok) break;
      const uint32_t stage = tiles + s * Tile::STAGE_BYTES, scales = stage + Tile::A_BYTES + Tile::B_BYTES;
      const uint32_t scale_a = place + s * 8, scale_b = scale_a + 4;
      uint64_t* freed = &stage_free[s];
      s = s + 1 == STAGES ? 0 : s + 1;
      round ^= s == 0 ? 1u : 0u;
      fence_to_tensor_core();
      tc_fence_after();
      ready = i + 1 < n && mbar_complete(&landed[s], round);
      const uint64_t a = smem_desc_sw128(stage), b = smem_desc_sw128(stage + Tile::A_BYTES);
      if (chosen) {
        scales_to_tmem(scale_a, scales);
        scales_to_tmem(scale_b, scales + 512);
#pragma unroll
        for (int j = 0; j < 4; ++j) umma_mx(sums, a + 2 * j, b + 2 * j, mx_idesc(E2M1, E4M3, 128, BN, j), scale_a, scale_b, j ? 1u : add);
        umma_commit(freed);
      }
      add = 1;
      if (--left == 0) ++run, left = run_slices + (run < longer ? 1 : 0), sums += BN, add = 0;
    }
    if (chosen) {
      umma_commit(&sums_done);
      if (__builtin_expect(!ok, 0)) {
        drain(&sums_done, 0);  // the products issued so far end before tensor memory is given back
        // and the copies asked for land before the sums take the ring's room, or another CTA this one's: the last slice in each
        // stage, where a warp that gave up first did not ask for its part of it without that part
        drain(&asked_all, 0);
        const int w = *(volatile int*)&asked[0], x = *(volatile int*)&asked[1], most = max(w, x);
        for (int j = max(0, most - STAGES); j < most; ++j) {
          if (j >= w) arrive_for(&landed[j % STAGES], BY_WEIGHTS);
          if (j >= x) arrive_for(&landed[j % STAGES], BY_TOKENS);
          drain(&landed[j % STAGES], (uint32_t)(j / STAGES) & 1u);
        }
      }
      mbar_arrive(&quiet);
    }
  }
  if (warp == 4) copies_wait();  // landed long ago, unless a wait ran out
  __syncwarp();

  const int live = min(BN, args.T - t0);
  if (warp < 4) {
    const bool good = mbar_wait(&sums_done, 0, &abort_flag) && !*(volatile int*)&abort_flag;
    tc_fence_after();
    if (__builtin_expect(!good, 0)) drain(&quiet, 0, (STAGES + 3) * DRAIN_LIMIT);  // longer than what arrives there may take
    if (!good && threadIdx.x == 0 && args.status) atomicExch(args.status, 2);
    const uint32_t mine = tiles + (uint32_t)(warp * 32 + lane) * 4;
    for (int c = 0; c < live; c += 16) {
      uint32_t r[16];
      tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, r);
      tmem_ld_wait();
      for (int z = 1; z < runs; ++z) {
        uint32_t q[16];
        tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + z * BN + c, q);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(q[j]));
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + (uint32_t)((c + j) * SUM_PITCH * 4)), "f"(good ? __uint_as_float(r[j]) : __uint_as_float(0x7fc00000u)) : "memory");
    }
  }
  tc_fence_before();
  __syncwarp();
  if (parts > 1) cluster_sync_all();
  else __syncthreads();
  pdl_wait();  // what is written now, an earlier kernel may have been reading
  // Nobody leaves while its sums are read.  A warp with one token at most says that it has read them before it stores what comes
  // of them: the arrival need not wait for the stores, 0.1 to 0.3 us of 3 to 6 with tiles of 16 tokens (of 32, none).  With more
  // tokens it waits for the first ones' in either place, and later is better (32 in four parts 4.3 us, and 4.8 so).
  const int step = parts * (FEW_THREADS / 32);
  const bool early = BN == 16 && parts > 1 && live <= step;
  if (early && part + parts * warp >= live) cluster_arrive();
  for (int t = part + parts * warp; t < live; t += step) {
    const uint32_t local = tiles + (uint32_t)(t * SUM_PITCH + lane * 4) * 4;
    float4 v[FEW_PARTS];
#pragma unroll
    for (int z = 0; z < FEW_PARTS; ++z) {
      v[z] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (z < parts) {
        if (parts > 1) {
          uint32_t there;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(local), "r"(z));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[z].x), "=f"(v[z].y), "=f"(v[z].z), "=f"(v[z].w) : "r"(there) : "memory");
        } else {
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[z].x), "=f"(v[z].y), "=f"(v[z].z), "=f"(v[z].w) : "r"(local) : "memory");
        }
      }
    }
#pragma unroll
    for (int z = 1; z < FEW_PARTS; ++z)
      if (z < parts) v[0].x += v[z].x, v[0].y += v[z].y, v[0].z += v[z].z, v[0].w += v[z].w;
    if (early) cluster_arrive();
    if (!args.F) few_stored_token(args, v[0], t0 + t, f0 + lane * 4);
    else if (args.gate_alpha == 0.f) few_gated_token<false>(args, v[0], t0 + t, f_tile * (MX_TILE_ROWS / 2), lane);
    else few_gated_token<true>(args, v[0], t0 + t, f_tile * (MX_TILE_ROWS / 2), lane);
  }
  if (parts > 1 && !early) cluster_arrive();
  if (parts > 1) cluster_wait();
  else __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// ---------------------------------------------------------------------------
// Prompts.  A pair of CTAs (a cluster of two, one CTA an SM) works through tiles of 256 tokens and 256 rows of
// the weight with products of M = 256 that the first CTA issues for both: each CTA fetches its own 128 tokens and
// its own 128 rows, 25 KB a k-slice for 512 clocks of the tensor cores, about what an SM can pull out of L2.  The
// scales of all 256 rows stand in both CTAs' tensor memory, those of its own tokens in each.
//
// Tensor memory holds 512 columns: two accumulators of 256 and the scales do not fit.  The accumulators therefore
// share 64 columns (0-255 and 192-447), and the epilogue takes those first: the next tile's products begin when it has
// them in registers, and run beside the rest of the epilogue.  Scales have five places in turn: those of a slice are
// written when the products of the slice before it there are complete.
//
// A slice's way round the ring (its room freed, its copies asked for, landed, its products issued, complete) takes
// several times as long as its products, so nothing may stand on it that need not: the copies of both CTAs count on
// the first one's barrier, and the tokens' scales, which no copy of the tensor kind can fetch (rows of 4 bytes a slice),
// come eight slices at a time, ahead of the ring, by loads of a warp of their own.
//
// In a graph, 7B's gate and up projections, 2,048 tokens 249 us: 2.2 PFLOP/s, the tensor cores busy 65 to 69 % of the time at a clock
// that the power cap holds to 1.6 to 1.8 GHz; q, k and v 30.2 us (144 tiles on 74 pairs, two rounds, each with a beginning and an end;
// 46 to 51 % busy), the down projection 122 (112 tiles: half of the pairs idle in the second round).  A slice takes 560 to 590 clocks, 800 while
// the epilogue of the tile before it runs.
// ---------------------------------------------------------------------------
constexpr int PAIR_THREADS = 384;  // warp 0 weights, 1 tokens, 2 products (first CTA), 3 the tokens' scales, 4-11 epilogue
constexpr int PAIR_STAGES = 6;
constexpr uint32_t PAIR_STAGE_BYTES = 2 * 128 * MX_GROUP + 1024;  // tokens, weight rows, the scales of 256 weight rows
constexpr int PAIR_CHUNK = 8;  // slices whose token scales are fetched together: 512 bytes each, two chunks' room
constexpr int TURN_PITCH = 17;  // 32 rows of 16 sums, an epilogue warp's room to turn them
constexpr uint32_t PAIR_TURN = PAIR_STAGES * PAIR_STAGE_BYTES + 2 * PAIR_CHUNK * 512;
constexpr uint32_t PAIR_SMEM = PAIR_TURN + 8 * 32 * TURN_PITCH * 4 + 1024;
constexpr uint32_t PAIR_SECOND = 192, PAIR_SCALES = 448;  // columns of the second accumulator, and of the scales
constexpr int PAIR_SCALE_PLACES = 5;  // of 12 columns

__device__ __forceinline__ void pair_load64(uint32_t tmem, uint32_t (&r)[64]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t q[16];
    tmem_ld16(tmem + j * 16, q);
#pragma unroll
    for (int i = 0; i < 16; ++i) r[j * 16 + i] = q[i];
  }
  tmem_ld_wait();
}

// What a run left, on top of the runs before it (`first`: there are none).  `have()` when it is in registers.
template <typename Have>
__device__ __forceinline__ void pair_take64(uint32_t tmem, uint32_t (&r)[64], bool first, Have have) {
  if (first) {
    pair_load64(tmem, r);
    have();
  } else {
    uint32_t a[64];
    pair_load64(tmem, a);
    have();
#pragma unroll
    for (int i = 0; i < 64; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(a[i]));
  }
}

// 64 rows' sums of one token of a gated weight: one block of codes and its scale.  The clamped form, gates far below zero and the
// last features' zeros are told apart once, not for every number: this is what the tensor cores wait for when the depth is short.
template <bool CLAMPED>
__device__ __forceinline__ void pair_gated64(const MxArgs& args, const uint32_t (&r)[64], int t, int row, bool good) {
  const int f = row / 2, fp = (args.F + MX_GROUP - 1) / MX_GROUP * MX_GROUP;
  if (f >= fp) return;
  float v[32], least = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) least = fminf(least, __uint_as_float(r[(j / 16) * 32 + j % 16]));
  if (!mx_gate_far<CLAMPED>(least, args.gate_alpha)) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int at = (j / 16) * 32 + j % 16;
      v[j] = mx_gate_times<CLAMPED, false>(__uint_as_float(r[at]), __uint_as_float(r[at + 16]), args.gate_alpha, args.gate_limit);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int at = (j / 16) * 32 + j % 16;
      v[j] = mx_gate_times<CLAMPED, true>(__uint_as_float(r[at]), __uint_as_float(r[at + 16]), args.gate_alpha, args.gate_limit);
    }
  }
  if (f + 32 > args.F) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = f + j < args.F ? v[j] : 0.f;
  }
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) largest = max(largest, mx_size(v[j]));
  const uint32_t s = good ? mx_row_scale(largest) : 255u;
  const float over = mx_over(s);
  uint32_t c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = mx_e4m3(v[4 * j] * over, v[4 * j + 1] * over, v[4 * j + 2] * over, v[4 * j + 3] * over);
  if (s == 255u) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 0u;
  }
  uint4* codes = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(args.out) + (size_t)t * fp + f);
  codes[0] = make_uint4(c[0], c[1], c[2], c[3]);
  codes[1] = make_uint4(c[4], c[5], c[6], c[7]);
  args.out_scales[(size_t)t * (fp / MX_BLOCK) + f / MX_BLOCK] = (uint8_t)s;
}

// The same sums of a product that is stored.  A lane has a token's 64 sums; they are turned in shared memory 16 at a time, so
// that a warp's stores (and loads of what is added) are of eight tokens' whole 32 or 64 bytes, or, at a width that is no
// multiple of four, of two tokens' numbers one by one: 1,999 x 4,608 of depth 3,584 added to another tensor 50.5 us with every
// lane at its own token and 37.5 so, 4,601 rows 182.4 and 47.5.
__device__ __forceinline__ void pair_stored64(const MxArgs& args, const uint32_t (&r)[64], int t0, int row, bool good, float* turn, int lane) {
  const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int h = 0; h < 64; h += 16) {
    if (row + h >= args.N) return;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) turn[lane * TURN_PITCH + j] = good ? __uint_as_float(r[h + j]) : nan;
    __syncwarp();
    if (args.wide) {
      const int f = row + h + (lane & 3) * 4;  // a width of a multiple of four: all four numbers are there, or none
      float4 b = make_float4(0.f, 0.f, 0.f, 0.f), a[4];
      if (f < args.N && args.bias) b = *reinterpret_cast<const float4*>(args.bias + f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * 8 + (lane >> 2);
        a[i] = f < args.N && t < args.T && args.add ? *reinterpret_cast<const float4*>(args.add + (size_t)t * args.N + f) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = i * 8 + (lane >> 2), t = t0 + q;
        const float* v = turn + q * TURN_PITCH + (lane & 3) * 4;
        const float x = v[0] + b.x + a[i].x, y = v[1] + b.y + a[i].y, z = v[2] + b.z + a[i].z, w = v[3] + b.w + a[i].w;
        if (f >= args.N || t >= args.T) continue;
        const size_t at = (size_t)t * args.N + f;
        if (args.out_bf16) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(x, y), hi = __floats2bfloat162_rn(z, w);
          *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(args.out) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        } else {
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(args.out) + at) = make_float4(x, y, z, w);
        }
      }
    } else {
      const int f = row + h + (lane & 15);
      const float b = f < args.N && args.bias ? args.bias[f] : 0.f;
      if (args.add) {  // into the sums first, so that its loads are in flight together
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
          float a[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int t = t0 + (i + j) * 2 + (lane >> 4);
            a[j] = f < args.N && t < args.T ? args.add[(size_t)t * args.N + f] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) turn[((i + j) * 2 + (lane >> 4)) * TURN_PITCH + (lane & 15)] += a[j];
        }
      }
#pragma unroll 8
      for (int i = 0; i < 16; ++i) {
        const int q = i * 2 + (lane >> 4), t = t0 + q;
        if (f >= args.N || t >= args.T) continue;
        const size_t at = (size_t)t * args.N + f;
        const float z = turn[q * TURN_PITCH + (lane & 15)] + b;
        if (args.out_bf16) reinterpret_cast<bf16*>(args.out)[at] = __float2bfloat16_rn(z);
        else reinterpret_cast<float*>(args.out)[at] = z;
      }
    }
  }
}

// LONG: depths of several runs (RUN_SLICES).  Each has an accumulator to itself, in turns as tiles have where they are one run,
// and the epilogue's warps keep the tile's sums in registers, 128 a thread.  The four other warps hand over what those need: of the
// 168 registers that 384 threads are launched with, 128 threads keep 88 and 256 have 208, which is all of them.
template <bool LONG>
__global__ void __launch_bounds__(PAIR_THREADS, 1) mx_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s, const __grid_constant__ CUtensorMap map_x, const MxArgs args) {
  constexpr int STAGES = PAIR_STAGES;
  constexpr uint32_t A_BYTES = 128 * MX_GROUP, B_BYTES = 128 * MX_GROUP;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  // landed (first CTA): the copies of a slice, those of both CTAs; scales_in (first CTA), chunk_free: a chunk of the tokens' scales; sums_ready, sums_taken: a tile's accumulator
  __shared__ uint64_t landed[STAGES], stage_free[STAGES], scales_in[2], chunk_free[2], sums_ready, sums_taken, gave_up;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;

  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = uniform(cta_in_cluster());
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, slices = args.slices;
  const int f_tiles = (args.N + 255) / 256, n_tiles = f_tiles * ((args.T + 255) / 256);  // the weight's tiles innermost
  const int last_weight_tile = (args.N + MX_TILE_ROWS - 1) / MX_TILE_ROWS - 1;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&landed[s], 1);
      mbar_init(&stage_free[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&scales_in[b], 2);
      mbar_init(&chunk_free[b], 1);
    }
    mbar_init(&sums_ready, 1);
    mbar_init(&sums_taken, 16);  // the epilogue warps of both CTAs
    mbar_init(&gave_up, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) tmem_alloc_pair(&tmem_base_smem, 512);
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers stand before either signals the other's
  tc_fence_after();
  const uint32_t tmem = tmem_base_smem;

  const int most = args.F ? RUN_SLICES : RUN_SLICES_STORED;
  const int runs = LONG ? (slices + most - 1) / most : 1, run_slices = LONG ? slices / runs : slices, longer = slices - runs * run_slices;  // the first `longer` runs have one slice more
  const uint32_t chunk_room = tiles + STAGES * PAIR_STAGE_BYTES;
  static_assert(128 * 88 + (PAIR_THREADS - 128) * 208 <= PAIR_THREADS * 168, "the shares are of what the block was launched with");
  if (warp < 4) {
    if constexpr (LONG) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < 2) {
      // warp 0 the weight's rows and the scales of all 256, warp 1 the tokens: both CTAs' copies count on the first one's barrier
      if (warp == 1) {
        pdl_wait();
        pdl_launch();
      }
      const bool chosen = elect_lane();
      int it = 0, s = 0;  // slices asked for so far, over all tiles; the ring's stage
      uint32_t round = 1;  // parity of the phase in which it was last freed; the first round waits for nothing
      bool ok = true, free = true;
      const uint32_t first_landed = uniform(in_cluster_cta(&landed[0], 0));
      for (int tile = pair; tile < n_tiles && ok; tile += n_pairs) {
        // a number of rows that is no multiple of 256 leaves the second CTA without any: it reads the last ones, and what comes of them is not stored
        const int even = tile % f_tiles * 2 * slices, odd = min(tile % f_tiles * 2 + 1, last_weight_tile) * slices;
        const int t0 = tile / f_tiles * 256 + (int)rank * 128;
        for (int i = 0; i < slices; ++i, ++it) {
          if (!all_lanes(free)) ok = all_lanes(mbar_wait(&stage_free[s], round, &abort_flag));
          if (!ok) break;
          const uint32_t stage = tiles + s * PAIR_STAGE_BYTES, bar = first_landed + (uint32_t)s * 8;
          uint64_t* mine = &landed[s];
          s = s + 1 == STAGES ? 0 : s + 1;
          round ^= s == 0 ? 1u : 0u;
          free = it + 1 < STAGES || mbar_complete(&stage_free[s], round);
          if (chosen) {
            if (warp == 0) {
              if (rank == 0) mbar_expect_tx(mine, 2 * (A_BYTES + MX_TILE_CODES + 1024));
              load_tile_pair(stage + A_BYTES, &map_w, bar, 0, ((rank ? odd : even) + i) * MX_TILE_MAP_ROWS);
              load_tile_pair(stage + A_BYTES + B_BYTES, &map_s, bar, 0, (even + i) * MX_TILE_MAP_ROWS + MX_TILE_ROWS);
              load_tile_pair(stage + A_BYTES + B_BYTES + 512, &map_s, bar, 0, (odd + i) * MX_TILE_MAP_ROWS + MX_TILE_ROWS);
            } else {
              load_tile_pair(stage, &map_x, bar, i * MX_GROUP, t0);
            }
          }
        }
      }
      // what the first CTA's products say to this one's barriers has come before this one leaves
      for (int j = max(0, it - STAGES); warp == 0 && ok && j < it; ++j) ok = all_lanes(mbar_wait(&stage_free[j % STAGES], (uint32_t)(j / STAGES) & 1u, &abort_flag));
    } else if (warp == 3) {
      pdl_wait();
      const int row_bytes = 4 * slices;
      const bool wide = slices % 4 == 0 && (uintptr_t)args.x_scales % 16 == 0;
      const uint32_t tell = in_cluster_cta(&scales_in[0], 0);
      int c = 0;  // chunks so far
      bool ok = true;
      for (int tile = pair; tile < n_tiles && ok; tile += n_pairs) {
        const int t0 = tile / f_tiles * 256 + (int)rank * 128;
        for (int i = 0; i < slices; i += PAIR_CHUNK, ++c) {
          const int have = min(PAIR_CHUNK, slices - i);
          uint32_t v[4][PAIR_CHUNK];
  #pragma unroll
          for (int r = 0; r < 4; ++r) {  // a lane has rows lane, 32 + lane, ...
            const int t = t0 + r * 32 + lane;
            const uint8_t* src = args.x_scales + (size_t)min(t, args.T - 1) * row_bytes + 4 * i;
            if (wide && have >= 4) {
              const uint4 a = *reinterpret_cast<const uint4*>(src);
              const uint4 b = have == 8 ? *reinterpret_cast<const uint4*>(src + 16) : make_uint4(0u, 0u, 0u, 0u);
              v[r][0] = a.x, v[r][1] = a.y, v[r][2] = a.z, v[r][3] = a.w, v[r][4] = b.x, v[r][5] = b.y, v[r][6] = b.z, v[r][7] = b.w;
            } else {
  #pragma unroll
              for (int j = 0; j < PAIR_CHUNK; ++j) v[r][j] = j < have ? *reinterpret_cast<const uint32_t*>(src + 4 * j) : 0u;
            }
          }
          if (c >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&chunk_free[c & 1], (uint32_t)(c / 2 - 1) & 1u, &abort_flag));
          if (!ok) break;
          const uint32_t room = chunk_room + (uint32_t)((c & 1) * PAIR_CHUNK * 512 + lane * 16);
  #pragma unroll
          for (int j = 0; j < PAIR_CHUNK; ++j)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(room + j * 512), "r"(v[0][j]), "r"(v[1][j]), "r"(v[2][j]), "r"(v[3][j]) : "memory");
          fence_to_tensor_core();
          __syncwarp();
          if (lane == 0) mbar_arrive_in_cluster(tell + (uint32_t)(c & 1) * 8);
        }
      }
      for (int j = max(0, c - 2); ok && j < c; ++j) ok = __all_sync(0xffffffffu, mbar_wait(&chunk_free[j & 1], (uint32_t)(j / 2) & 1u, &abort_flag));
    } else if (warp == 2) {
      if (rank == 0) {
        const bool chosen = elect_lane();
        const uint32_t base = uniform(tmem);
        int done = 0, it = 0, c = 0, s = 0, place = 0;  // runs begun, slices and chunks so far, the ring's stage, the scales' place
        uint32_t round = 0;
        bool ok = true, ready = false, place_free = true;
        for (int tile = pair; tile < n_tiles && ok; tile += n_pairs, ++done) {
          // the tile's first slice and scales are there before the epilogue has the columns that this accumulator shares with the last one
          ok = all_lanes(mbar_wait_in_cluster(&scales_in[c & 1], (uint32_t)(c / 2) & 1u, &abort_flag));
          if (ok && !all_lanes(ready)) ok = all_lanes(mbar_wait(&landed[s], round, &abort_flag));
          ready = true;
          if (ok && done) ok = all_lanes(mbar_wait(&sums_taken, (uint32_t)(done - 1) & 1u, &abort_flag));
          if (!ok) break;
          tc_fence_after();
          uint32_t sums = base + (done & 1 ? PAIR_SECOND : 0), add = 0;  // a run's first products begin its sums
          int run = 0, left = run_slices + (LONG && longer > 0 ? 1 : 0);
          for (int i = 0; i < slices; ++i, ++it) {
            if (i % PAIR_CHUNK == 0 && i) ok = all_lanes(mbar_wait_in_cluster(&scales_in[c & 1], (uint32_t)(c / 2) & 1u, &abort_flag));
            if (ok && !all_lanes(ready)) ok = all_lanes(mbar_wait(&landed[s], round, &abort_flag));
            // the slice before it in this place of the scales: five slices ago, whose stage is the next one's now
            if (ok && !all_lanes(place_free)) ok = all_lanes(mbar_wait(&stage_free[s + 1 == STAGES ? 0 : s + 1], (uint32_t)((it - PAIR_SCALE_PLACES) / STAGES) & 1u, &abort_flag));
            if (LONG && left == 0) {  // the next run: the same waits as for a tile's first one
              if (ok) ok = all_lanes(mbar_wait(&sums_taken, (uint32_t)done & 1u, &abort_flag));
              ++done, ++run, left = run_slices + (run < longer ? 1 : 0), add = 0;
              sums = base + (done & 1 ? PAIR_SECOND : 0);
            }
            if (!ok) break;
            const uint32_t stage = tiles + s * PAIR_STAGE_BYTES, scales = stage + A_BYTES + B_BYTES;
            const uint32_t token_scales = chunk_room + (uint32_t)((c & 1) * PAIR_CHUNK + i % PAIR_CHUNK) * 512;
            const uint32_t scale_a = base + PAIR_SCALES + place * 12, scale_b = scale_a + 4;
            uint64_t* freed = &stage_free[s];
            s = s + 1 == STAGES ? 0 : s + 1;
            place = place + 1 == PAIR_SCALE_PLACES ? 0 : place + 1;
            round ^= s == 0 ? 1u : 0u;
            tc_fence_after();
            ready = mbar_complete(&landed[s], round);
            place_free = it + 1 < PAIR_SCALE_PLACES || mbar_complete(&stage_free[s + 1 == STAGES ? 0 : s + 1], (uint32_t)((it + 1 - PAIR_SCALE_PLACES) / STAGES) & 1u);
            const uint64_t a = smem_desc_sw128(stage), b = smem_desc_sw128(stage + A_BYTES);
            const bool chunk_ends = i % PAIR_CHUNK == PAIR_CHUNK - 1 || i == slices - 1;
            if (chosen) {
              scales_to_tmem_pair(scale_a, token_scales);
              scales_to_tmem_pair(scale_b, scales);
              scales_to_tmem_pair(scale_b + 4, scales + 512);
  #pragma unroll
              for (int j = 0; j < 4; ++j) umma_mx_pair(sums, a + 2 * j, b + 2 * j, mx_idesc(E4M3, E2M1, 256, 256, j), scale_a, scale_b, j ? 1u : add);
              umma_commit_pair(freed, 3);
              if (chunk_ends) umma_commit_pair(&chunk_free[c & 1], 3);
              if (LONG && left == 1 && i + 1 < slices) umma_commit_pair(&sums_ready, 3);
            }
            c += chunk_ends ? 1 : 0;
            add = 1;
            if (LONG) --left;
          }
          if (ok && chosen) umma_commit_pair(&sums_ready, 3);
        }
        if (!ok && chosen) {  // the products issued so far end before tensor memory is given back
          umma_commit_pair(&gave_up, 3);
          drain(&gave_up, 0);
          // and the copies asked for land
          for (int j = 0; j < STAGES; ++j) drain(&landed[j], 0), drain(&landed[j], 1);
        }
      }
    }
  } else {
    if constexpr (LONG) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int q = warp & 3, half = (warp - 4) >> 2;  // a quarter of the lanes (warps read 32 (w % 4) and on), half of the columns
    pdl_wait();  // what is written here, an earlier kernel may have been reading
    const uint32_t taken = in_cluster_cta(&sums_taken, 0);
    float* turn = reinterpret_cast<float*>(smem_raw + (tiles - smem_u32(smem_raw)) + PAIR_TURN) + (warp - 4) * 32 * TURN_PITCH;
    bool good = true;
    int done = 0;  // runs so far
    auto finish = [&](const uint32_t (&r)[64], int t, int row) {
      if (!args.F) pair_stored64(args, r, t - lane, row, good, turn, lane);
      else if (t >= args.T) ;
      else if (args.gate_alpha == 0.f) pair_gated64<false>(args, r, t, row, good);
      else pair_gated64<true>(args, r, t, row, good);
      __syncwarp();
    };
    for (int tile = pair; tile < n_tiles; tile += n_pairs, ++done) {
      const int row0 = (tile % f_tiles) * 256 + half * 128, t = tile / f_tiles * 256 + (int)rank * 128 + q * 32 + lane;
      uint32_t lo[LONG ? 64 : 1], hi[LONG ? 64 : 1];
#pragma unroll 1
      for (int run = 0;; ++run, ++done) {
        good = good && __all_sync(0xffffffffu, mbar_wait(&sums_ready, (uint32_t)done & 1u, &abort_flag));
        tc_fence_after();
        const bool second = done & 1, shared_half = half == (second ? 0 : 1);  // the shared columns: the first accumulator's last, the second's first
        const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (second ? PAIR_SECOND : 0) + half * 128;
        auto have_shared = [&]() {
          if (!shared_half) return;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) tell_in_cluster(taken);
        };
        if (!shared_half && lane == 0) tell_in_cluster(taken);  // this half's columns are no part of the next accumulator
        if constexpr (LONG) {  // the block with the shared columns first
          if (second) {
            pair_take64(at, lo, run == 0, have_shared);
            pair_take64(at + 64, hi, run == 0, [] {});
          } else {
            pair_take64(at + 64, hi, run == 0, have_shared);
            pair_take64(at, lo, run == 0, [] {});
          }
          if (run + 1 < runs) {
            tc_fence_before();
            continue;
          }
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {  // the epilogue's instructions once
            finish(lo, t, row0 + k * 64);
#pragma unroll
            for (int j = 0; j < 64; ++j) lo[j] = hi[j];
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < 2; ++k) {
            const int block = second ? k : 1 - k;
            uint32_t r[64];
            pair_load64(at + block * 64, r);
            if (k == 0) have_shared();
            finish(r, t, row0 + block * 64);
          }
        }
        tc_fence_before();
        break;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // neither CTA leaves, or frees tensor memory, while the other may still signal or read it
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
  if (threadIdx.x == 0 && abort_flag && args.status) atomicExch(args.status, 2);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static bool make_rows_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t bytes, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)bytes};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Two maps of a weight's tiles as rows of 64 bytes, 256 bytes at `maps`: 128 numbers of 4 bits, boxes of 128 rows (a tile's
// codes, unpacked on the way); bytes, boxes of 8 rows (its scales).
ALOFA_API int alofa_mx_weight_maps(void* maps, const void* tiles, long long n_tiles) {
  EncodeTiledFn fn = encode_fn();
  if (!fn || (uintptr_t)tiles % 32 || n_tiles <= 0 || n_tiles * MX_TILE_MAP_ROWS > 0x7fffffffll) return ALOFA_ERR_ARGUMENT;
  cuuint64_t rows = (cuuint64_t)(n_tiles * MX_TILE_MAP_ROWS), codes[2] = {MX_GROUP, rows}, bytes[2] = {MX_GROUP / 2, rows}, strides[1] = {MX_GROUP / 2};
  cuuint32_t codes_box[2] = {MX_GROUP, MX_TILE_ROWS}, bytes_box[2] = {MX_GROUP / 2, MX_TILE_MAP_ROWS - MX_TILE_ROWS}, elem[2] = {1, 1};
  CUtensorMap m[2];
  if (fn(&m[0], CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2, const_cast<void*>(tiles), codes, strides, codes_box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return ALOFA_ERR_ARGUMENT;
  if (fn(&m[1], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(tiles), bytes, strides, bytes_box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return ALOFA_ERR_ARGUMENT;
  memcpy(maps, m, sizeof(m));
  return ALOFA_OK;
}

// A kernel's shared memory is asked for once a device (a bit of `done` each; asking takes as long as a launch).
static bool allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
template <int BN> static std::atomic<uint64_t> few_allowed{0};
template <bool LONG> static std::atomic<uint64_t> pair_allowed{0};

template <int BN>
static int launch_few(const CUtensorMap& map_w, const CUtensorMap& map_x, const MxArgs& args, int parts, cudaStream_t stream) {
  const long long wide = (((long long)args.N + MX_TILE_ROWS - 1) / MX_TILE_ROWS) * parts, tall = ((long long)args.T + BN - 1) / BN;
  if (wide > 0x7fffffffll || tall > 65535) return ALOFA_ERR_ARGUMENT;
  if (!allow_shared((const void*)mx_few_kernel<BN>, (int)FewTile<BN>::SMEM, few_allowed<BN>)) return ALOFA_ERR_LAUNCH;
  launch_dep_cluster(mx_few_kernel<BN>, dim3((unsigned)wide, (unsigned)tall), FEW_THREADS, FewTile<BN>::SMEM, stream, parts, map_w, map_x, args, parts);
  return launch_status();
}

template <bool LONG>
static int launch_pair(const CUtensorMap& map_w, const CUtensorMap& map_s, const CUtensorMap& map_x, const MxArgs& args, unsigned grid, cudaStream_t stream) {
  if (!allow_shared((const void*)mx_pair_kernel<LONG>, (int)PAIR_SMEM, pair_allowed<LONG>)) return ALOFA_ERR_LAUNCH;
  launch_dep_cluster(mx_pair_kernel<LONG>, dim3(grid), PAIR_THREADS, PAIR_SMEM, stream, 2, map_w, map_s, map_x, args);
  return launch_status();
}

// A product as its caller packs it: one argument, where twenty-two would take longer to hand over than the launch.
// bn: 256: pairs of CTAs (`parts` 1, a grid of `ctas` of them); 16, 32, 64, 96 or 128 tokens a CTA, the depth in `parts` parts.
// features > 0: out are the codes and out_scales the scales of that many gated features, n the rows of the gated weight.
// weight_maps: alofa_mx_weight_maps' of the tiles.
struct MxCall {
  void* out;
  void* out_scales;
  const void* x_codes;
  const void* x_scales;
  const void* tiles;
  const void* weight_maps;
  const float* bias;
  const float* add;
  int* status;
  int t, n, k, features;
  float gate_alpha, gate_limit;
  int bn, parts, ctas, out_bf16;
};
static_assert(sizeof(MxCall) == 9 * 8 + 10 * 4, "as the caller packs it");

ALOFA_API int alofa_mx_gemm(const MxCall* call, void* stream) {
  void *out = call->out, *out_scales = call->out_scales;
  const void *x_codes = call->x_codes, *x_scales = call->x_scales, *tiles = call->tiles, *weight_maps = call->weight_maps;
  const float *bias = call->bias, *add = call->add;
  const int t = call->t, n = call->n, k = call->k, features = call->features, bn = call->bn, parts = call->parts, ctas = call->ctas, out_bf16 = call->out_bf16;
  const float gate_alpha = call->gate_alpha, gate_limit = call->gate_limit;
  int* status = call->status;
  if (t < 0 || n <= 0 || k <= 0 || k > (1 << 30) || n > (1 << 30) || (uintptr_t)x_codes % 16 || (uintptr_t)x_scales % 4 || (uintptr_t)tiles % 32) return ALOFA_ERR_ARGUMENT;
  if (features < 0 || (features && (n != 2 * ((features + 15) / 16 * 16) || !out_scales || (uintptr_t)out % 16))) return ALOFA_ERR_ARGUMENT;
  if (t == 0) return ALOFA_OK;
  MxArgs args = {};
  args.tiles = (const uint8_t*)tiles, args.x_scales = (const uint8_t*)x_scales;
  args.out = out, args.out_scales = (uint8_t*)out_scales, args.bias = bias, args.add = add;
  args.T = t, args.N = n, args.slices = (k + MX_GROUP - 1) / MX_GROUP, args.F = features, args.out_bf16 = out_bf16, args.status = status;
  args.gate_alpha = gate_alpha, args.gate_limit = gate_limit;
  args.wide = n % 4 == 0 && ((uintptr_t)out | (uintptr_t)bias | (uintptr_t)add) % 16 == 0;
  const bool few = bn == 16 || bn == 32 || bn == 64 || bn == 96 || bn == 128;
  if (!few && bn != 256) return ALOFA_ERR_ARGUMENT;
  if (parts < 1 || parts > args.slices || parts > (few ? FEW_PARTS : 1)) return ALOFA_ERR_ARGUMENT;
  CUtensorMap map_w, map_s, map_x;
  memcpy(&map_w, weight_maps, sizeof(map_w));
  memcpy(&map_s, (const uint8_t*)weight_maps + sizeof(map_w), sizeof(map_s));
  if (!make_rows_map(&map_x, x_codes, (uint64_t)t, (uint64_t)args.slices * MX_GROUP, few ? bn : 128)) return ALOFA_ERR_ARGUMENT;
  cudaStream_t s = (cudaStream_t)stream;
  switch (bn) {
    case 16: return launch_few<16>(map_w, map_x, args, parts, s);
    case 32: return launch_few<32>(map_w, map_x, args, parts, s);
    case 64: return launch_few<64>(map_w, map_x, args, parts, s);
    case 96: return launch_few<96>(map_w, map_x, args, parts, s);
    case 128: return launch_few<128>(map_w, map_x, args, parts, s);
  }
  const long long pair_tiles = (((long long)n + 255) / 256) * (((long long)t + 255) / 256);
  if (ctas < 2 || pair_tiles > 0x3fffffffll) return ALOFA_ERR_ARGUMENT;
  const unsigned grid = (unsigned)(2 * pair_tiles < ctas ? 2 * pair_tiles : ctas / 2 * 2);
  return args.slices > (features ? RUN_SLICES : RUN_SLICES_STORED) ? launch_pair<true>(map_w, map_s, map_x, args, grid, s) : launch_pair<false>(map_w, map_s, map_x, args, grid, s);
}
