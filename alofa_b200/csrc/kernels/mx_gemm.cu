// Product of rows in 8 bits and a weight in 4 (mx.cuh) on the 5th-generation tensor cores:
//   y[t, f] = sum_b 2^(sx[t, b] + sw[f, b] - 254) sum_{k in block b} x[t, k] w[f, k]   (+ bias[f]) (+ add[t, f])
// One tcgen05.mma.kind::mxf8f6f4.block_scale takes 128 weight rows, BN tokens and one block of 32 numbers;
// the scales are its operands too, in tensor memory, so sums are of the numbers themselves and in fp32.
//
// A k-slice is 128 numbers: four blocks.  A weight's tile of a slice is 8,704 contiguous bytes of memory
// (8,192 of codes, 512 of scales).  Shared memory holds 4-bit operands as 16 numbers in 8 bytes and 8 bytes
// of room, rows of 128 bytes with 128-byte swizzle: four warps copy them there 8 bytes at a time with
// cp.async, which spreads them on the way; each thread makes its own copies visible to the tensor core
// (fence.proxy.async) when they have landed.  Tokens come by TMA, their scales 4 bytes a row.  The weights
// depend on no earlier kernel of the stream: the first ring of them is asked for before the dependency wait.
//
// Scales in tensor memory have as many places as the ring has stages, so those of a slice are written
// only when the products that read the slice before them in that place are complete.
//
// Every wait on an mbarrier is bounded: after the limit the CTA raises the status word, lets its copies
// land, frees its tensor memory and returns.
#include "mx.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

#include <atomic>

constexpr int MX_THREADS = 192;  // warps 0-3 weights, then the epilogue; warp 4 tokens; warp 5 products

struct MxArgs {
  const uint8_t* tiles;     // the weight: [ceil(N / 128), slices, MX_TILE_BYTES]
  const uint8_t* x_scales;  // [T, 4 * slices]
  void* out;                // [T, N] bf16 or fp32
  const float* bias;        // [N] or null
  const float* add;         // [T, N] or null
  float* partial;           // [splits, T, N]: the sums of each part of the depth are left here, and nothing else done
  int T, N, slices, per_split, out_bf16;
  int* status;
};

__device__ __forceinline__ void copy8(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void copies_wait_but(int n) {  // all of this thread's groups but the last n
  switch (n) {
    case 0: copies_wait<0>(); break;
    case 1: copies_wait<1>(); break;
    case 2: copies_wait<2>(); break;
    case 3: copies_wait<3>(); break;
    case 4: copies_wait<4>(); break;
    case 5: copies_wait<5>(); break;
    default: copies_wait<6>(); break;
  }
}
__device__ __forceinline__ void fence_to_tensor_core() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 512 bytes of scales (32 rows of 16) to four columns of tensor memory, the same in all four quarters of its lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t smem) {
  const uint64_t desc = (uint64_t)((smem & 0x3FFFFu) >> 4) | (8ull << 16) | (8ull << 32) | (1ull << 46);  // rows of 16 bytes, groups of 8 rows 128 bytes apart, no swizzle
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mx(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)
      : "memory");
}
// Instruction: E2M1 (5) times E4M3 (0), scales E8M0, M = 128, N, the scales' byte `block` of their column.
constexpr uint32_t mx_idesc(int n, int block) { return (5u << 7) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (1u << 27) | ((uint32_t)block << 29) | ((uint32_t)block << 4); }

template <int BN>
struct MxTile {
  static constexpr int STAGES = BN <= 32 ? 5 : BN == 64 ? 4 : BN == 128 ? 3 : 4;
  static constexpr int B_ATOMS = BN > 128 ? 2 : 1;
  static constexpr uint32_t A_BYTES = MX_TILE_ROWS * MX_GROUP, B_BYTES = BN * MX_GROUP;
  static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES + (BN > 128 ? 2048 : 1024);  // tiles, 512 bytes of the weight's scales, the tokens'
  static constexpr uint32_t SMEM = STAGES * STAGE_BYTES + 1024;
  static constexpr int SCALE_COLS = 4 + 4 * B_ATOMS;
  static constexpr int COLS = BN + STAGES * SCALE_COLS;
  static constexpr uint32_t TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
};

template <int BN>
__global__ void __launch_bounds__(MX_THREADS, BN == 256 ? 1 : 2) mx_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const MxArgs args) {
  using Tile = MxTile<BN>;
  constexpr int STAGES = Tile::STAGES, AHEAD = STAGES - 1;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ uint64_t weights_in[STAGES], tokens_in[STAGES], stage_free[STAGES], sums_done;
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int f0 = blockIdx.x * MX_TILE_ROWS, t0 = blockIdx.y * BN;
  const int first = blockIdx.z * args.per_split, n = min(args.slices, first + args.per_split) - first;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&weights_in[s], 128);
      mbar_init(&tokens_in[s], 32 + 1);
      mbar_init(&stage_free[s], 1);
    }
    mbar_init(&sums_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) tmem_alloc(&tmem_base_smem, Tile::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_smem;

  if (warp < 4) {
    const uint8_t* src = args.tiles + ((size_t)blockIdx.x * args.slices + first) * MX_TILE_BYTES;
    const int row = threadIdx.x >> 3, chunk = threadIdx.x & 7;
    const uint32_t to = (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));  // rows 16 apart: the same place in their groups of 8
    int i = 0;
    for (; i < n; ++i) {
      const int s = i % STAGES;
      if (i >= STAGES && !mbar_wait(&stage_free[s], (uint32_t)(i / STAGES - 1) & 1u, &abort_flag)) break;
      const uint32_t stage = tiles + s * Tile::STAGE_BYTES;
      const uint8_t* from = src + (size_t)i * MX_TILE_BYTES;
#pragma unroll
      for (int j = 0; j < 8; ++j) copy8(stage + to + j * 16 * 128, from + j * 1024 + threadIdx.x * 8);
      if (threadIdx.x < 32) copy16(stage + Tile::A_BYTES + Tile::B_BYTES + threadIdx.x * 16, from + MX_TILE_CODES + threadIdx.x * 16);
      copies_end_group();
      if (i >= AHEAD) {
        copies_wait<AHEAD>();
        fence_to_tensor_core();
        mbar_arrive(&weights_in[(i - AHEAD) % STAGES]);
      }
    }
    for (int j = max(0, i - AHEAD); j < i; ++j) {
      copies_wait_but(i - 1 - j);
      fence_to_tensor_core();
      mbar_arrive(&weights_in[j % STAGES]);
    }
  } else if (warp == 4) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    pdl_launch();
    const int row_bytes = 4 * args.slices;
    int i = 0;
    for (; i < n; ++i) {
      const int s = i % STAGES;
      if (i >= STAGES && !mbar_wait(&stage_free[s], (uint32_t)(i / STAGES - 1) & 1u, &abort_flag)) break;
      const uint32_t stage = tiles + s * Tile::STAGE_BYTES, scales = stage + Tile::A_BYTES + Tile::B_BYTES + 512;
      if (lane == 0) {
        mbar_expect_tx(&tokens_in[s], Tile::B_BYTES);
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(stage + Tile::A_BYTES), "l"(&map_x),
                     "r"(smem_u32(&tokens_in[s])), "r"((first + i) * MX_GROUP), "r"(t0)
                     : "memory");
      }
#pragma unroll
      for (int r = 0; r < BN; r += 32) {
        const int t = r + lane;
        if (t < BN && t0 + t < args.T) copy4(scales + (uint32_t)((t >> 7) * 512 + mx_scale_at(t & 127, 0)), args.x_scales + (size_t)(t0 + t) * row_bytes + 4 * (first + i));
      }
      copies_end_group();
      if (i >= AHEAD) {
        copies_wait<AHEAD>();
        fence_to_tensor_core();
        mbar_arrive(&tokens_in[(i - AHEAD) % STAGES]);
      }
    }
    for (int j = max(0, i - AHEAD); j < i; ++j) {
      copies_wait_but(i - 1 - j);
      fence_to_tensor_core();
      mbar_arrive(&tokens_in[j % STAGES]);
    }
    // every slice asked for has its arrivals now: what is still in flight lands in a bounded time
    if (*(volatile int*)&abort_flag)
      for (int j = max(0, i - STAGES); j < i; ++j)
        for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(&tokens_in[j % STAGES], (uint32_t)(j / STAGES) & 1u); ++w) {
        }
  } else if (lane == 0) {
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int s = i % STAGES;
      const uint32_t parity = (uint32_t)(i / STAGES) & 1u;
      ok = mbar_wait(&weights_in[s], parity, &abort_flag) && mbar_wait(&tokens_in[s], parity, &abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t stage = tiles + s * Tile::STAGE_BYTES, scales = stage + Tile::A_BYTES + Tile::B_BYTES;
      const uint32_t scale_a = tmem + BN + s * Tile::SCALE_COLS, scale_b = scale_a + 4;
      scales_to_tmem(scale_a, scales);
#pragma unroll
      for (int a = 0; a < Tile::B_ATOMS; ++a) scales_to_tmem(scale_b + 4 * a, scales + 512 + 512 * a);
      const uint64_t a = smem_desc_sw128(stage), b = smem_desc_sw128(stage + Tile::A_BYTES);
#pragma unroll
      for (int j = 0; j < 4; ++j) umma_mx(tmem, a + 2 * j, b + 2 * j, mx_idesc(BN, j), scale_a, scale_b, (i | j) ? 1u : 0u);
      umma_commit(&stage_free[s]);
    }
    umma_commit(&sums_done);
    if (!ok)  // the products issued so far end before tensor memory is given back
      for (uint32_t w = 0; w < WAIT_LIMIT && !mbar_try_wait(&sums_done, 0); ++w) {
      }
  }
  __syncwarp();

  if (warp < 4) {
    if (mbar_wait(&sums_done, 0, &abort_flag) && !*(volatile int*)&abort_flag) {
      tc_fence_after();
      const int f = f0 + warp * 32 + lane;
      const bool live = f < args.N;
      asm volatile("griddepcontrol.wait;" ::: "memory");  // what is written here, an earlier kernel may still read
      const float bias = live && args.bias ? args.bias[f] : 0.f;
      for (int c = 0; c < BN && t0 + c < args.T; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c, r);
        tmem_ld_wait();
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = t0 + c + j;
          if (t >= args.T) break;
          const size_t at = (size_t)t * args.N + f;
          float v = __uint_as_float(r[j]);
          if (args.partial) {
            args.partial[(size_t)blockIdx.z * args.T * args.N + at] = v;
            continue;
          }
          v += bias;
          if (args.add) v += args.add[at];
          if (args.out_bf16) reinterpret_cast<bf16*>(args.out)[at] = __float2bfloat16_rn(v);
          else reinterpret_cast<float*>(args.out)[at] = v;
        }
      }
    } else if (threadIdx.x == 0 && args.status) {
      atomicExch(args.status, 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, Tile::TMEM_COLS);
}

// The sums of a depth's parts, in their order.
template <typename T>
__global__ void __launch_bounds__(256) mx_join_kernel(T* __restrict__ out, const float* __restrict__ partial, const float* __restrict__ bias, const float* __restrict__ add, long long count, int n, int splits) {
  pdl_wait();
  pdl_launch();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= count) return;
  float v = 0.f;
  for (int z = 0; z < splits; ++z) v += partial[z * count + i];
  if (bias) v += bias[i % n];
  if (add) v += add[i];
  out[i] = from_f<T>(v);
}

static bool make_rows_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t bytes, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)bytes};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, elem[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A kernel's shared memory is asked for once a device (a bit of `done` each; asking takes as long as a launch).
static bool allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
template <int BN> static std::atomic<uint64_t> configured{0};

template <int BN>
static int launch_mx(const CUtensorMap& map, const MxArgs& args, int splits, cudaStream_t stream) {
  const long long tall = ((long long)args.N + MX_TILE_ROWS - 1) / MX_TILE_ROWS, wide = ((long long)args.T + BN - 1) / BN;
  if (tall > 0x7fffffffll || wide > 65535 || splits > 65535) return ALOFA_ERR_ARGUMENT;
  if (!allow_shared((const void*)mx_gemm_kernel<BN>, (int)MxTile<BN>::SMEM, configured<BN>)) return ALOFA_ERR_LAUNCH;
  launch_dep(mx_gemm_kernel<BN>, dim3((unsigned)tall, (unsigned)wide, (unsigned)splits), MX_THREADS, MxTile<BN>::SMEM, stream, map, args);
  return launch_status();
}

// How many parts a depth of k really goes in when `splits` are asked for (every part has a slice).
ALOFA_API int alofa_mx_splits(int k, int splits) {
  const int slices = (k + MX_GROUP - 1) / MX_GROUP, per = (slices + splits - 1) / splits;
  return (slices + per - 1) / per;
}

// partial: [splits, T, N] for splits > 1; leave: the sums of the parts are the result, nothing is joined.
ALOFA_API int alofa_mx_gemm(void* out, float* partial, const void* x_codes, const void* x_scales, const void* tiles, const float* bias, const float* add, int t, int n, int k, int bn, int splits,
                            int leave, int out_bf16, int* status, void* stream) {
  if (t < 0 || n <= 0 || k <= 0 || k > (1 << 30) || splits < 1 || (uintptr_t)x_codes % 16 || (uintptr_t)x_scales % 4 || (uintptr_t)tiles % 16) return ALOFA_ERR_ARGUMENT;
  if (t == 0) return ALOFA_OK;
  const int slices = (k + MX_GROUP - 1) / MX_GROUP;
  if (splits > slices || alofa_mx_splits(k, splits) != splits || ((splits > 1 || leave) && !partial)) return ALOFA_ERR_ARGUMENT;
  MxArgs args = {};
  args.tiles = (const uint8_t*)tiles, args.x_scales = (const uint8_t*)x_scales;
  args.out = out, args.bias = bias, args.add = add, args.partial = splits > 1 || leave ? partial : nullptr;
  args.T = t, args.N = n, args.slices = slices, args.per_split = (slices + splits - 1) / splits, args.out_bf16 = out_bf16, args.status = status;
  CUtensorMap map;
  if (!make_rows_map(&map, x_codes, (uint64_t)t, (uint64_t)slices * MX_GROUP, bn)) return ALOFA_ERR_ARGUMENT;
  cudaStream_t s = (cudaStream_t)stream;
  int rc = ALOFA_ERR_ARGUMENT;
  switch (bn) {
    case 16: rc = launch_mx<16>(map, args, splits, s); break;
    case 32: rc = launch_mx<32>(map, args, splits, s); break;
    case 64: rc = launch_mx<64>(map, args, splits, s); break;
    case 128: rc = launch_mx<128>(map, args, splits, s); break;
    case 256: rc = launch_mx<256>(map, args, splits, s); break;
  }
  if (rc || leave || splits == 1) return rc;
  const long long count = (long long)t * n, blocks = (count + 255) / 256;
  if (blocks > 0x7fffffffll) return ALOFA_ERR_ARGUMENT;
  if (out_bf16) launch_dep(mx_join_kernel<bf16>, (unsigned)blocks, 256, 0, s, (bf16*)out, (const float*)partial, bias, add, count, n, splits);
  else launch_dep(mx_join_kernel<float>, (unsigned)blocks, 256, 0, s, (float*)out, (const float*)partial, bias, add, count, n, splits);
  return launch_status();
}
