// What makes microscaled numbers (mx.cuh), and what turns them back:
//   alofa_mx_rows        rows [T, K] in bf16 or fp32 -> E4M3 codes [T, Kp], scales [T, Kp / 32]
//   alofa_mx_norm        h = base + sum_z owed[z] (+ bias); the RMSNorm (or layer norm) of h's rows as such rows
//   alofa_mx_merge       the key splits of decode attention, joined, as such rows
//   alofa_mx_pack        a weight [N, K] in bf16 or fp32 -> tiles of E2M1 codes and scales
//   alofa_mx_rows_values, alofa_mx_weight_values   the numbers that rows, or a weight, stand for
// Kp is K rounded up to whole groups of 128; the codes behind K are zeros.
//
// All of them are bound by memory, and all but the packing are there twice.  WHOLE: rows that begin on 16 bytes and are whole groups
// of eight numbers: a lane takes eight or sixteen neighbouring ones with 16-byte loads, and the lanes that share a
// block find its largest magnitude by one or two shuffles.  Every other width: a block is 32 lanes, a number each
// (one instruction finds the largest), and a lane takes the same place of eight blocks: loads and stores of 2 or 4
// bytes, but of whole lines a warp (1,999 rows of 1,537 numbers turned back: 22.2 us when each lane took eight
// neighbouring ones, 9.2 so; the norm of as many with a plane 16.3 and 11.8).  Packing has four reductions a lane
// that way where it has one with neighbours: 8,960 x 1,537 41.6 us, and 17.4 with eight loads of a number each.
#include <string.h>

#include "mx.cuh"

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* src, int have, bool whole) {
  if (whole && have >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 p = *reinterpret_cast<const uint4*>(src);
      const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < have ? to_f(src[j]) : 0.f;
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8], int have, bool whole) {
  if (whole && have >= 8) {
    if constexpr (sizeof(T) == 2) {
      uint4 p;
      __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      __nv_bfloat162 c = __floats2bfloat162_rn(v[4], v[5]), d = __floats2bfloat162_rn(v[6], v[7]);
      p.x = *reinterpret_cast<uint32_t*>(&a), p.y = *reinterpret_cast<uint32_t*>(&b);
      p.z = *reinterpret_cast<uint32_t*>(&c), p.w = *reinterpret_cast<uint32_t*>(&d);
      *reinterpret_cast<uint4*>(dst) = p;
    } else {
      reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < have) dst[j] = from_f<T>(v[j]);
}

// Where a thread's eight numbers are: WHOLE eight neighbouring ones, else the lane's place in eight blocks that the warp
// has in turn.  `unit` counts threads along the row, 32 to a warp.
template <bool WHOLE>
struct Eight {
  int at;
  __device__ __forceinline__ explicit Eight(int unit) : at(WHOLE ? unit * 8 : (unit >> 5) * 256 + (unit & 31)) {}
  __device__ __forceinline__ int operator[](int j) const { return at + (WHOLE ? j : 32 * j); }
};
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_eight(float (&v)[8], const T* row, Eight<WHOLE> e, int k) {
  if constexpr (WHOLE) {
    load8(v, row + e.at, k - e.at, true);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = e[j] < k ? to_f(row[e[j]]) : 0.f;
  }
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store_eight(T* row, const float (&v)[8], Eight<WHOLE> e, int k) {
  if constexpr (WHOLE) {
    store8(row + e.at, v, k - e.at, true);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e[j] < k) row[e[j]] = from_f<T>(v[j]);
  }
}
// The same eight numbers as codes and scales of a row (every lane of the warp takes part).
template <bool WHOLE>
__device__ __forceinline__ void put_eight(const float (&v)[8], uint8_t* codes, uint8_t* scales, Eight<WHOLE> e, int kp, bool live) {
  if constexpr (WHOLE) {
    mx_put8(v, codes + e.at, scales + e.at / MX_BLOCK, live && e.at < kp);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t s = mx_row_scale(__reduce_max_sync(0xffffffffu, mx_size(v[j])));
      if (!live || e[j] >= kp) continue;
      codes[e[j]] = s == 255u ? (uint8_t)0 : (uint8_t)mx_e4m3(v[j] * mx_over(s), 0.f, 0.f, 0.f);
      if ((threadIdx.x & 31) == 0) scales[e[j] / MX_BLOCK] = (uint8_t)s;
    }
  }
}

static inline int padded(int k) { return (k + MX_GROUP - 1) / MX_GROUP * MX_GROUP; }
static inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// ---------------------------------------------------------------------------
// Rows: a lane has sixteen neighbouring numbers, two lanes a block.  Lanes are numbered over all rows in 32 bits
// (a 64-bit division by the row's length was a third of the instructions); what they address is 64.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) mx_rows_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ x, unsigned chunks, int k, int kp) {
  pdl_wait();
  pdl_launch();
  const unsigned i = blockIdx.x * blockDim.x + threadIdx.x, per_row = (unsigned)kp >> 4;  // a multiple of 8: a block's two lanes are in one row
  const bool live = i < chunks;
  const unsigned row = live ? i / per_row : 0u;
  const int c = live ? (int)(i - row * per_row) * 16 : 0;
  float v[2][8];
#pragma unroll
  for (int h = 0; h < 2; ++h) load8(v[h], x + (size_t)row * k + c + 8 * h, live ? k - c - 8 * h : 0, true);
  uint32_t largest = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) largest = max(largest, mx_size(v[j >> 3][j & 7]));
  largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
  if (!live) return;
  const uint32_t s = mx_row_scale(largest);
  const float over = mx_over(s);
  uint4 q = make_uint4(0u, 0u, 0u, 0u);
  if (s != 255u) {
    q.x = mx_e4m3(v[0][0] * over, v[0][1] * over, v[0][2] * over, v[0][3] * over);
    q.y = mx_e4m3(v[0][4] * over, v[0][5] * over, v[0][6] * over, v[0][7] * over);
    q.z = mx_e4m3(v[1][0] * over, v[1][1] * over, v[1][2] * over, v[1][3] * over);
    q.w = mx_e4m3(v[1][4] * over, v[1][5] * over, v[1][6] * over, v[1][7] * over);
  }
  *reinterpret_cast<uint4*>(codes + (size_t)row * kp + c) = q;
  if ((threadIdx.x & 1) == 0) scales[(size_t)row * (kp / MX_BLOCK) + c / MX_BLOCK] = (uint8_t)s;
}

// Every other width: a warp has 256 numbers of a row.
template <typename T>
__global__ void __launch_bounds__(256) mx_rows_any_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const T* __restrict__ x, unsigned warps, int k, int kp) {
  pdl_wait();
  pdl_launch();
  const unsigned warp = blockIdx.x * 8 + (threadIdx.x >> 5), per_row = (unsigned)(kp + 255) >> 8;
  const bool live = warp < warps;
  const size_t row = live ? warp / per_row : 0u;
  const Eight<false> e((int)(live ? warp % per_row : 0u) * 32 + (int)(threadIdx.x & 31));
  float v[8];
  load_eight(v, x + row * k, e, live ? k : 0);
  put_eight(v, codes + row * kp, scales + row * (kp / MX_BLOCK), e, kp, live);
}

ALOFA_API int alofa_mx_rows(void* codes, void* scales, const void* x, int t, int k, int bf16_x, void* stream) {
  if (t < 0 || k <= 0 || k > (1 << 30) || !aligned(codes, 16)) return ALOFA_ERR_ARGUMENT;
  if (t == 0) return ALOFA_OK;
  const int kp = padded(k);
  const bool whole = k % 8 == 0 && aligned(x, 16);
  const long long units = whole ? (long long)t * (kp / 16) : (long long)t * ((kp + 255) / 256);  // lanes, or warps
  if (units > 0x7fffffffll) return ALOFA_ERR_ARGUMENT;
  const unsigned blocks = (unsigned)(whole ? (units + 255) / 256 : (units + 7) / 8);
  cudaStream_t s = (cudaStream_t)stream;
  uint8_t *c = (uint8_t*)codes, *e = (uint8_t*)scales;
  if (whole && bf16_x) launch_dep(mx_rows_kernel<bf16>, blocks, 256, 0, s, c, e, (const bf16*)x, (unsigned)units, k, kp);
  else if (whole) launch_dep(mx_rows_kernel<float>, blocks, 256, 0, s, c, e, (const float*)x, (unsigned)units, k, kp);
  else if (bf16_x) launch_dep(mx_rows_any_kernel<bf16>, blocks, 256, 0, s, c, e, (const bf16*)x, (unsigned)units, k, kp);
  else launch_dep(mx_rows_any_kernel<float>, blocks, 256, 0, s, c, e, (const float*)x, (unsigned)units, k, kp);
  return launch_status();
}

// Turned back: a lane has eight numbers (a warp's stores are whole lines; with sixteen they were every other 16 bytes: 1,999
// rows of 18,944 24.3 us, and 21.0 so), a thread two such places.
constexpr int VALUES_THREADS = 256, VALUES_PLACES = 2 * VALUES_THREADS;

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(VALUES_THREADS) mx_rows_values_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, unsigned units, int k, int kp) {
  pdl_wait();
  pdl_launch();
  const unsigned per_row = WHOLE ? (unsigned)k >> 3 : (unsigned)(kp + 255) / 256 * 32;  // not WHOLE: whole warps
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned i = blockIdx.x * VALUES_PLACES + h * VALUES_THREADS + threadIdx.x;
    if (i >= units) return;
    const size_t row = i / per_row;
    const Eight<WHOLE> e((int)(i - (unsigned)row * per_row));
    const uint8_t *c = codes + row * kp, *s = scales + row * (kp / MX_BLOCK);
    float v[8];
    if constexpr (WHOLE) {
      const uint2 p = *reinterpret_cast<const uint2*>(c + e.at);
      const float by = mx_power(s[e.at / MX_BLOCK]);
      const uint32_t w[2] = {p.x, p.y};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 two = mx_from_e4m3((uint16_t)(w[j >> 1] >> (16 * (j & 1))));
        v[2 * j] = two.x * by, v[2 * j + 1] = two.y * by;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = e[j] < k ? mx_from_e4m3(c[e[j]]).x * mx_power(s[e[j] / MX_BLOCK]) : 0.f;
    }
    store_eight(out + row * k, v, e, k);
  }
}

ALOFA_API int alofa_mx_rows_values(void* out, const void* codes, const void* scales, int t, int k, int bf16_out, void* stream) {
  if (t < 0 || k <= 0 || k > (1 << 30) || !aligned(codes, 16)) return ALOFA_ERR_ARGUMENT;
  if (t == 0) return ALOFA_OK;
  const int kp = padded(k);
  const bool whole = k % 8 == 0 && aligned(out, 16);
  const long long units = (long long)t * (whole ? k / 8 : (kp + 255) / 256 * 32);
  if (units > 0x7fffffffll) return ALOFA_ERR_ARGUMENT;
  const unsigned blocks = (unsigned)((units + VALUES_PLACES - 1) / VALUES_PLACES);
  cudaStream_t s = (cudaStream_t)stream;
  const uint8_t *c = (const uint8_t*)codes, *e = (const uint8_t*)scales;
  if (whole && bf16_out) launch_dep(mx_rows_values_kernel<bf16, true>, blocks, VALUES_THREADS, 0, s, (bf16*)out, c, e, (unsigned)units, k, kp);
  else if (whole) launch_dep(mx_rows_values_kernel<float, true>, blocks, VALUES_THREADS, 0, s, (float*)out, c, e, (unsigned)units, k, kp);
  else if (bf16_out) launch_dep(mx_rows_values_kernel<bf16, false>, blocks, VALUES_THREADS, 0, s, (bf16*)out, c, e, (unsigned)units, k, kp);
  else launch_dep(mx_rows_values_kernel<float, false>, blocks, VALUES_THREADS, 0, s, (float*)out, c, e, (unsigned)units, k, kp);
  return launch_status();
}

// ---------------------------------------------------------------------------
// The norm.  A block has a row and a thread CH chunks of eight numbers of it, which stay in registers: the row is
// read once, with all its loads in flight together, four planes of owed sums at a time.  Sums are taken in a
// fixed order.  Formula: src/alofa/kernels/cpu/scalar.mojo:93-129.
// ---------------------------------------------------------------------------
template <int CH, bool WHOLE>
__global__ void __launch_bounds__(512) mx_norm_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, float* h, const float* base, const float* __restrict__ owed, int splits,
                                                      const float* __restrict__ bias, const float* __restrict__ w, const float* __restrict__ shift, int t, int k, int kp, float eps) {
  __shared__ float scratch[32];
  pdl_wait();
  const int row = blockIdx.x;
  const size_t at = (size_t)row * k, plane = (size_t)t * k;
  constexpr int PLANES = CH == 1 ? 4 : 1;
  auto place = [&](int i) { return Eight<WHOLE>((int)(threadIdx.x + i * blockDim.x)); };
  float v[CH][8], g[CH == 1 ? 1 : CH][8];
  float ss = 0.f, sum = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    load_eight(v[i], base + at, place(i), k);
    if (CH == 1) load_eight(g[i], w, place(i), k);
  }
  int z = 0;
  for (; z + PLANES <= splits; z += PLANES) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float p[PLANES][8];
#pragma unroll
      for (int q = 0; q < PLANES; ++q) load_eight(p[q], owed + (z + q) * plane + at, place(i), k);
#pragma unroll
      for (int q = 0; q < PLANES; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += p[q][j];
    }
  }
  for (; z < splits; ++z) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float p[8];
      load_eight(p, owed + z * plane + at, place(i), k);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += p[j];
    }
  }
  pdl_launch();
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (bias) {
      float p[8];
      load_eight(p, bias, place(i), k);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += p[j];
    }
    if (owed || bias || h != base) store_eight(h + at, v[i], place(i), k);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(v[i][j], v[i][j], ss);
      sum += v[i][j];
    }
  }
  float mean = 0.f;
  if (shift) {
    mean = block_sum(sum, scratch) / (float)k;
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = place(i)[j] < k ? v[i][j] - mean : 0.f;
        ss = fmaf(d, d, ss);
      }
    }
  }
  ss = block_sum(ss, scratch);
  const float scale = 1.0f / sqrtf(ss / (float)k + eps);
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    float s[8];
    if (CH > 1) load_eight(g[i], w, place(i), k);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 0.f;
    if (shift) load_eight(s, shift, place(i), k);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = place(i)[j] < k ? fmaf((v[i][j] - mean) * scale, g[i][j], s[j]) : 0.f;
    put_eight(v[i], codes + (size_t)row * kp, scales + (size_t)row * (kp / MX_BLOCK), place(i), kp, true);
  }
}

ALOFA_API int alofa_mx_norm(void* codes, void* scales, float* h, const float* base, const float* owed, int splits, const float* bias, const float* w, const float* shift, int t, int k, float eps,
                            void* stream) {
  if (t < 0 || k <= 0 || splits < 0 || !aligned(codes, 8)) return ALOFA_ERR_ARGUMENT;
  if (t == 0) return ALOFA_OK;
  if (!splits) owed = nullptr;
  const int kp = padded(k), chunks = kp / 8;
  // a chunk a thread where the rows are few and a row's time is what counts, two where they are many: 2,048 rows of 3,584
  // with one plane 21.4 and 18.9 us, one row of 896 with four planes 3.8 and 5.8 (blocks that stay and ask for their next
  // row ahead: 18.9 us, and without a plane 16.9 instead of 13.8)
  const int per = chunks <= (t >= 2 * 148 ? 256 : 512) ? 1 : chunks <= 1024 ? 2 : chunks <= 2048 ? 4 : 8, threads = ((chunks + per - 1) / per + 31) / 32 * 32;
  if (threads > 512) return ALOFA_ERR_ARGUMENT;
  const bool whole = k % 8 == 0 && aligned(h, 16) && aligned(base, 16) && aligned(owed, 16) && aligned(bias, 16) && aligned(w, 16) && aligned(shift, 16);
#define GO(CH)                                                                                                                                                                        \
  do {                                                                                                                                                                                \
    if (whole) launch_dep(mx_norm_kernel<CH, true>, t, threads, 0, (cudaStream_t)stream, (uint8_t*)codes, (uint8_t*)scales, h, base, owed, splits, bias, w, shift, t, k, kp, eps);        \
    else launch_dep(mx_norm_kernel<CH, false>, t, threads, 0, (cudaStream_t)stream, (uint8_t*)codes, (uint8_t*)scales, h, base, owed, splits, bias, w, shift, t, k, kp, eps);             \
  } while (0)
  switch (per) {
    case 1: GO(1); break;
    case 2: GO(2); break;
    case 4: GO(4); break;
    default: GO(8); break;
  }
#undef GO
  return launch_status();
}

// ---------------------------------------------------------------------------
// Attention's output as rows: decode tokens whose keys were split over CTAs have an output, a maximum and a sum for
// each split (scores in log2 units), and here they become one, o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, as
// attention_combine_kernel has it (src/alofa/kernels/cpu/scalar.mojo:392-470), and go to 8 bits without a stop in
// bfloat16.  A lane has eight channels; the loads of eight splits are in flight together.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(128) mx_merge_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, const float* __restrict__ po, const float* __restrict__ pml, const int* __restrict__ positions,
                                                       unsigned chunks, int t, int heads, int hd, int kp, int splits, int window, int split_keys) {
  pdl_wait();
  pdl_launch();
  const unsigned i = blockIdx.x * blockDim.x + threadIdx.x, per_row = (unsigned)kp >> 3;
  const bool live = i < chunks;
  const int row = live ? (int)(i / per_row) : 0, c = live ? (int)(i % per_row) * 8 : 0;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if (live && c < heads * hd) {
    const int head = c / hd, d = c - head * hd, p = positions[row];
    const size_t rows = (size_t)t * heads, at = (size_t)row * heads + head;
    // splits that hold keys of this token: none before the first position
    const int first = (window > 0 ? max(0, p - window + 1) : 0) / split_keys, last = p < 0 ? -1 : min(p / split_keys, splits - 1);
    float m = -INFINITY, l = 0.f;
    for (int s0 = first; s0 <= last; s0 += 8) {
      float2 ml[8];
      float4 lo[8], hi[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const size_t s = (size_t)min(s0 + k, last) * rows + at;
        ml[k] = *reinterpret_cast<const float2*>(pml + s * 2);
        const float4* o = reinterpret_cast<const float4*>(po + s * hd + d);
        lo[k] = o[0], hi[k] = o[1];
        if (s0 + k > last) ml[k].x = -INFINITY;
      }
      float next = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) next = fmaxf(next, ml[k].x);
      if (next == -INFINITY) continue;  // splits that see nothing so far
      const float keep = exp2f(m - next);
      m = next, l *= keep;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= keep;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (ml[k].x == -INFINITY) continue;
        const float w = exp2f(ml[k].x - m);
        l = fmaf(ml[k].y, w, l);
        v[0] = fmaf(lo[k].x, w, v[0]), v[1] = fmaf(lo[k].y, w, v[1]), v[2] = fmaf(lo[k].z, w, v[2]), v[3] = fmaf(lo[k].w, w, v[3]);
        v[4] = fmaf(hi[k].x, w, v[4]), v[5] = fmaf(hi[k].y, w, v[5]), v[6] = fmaf(hi[k].z, w, v[6]), v[7] = fmaf(hi[k].w, w, v[7]);
      }
    }
    const float over = 1.0f / l;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= over;
  }
  mx_put8(v, codes + (size_t)row * kp + c, scales + (size_t)row * (kp / MX_BLOCK) + c / MX_BLOCK, live);
}

ALOFA_API int alofa_mx_merge(void* codes, void* scales, const float* po, const float* pml, const int* positions, int t, int heads, int hd, int splits, int window, int split_keys, void* stream) {
  if (t < 0 || heads <= 0 || hd <= 0 || hd % 8 || heads > (1 << 30) / hd || splits < 0 || window < 0 || split_keys <= 0 || !aligned(codes, 16) || !aligned(po, 16) || !aligned(pml, 8)) return ALOFA_ERR_ARGUMENT;
  if (t == 0) return ALOFA_OK;
  const int kp = padded(heads * hd);
  const long long chunks = (long long)t * (kp / 8);
  if (chunks > 0x7fffffffll) return ALOFA_ERR_ARGUMENT;
  launch_dep(mx_merge_kernel, (unsigned)((chunks + 127) / 128), 128, 0, (cudaStream_t)stream, (uint8_t*)codes, (uint8_t*)scales, po, pml, positions, (unsigned)chunks, t, heads, hd, kp, splits, window, split_keys);
  return launch_status();
}

// ---------------------------------------------------------------------------
// Weights: a block makes tiles of 128 rows and 128 numbers of each, up to four along the depth; a lane has eight
// neighbouring numbers of four rows of a tile, and asks for the next tile's before it works on this one's.
// `features` > 0: a gated weight whose row f is the gate's and features + f the up projection's.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int weight_source_row(int r, int n, int features) {
  if (!features) return r < n ? r : -1;
  const int f = r / (2 * MX_GATE_ROWS) * MX_GATE_ROWS + r % MX_GATE_ROWS, half = r / MX_GATE_ROWS % 2;
  return f < features ? half * features + f : -1;
}

constexpr int PACK_THREADS = 512, PACK_TILES = 4;  // tiles of a block, where there are enough for two blocks an SM (one each otherwise)

template <typename T, bool WHOLE>
struct Raw8 {  // eight neighbouring numbers as they are loaded, the first `have` of them
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* src, int have) {
    if constexpr (WHOLE) {
#pragma unroll
      for (int j = 0; j < (int)(sizeof(T) / 2); ++j) q[j] = have > 0 ? reinterpret_cast<const uint4*>(src)[j] : make_uint4(0u, 0u, 0u, 0u);
    } else {
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < have ? src[j] : from_f<T>(0.f);
      memcpy(q, v, sizeof(v));
    }
  }
  __device__ __forceinline__ void numbers(float (&v)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t w[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      memcpy(v, q, sizeof(v));
    }
  }
};

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(PACK_THREADS, sizeof(T) == 2 ? 2 : 1) mx_pack_kernel(uint8_t* __restrict__ tiles, const T* __restrict__ w, int n, int k, int slices, int each, int features) {
  const int c = (threadIdx.x & 15) * 8, r0 = threadIdx.x >> 4, first = blockIdx.x * each, last = min(slices, first + each);
  const T* src[4];
  bool there[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = weight_source_row(blockIdx.y * MX_TILE_ROWS + i * 32 + r0, n, features);
    there[i] = row >= 0;
    src[i] = w + (size_t)max(row, 0) * k + c;
  }
  Raw8<T, WHOLE> next[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) next[i].load(src[i] + first * MX_GROUP, there[i] ? k - c - first * MX_GROUP : 0);
  for (int s = first; s < last; ++s) {
    uint8_t* tile = tiles + ((size_t)blockIdx.y * slices + s) * MX_TILE_BYTES;
    Raw8<T, WHOLE> now[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) now[i] = next[i];
    if (s + 1 < last) {
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i].load(src[i] + (s + 1) * MX_GROUP, there[i] ? k - c - (s + 1) * MX_GROUP : 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 32 + r0;
      float v[8];
      now[i].numbers(v);
      const uint32_t e = mx_weight_scale(mx_largest4(v));
      const float over = mx_over(e);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= over;
      *reinterpret_cast<uint32_t*>(tile + r * (MX_GROUP / 2) + c / 2) = e == 255u ? 0u : mx_e2m1(v);
      if ((threadIdx.x & 3) == 0) tile[MX_TILE_CODES + mx_scale_at(r, c / MX_BLOCK)] = (uint8_t)e;
    }
  }
}

// Products read a weight before the kernel ahead of them in the stream has ended (it is constant by then).  What
// makes one therefore ends with this: an ordinary launch, which begins when the tiles are complete and visible, and
// so does whatever may begin beside it.
__global__ void mx_settle_kernel() {}

ALOFA_API int alofa_mx_settle(void* stream) {
  launch_whole(mx_settle_kernel, 1, 32, 0, (cudaStream_t)stream);
  return launch_status();
}

// n: rows of the weight; gated: they are the gate's n / 2 and the up projection's.
ALOFA_API int alofa_mx_pack(void* tiles, const void* w, int n, int k, int gated, int bf16_w, void* stream) {
  if (n <= 0 || k <= 0 || k > (1 << 30) || (gated && n % 2) || !aligned(tiles, 16)) return ALOFA_ERR_ARGUMENT;
  const long long rows = gated ? 2ll * ((n / 2 + 15) / 16 * 16) : n, tall = (rows + MX_TILE_ROWS - 1) / MX_TILE_ROWS;
  if (tall > 65535) return ALOFA_ERR_ARGUMENT;
  const int slices = padded(k) / MX_GROUP;
  const bool whole = k % 8 == 0 && aligned(w, 16);
  const int each = whole && slices * tall >= 2 * 148 * PACK_TILES ? PACK_TILES : 1;
  const dim3 grid((unsigned)((slices + each - 1) / each), (unsigned)tall);
  const int features = gated ? n / 2 : 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (whole && bf16_w) launch_whole(mx_pack_kernel<bf16, true>, grid, PACK_THREADS, 0, s, (uint8_t*)tiles, (const bf16*)w, n, k, slices, each, features);
  else if (whole) launch_whole(mx_pack_kernel<float, true>, grid, PACK_THREADS, 0, s, (uint8_t*)tiles, (const float*)w, n, k, slices, each, features);
  else if (bf16_w) launch_whole(mx_pack_kernel<bf16, false>, grid, PACK_THREADS, 0, s, (uint8_t*)tiles, (const bf16*)w, n, k, slices, each, features);
  else launch_whole(mx_pack_kernel<float, false>, grid, PACK_THREADS, 0, s, (uint8_t*)tiles, (const float*)w, n, k, slices, each, features);
  const int rc = launch_status();
  return rc ? rc : alofa_mx_settle(stream);
}

template <typename T>
__global__ void __launch_bounds__(PACK_THREADS) mx_weight_values_kernel(T* __restrict__ out, const uint8_t* __restrict__ tiles, int n, int k, int features) {
  const uint8_t* tile = tiles + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * MX_TILE_BYTES;
  const int c = (threadIdx.x & 15) * 8, kc = blockIdx.x * MX_GROUP + c, r0 = threadIdx.x >> 4;
  pdl_wait();
  pdl_launch();
  uint32_t p[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = *reinterpret_cast<const uint32_t*>(tile + (i * 32 + r0) * (MX_GROUP / 2) + c / 2);
    s[i] = tile[MX_TILE_CODES + mx_scale_at(i * 32 + r0, c / MX_BLOCK)];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int src = weight_source_row(blockIdx.y * MX_TILE_ROWS + i * 32 + r0, n, features);
    const float by = mx_power(s[i]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 two = mx_from_e2m1(p[i] >> (8 * j));
      v[2 * j] = two.x * by, v[2 * j + 1] = two.y * by;
    }
    if (src >= 0 && kc < k) store8(out + (size_t)src * k + kc, v, k - kc, true);
  }
}

template <typename T>
__global__ void __launch_bounds__(PACK_THREADS) mx_weight_values_any_kernel(T* __restrict__ out, const uint8_t* __restrict__ tiles, int n, int k, int features) {
  const uint8_t* tile = tiles + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * MX_TILE_BYTES;
  const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * 8, kc = blockIdx.x * MX_GROUP + lane;
  pdl_wait();
  pdl_launch();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + i, src = weight_source_row(blockIdx.y * MX_TILE_ROWS + r, n, features);
    if (src < 0) continue;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t code = tile[r * (MX_GROUP / 2) + b * 16 + lane / 2] >> (4 * (lane & 1));
      if (kc + 32 * b < k) out[(size_t)src * k + kc + 32 * b] = from_f<T>(mx_from_e2m1(code & 15u).x * mx_power(tile[MX_TILE_CODES + mx_scale_at(r, b)]));
    }
  }
}

ALOFA_API int alofa_mx_weight_values(void* out, const void* tiles, int n, int k, int gated, int bf16_out, void* stream) {
  if (n <= 0 || k <= 0 || k > (1 << 30) || (gated && n % 2) || !aligned(tiles, 16)) return ALOFA_ERR_ARGUMENT;
  const long long rows = gated ? 2ll * ((n / 2 + 15) / 16 * 16) : n, tall = (rows + MX_TILE_ROWS - 1) / MX_TILE_ROWS;
  if (tall > 65535) return ALOFA_ERR_ARGUMENT;
  const dim3 grid((unsigned)(padded(k) / MX_GROUP), (unsigned)tall);
  const bool whole = k % 8 == 0 && aligned(out, 16);
  const int features = gated ? n / 2 : 0;
  cudaStream_t s = (cudaStream_t)stream;
  if (whole && bf16_out) launch_dep(mx_weight_values_kernel<bf16>, grid, PACK_THREADS, 0, s, (bf16*)out, (const uint8_t*)tiles, n, k, features);
  else if (whole) launch_dep(mx_weight_values_kernel<float>, grid, PACK_THREADS, 0, s, (float*)out, (const uint8_t*)tiles, n, k, features);
  else if (bf16_out) launch_dep(mx_weight_values_any_kernel<bf16>, grid, PACK_THREADS, 0, s, (bf16*)out, (const uint8_t*)tiles, n, k, features);
  else launch_dep(mx_weight_values_any_kernel<float>, grid, PACK_THREADS, 0, s, (float*)out, (const uint8_t*)tiles, n, k, features);
  return launch_status();
}
