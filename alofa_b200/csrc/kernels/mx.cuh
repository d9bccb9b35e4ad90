// Microscaled numbers: blocks of 32 along the depth that share a power of two, kept as a byte s
// that stands for 2^(s - 127) (255: not a number).  Rows are E4M3, weights E2M1.
//
// A block's scale is read off the bits of its largest magnitude, so it is exact:
//   rows     the smallest power of two by which that is no more than 448 = 1.75 * 2^8: nothing is
//            clipped (a clipped 511 would be off by an eighth, more than any rounding here);
//   weights  2^(floor(log2(largest)) - 2): between 4 and 8 by the scale, what is over 6 becomes 6.
//            The next power up would clip nothing but double the step of all 32 numbers, which
//            costs the other 31 more than the clipped one saves.
// A block that holds an infinity or a NaN has the scale 255: all of it is NaN, as is every sum it
// enters.  Dividing by the scale multiplies by a power of two that is a normal number, exact up to
// what falls below the smallest subnormal code anyway; the conversions round to nearest even.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

constexpr int MX_BLOCK = 32;       // numbers that share a scale
constexpr int MX_GROUP = 128;      // depths are padded to whole groups of this many (one tile of the product)
constexpr int MX_TILE_ROWS = 128;  // rows of a weight's tile
// A weight's tile: 128 rows of 64 bytes (128 numbers, the even ones in the low halves), then its scales as
// the tensor core reads them: 32 rows of 16 bytes, byte 4 j + b of row i the scale of row 32 j + i, block b.
constexpr int MX_TILE_CODES = MX_TILE_ROWS * MX_GROUP / 2;
constexpr int MX_TILE_BYTES = MX_TILE_CODES + MX_TILE_ROWS * (MX_GROUP / MX_BLOCK);
constexpr int MX_TILE_MAP_ROWS = MX_TILE_BYTES / (MX_GROUP / 2);  // a tile as rows of 64 bytes
constexpr int MX_GATE_ROWS = 16;   // a gated weight's rows: 16 of the gate, the same 16 of the up projection, and so on

__host__ __device__ __forceinline__ int mx_scale_at(int row, int block) { return (row & 31) * 16 + (row >> 5) * 4 + block; }

// The magnitude as bits: their order as whole numbers is that of the magnitudes, with infinity and NaN on top.
__device__ __forceinline__ uint32_t mx_size(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t mx_row_scale(uint32_t largest) {
  const int e = (int)(largest >> 23);
  if (e == 255) return 255u;
  return (uint32_t)max(0, e - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ uint32_t mx_weight_scale(uint32_t largest) {
  const int e = (int)(largest >> 23);
  return e == 255 ? 255u : (uint32_t)max(0, e - 2);
}
// 2^-(s - 127) for the scales above (s <= 252); 0 for a block of NaN, whose codes say nothing.
__device__ __forceinline__ float mx_over(uint32_t s) { return s == 255u ? 0.f : __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float mx_power(uint32_t s) { return s == 0u ? __uint_as_float(0x00400000u) : s == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(s << 23); }

// The codes of four numbers, the first in the lowest byte.  A block of NaN comes here as 0 * NaN, so codes are made of 0 there.
__device__ __forceinline__ uint32_t mx_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// Eight numbers in four bits each, the first in the lowest.
__device__ __forceinline__ uint32_t mx_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Two codes' numbers, the first in the low byte (half byte).  Every one of them is a half-precision number.
__device__ __forceinline__ float2 mx_from_e4m3(uint16_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(codes));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ float2 mx_from_e2m1(uint32_t codes) {
  uint32_t h;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t}"
      : "=r"(h)
      : "r"(codes));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// Eight neighbouring numbers a lane, four lanes a block: every lane gets the block's largest magnitude.
__device__ __forceinline__ uint32_t mx_largest4(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, mx_size(v[j]));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
// Eight numbers of a row (four lanes a block, every lane of the warp takes part): the codes at `codes`, the block's scale at `scale` from its first lane.
__device__ __forceinline__ void mx_put8(const float (&v)[8], uint8_t* codes, uint8_t* scale, bool live) {
  const uint32_t s = mx_row_scale(mx_largest4(v));
  if (!live) return;
  const float over = mx_over(s);
  uint2 c = make_uint2(0u, 0u);
  if (s != 255u) {
    c.x = mx_e4m3(v[0] * over, v[1] * over, v[2] * over, v[3] * over);
    c.y = mx_e4m3(v[4] * over, v[5] * over, v[6] * over, v[7] * over);
  }
  *reinterpret_cast<uint2*>(codes) = c;
  if ((threadIdx.x & 3) == 0) *scale = (uint8_t)s;
}

// silu(g) * u, or (CLAMPED) the clamped form (gate_times in common.cuh), where what comes out is rounded to 8 bits: a number
// near the border of two codes takes the other one if it is off by little, so e^-z is taken with the product z log2(e) in two
// parts (the rounding of that product alone would cost up to |z| / 2 units in the last place).  ex2.approx is within 2 units,
// rcp.approx within 1.  The logistic function is one from z = 30 up, infinity among them; from z = MX_GATE_FAR down, where e^-z and
// then its reciprocal leave the normal numbers, it is e^z to 2^-125 of itself, and its two halves e^(z/2) go to one factor each:
// g e^z alone would be zero, or a subnormal number of a few bits, beside a u that makes it large.
constexpr float MX_GATE_FAR = -87.f;
// 2^(c z) for c next to log2(e) or half of it: `rest` is what c as a float leaves out of it.
__device__ __forceinline__ float mx_power_of(float z, float c, float rest) {
  const float hi = c * z, lo = fmaf(c, z, -hi) + rest * z;
  float e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(hi));
  return fmaf(e, 0.6931471805599453f * lo, e);
}
__device__ __forceinline__ float mx_logistic(float z) {  // z above MX_GATE_FAR, or not a number
  z = fminf(z, 30.f);  // of what is not a number the factor beside this one is not either
  const float e = mx_power_of(z, -1.4426950408889634f, -1.92596299e-8f);  // log2(e) is 1.92596299e-8 more than the float
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
// FAR: gates below MX_GATE_FAR may be among them.
template <bool CLAMPED, bool FAR>
__device__ __forceinline__ float mx_gate_times(float g, float u, float alpha, float limit) {
  if (CLAMPED) {
    g = g > limit ? limit : g;  // not fminf: what is not a number stays so
    u = (u > limit ? limit : u < -limit ? -limit : u) + 1.0f;
  }
  const float z = CLAMPED ? alpha * g : g;
  if (FAR && z < MX_GATE_FAR) {
    const float half = mx_power_of(fmaxf(z, -1000.f), 0.7213475204444817f, 9.62981495e-9f);  // from -1,000 down it is zero, infinity among them
    return (g * half) * (u * half);
  }
  return g * mx_logistic(z) * u;
}
// Whether of several gates the least is so far below zero.
template <bool CLAMPED>
__device__ __forceinline__ bool mx_gate_far(float least, float alpha) { return (CLAMPED ? alpha * least : least) < MX_GATE_FAR; }
