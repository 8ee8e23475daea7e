// Device-side pieces shared by the kernels around 8-bit rows (rows8.hip holds the format's definition).
#pragma once
#include "rowio.h"

namespace mpnn {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));

// What a row's largest magnitude (as the bits of a float: infinities and NaN compare above every finite one) makes of it.
struct Quant {
  float inv, scale;
  uint32_t keep;   // all ones, or zeros for a row that is not finite
};
__device__ __forceinline__ Quant quant_of(uint32_t top) {
  const float t = __uint_as_float(top);
  const bool finite = top < 0x7f800000u, zero = t < 0x1p-100f;
  Quant r;
  r.inv = (zero || !finite) ? 0.f : 127.f / t;
  r.scale = !finite ? __builtin_nanf("") : (zero ? 0.f : t / 127.f);
  r.keep = finite ? ~0u : 0u;
  return r;
}
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The byte of v: 1.5 * 2^23 added in the same rounding leaves the whole number in the low byte.
__device__ __forceinline__ uint32_t quant_bits(float v, float inv) { return __float_as_uint(fmaf(v, inv, 12582912.f)); }
__device__ __forceinline__ uint32_t quant_word(float a, float b, float c, float d, const Quant& q) {
  const uint32_t lo = __builtin_amdgcn_perm(quant_bits(b, q.inv), quant_bits(a, q.inv), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(quant_bits(d, q.inv), quant_bits(c, q.inv), 0x04000c0cu);
  return (lo | hi) & q.keep;
}

// 16 bytes to a row that is not read here again.  Rows of whole 64-byte lines leave past the L2, which keeps the operands;
// other rows share lines with their neighbours, and the L2 must put the parts together: 1 M x 100 float32 results from
// 8-bit rows of 100 take 207 us past it and 147 through it, 1 M x 128 100 and 129.
__device__ __forceinline__ void store_chunk(void* p, i32x4 v, bool whole) {
  if (whole) {
    asm volatile("");   // on either side: keeps the two stores apart (joined, both would go through the L2)
    __builtin_nontemporal_store(v, static_cast<i32x4*>(p));
    asm volatile("");
  } else {
    *static_cast<i32x4*>(p) = v;
  }
}

// The widest stores that rows `pitch` bytes apart allow: 16 bytes, 8, or one output (0).  1 M x 100 bfloat16 results
// from 128 columns: 116 us with 8, 207 output by output.
inline int store_width(const void* y, int64_t pitch) {
  return ((uintptr_t)y | (uintptr_t)pitch) % 16 == 0 ? 16 : ((uintptr_t)y | (uintptr_t)pitch) % 8 == 0 ? 8 : 0;
}

// Results of a wave on their way to memory: ROWS rows x COLS outputs in LDS, from where whole row segments leave (128 bytes
// in bfloat16, 256 in float32; stores of 64 bytes per row took 1.65 instead of 1.20 ms for 4 M rows of 256 in float32).
// 16-byte chunk c of row r lies at c ^ r (mod the chunks of a row): writes by column and reads by row both spread.  Only
// the wave that owns the patch touches it.
template <typename Y, int ROWS, int COLS = 64>
struct Patch {
  static constexpr int VEC = 16 / sizeof(Y), CHUNKS = COLS / VEC, BYTES = ROWS * COLS * sizeof(Y);
  char* base;
  __device__ __forceinline__ void put(int row, int chunk, const float (&v)[VEC]) const {
    char* const p = base + row * (COLS * (int)sizeof(Y)) + ((chunk ^ row) & (CHUNKS - 1)) * 16;
    if constexpr (sizeof(Y) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
  // To rows r0 .. of y [N, ldy], outputs m .. m + COLS - 1 of which those below `end` exist, `width` bytes at a time (see
  // store_width).
  __device__ __forceinline__ void leave(void* y, int64_t ldy, int64_t N, int64_t r0, int m, int end, int width) const {
    const int lane = threadIdx.x & 63;
    const bool whole = (ldy * sizeof(Y)) % 64 == 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < ROWS * CHUNKS / 64; ++q) {
      const int r = q * (64 / CHUNKS) + lane / CHUNKS, chunk = lane % CHUNKS;
      const i32x4 v = *reinterpret_cast<const i32x4*>(base + r * (COLS * (int)sizeof(Y)) + ((chunk ^ r) & (CHUNKS - 1)) * 16);
      const int left = end - m - chunk * VEC;
      if (r0 + r >= N || left <= 0) continue;
      Y* const p = static_cast<Y*>(y) + (r0 + r) * ldy + m + chunk * VEC;
      if (width == 16 && left >= VEC) {
        store_chunk(p, v, whole);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (width >= 8 && left >= (h + 1) * (VEC / 2)) {
            *reinterpret_cast<i32x2*>(p + h * (VEC / 2)) = (i32x2){v[2 * h], v[2 * h + 1]};
          } else {
#pragma unroll
            for (int e = h * (VEC / 2); e < (h + 1) * (VEC / 2); ++e)
              if (e < left) {
                if constexpr (sizeof(Y) == 4) p[e] = __uint_as_float((uint32_t)v[e]);
                else p[e] = (Y)((uint32_t)v[e / 2] >> (16 * (e & 1)));
              }
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
};

}  // namespace mpnn
