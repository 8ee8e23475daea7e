// A Linear call whose inputs wait for the backward in 8 bits (rows8.hip), in one pass over them:
//
//   y = act(x W1^T [+ x2 W2^T])     and, from the same registers,     q, scale [, q2, scale2] = rows of x [, x2] in 8 bits,
//   bits = one bit per output, set where the relu is open
//
// (models/layers.py:104 and :140 without the concatenation).  Products on v_mfma_f32_16x16x32_bf16, float32 sums, one
// rounding.  The weights, [W1 | W2], stay in LDS; a wave takes 16 (or 32) rows at a time as they lie in memory, takes
// them to 8 bits and multiplies them with every 32 outputs in turn.  Results, 8-bit rows and bits leave through LDS as
// whole row segments.
//
//   bfloat16   a lane's 16-byte loads are the matrix operand: (row i, group g) holds columns 32 s + 8 g .. + 7 of step s.
//              Bound by memory: 4 M rows, 128 + 128 -> 128, in 0.90 to 0.96 ms (4.2 to 4.5 TB/s; a copy reaches 4.9), where a
//              product, two quantising passes and a pass over y took 0.64 + 0.60 + 0.24 ms.
//   float32    the three bfloat16 pieces and six products per pair of k_gemm_nt (gemm.hip) in its order, so that y is the same
//              to the bit with and without kept rows.  The weights' pieces lie in LDS, cut once per block; weights that do
//              not fit go in two slices, and x is read once per slice.  Bound by the matrix cores: 4 M rows, 128 -> 256, in 1.79 ms
//              (0.88 PFLOP/s of piece products, where a large bfloat16 product reaches 1.28; the separate passes 2.29), 128 -> 128
//              in 0.95 (1.44); 1 M rows, 64 + 64 -> 64, in 195 us (330).
//
// Without kept rows the same kernels are the input gradient of those calls, y = x W for W as it lies [K, M]: brought into
// place on its way to LDS, it saves the pass that transposes it (with that pass and gemm_nt: 18,432 x 64 -> 64 float32 16 us,
// here 9; 4 M x 128 -> 256 bfloat16 0.66 and 0.59 ms, float32 1.83 and 1.63).
#include "common.h"
#include "rows8.h"

#include <cstdlib>

namespace mpnn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kKeptThreads = 512;
constexpr int kKeptWaves = kKeptThreads / 64;
constexpr int kKeptWeights = 120 * 1024;

struct KeptSeg {
  const void* x; int64_t ldx;
  int8_t* q; int64_t ldq;
  float* scale;
  int K;
};
struct KeptArgs {
  KeptSeg a, b;                     // b.K = 0: one input
  const void* w; int64_t ldw;       // [M, K + K2]
  void* y; int64_t ldy;
  uint8_t* bits;                    // optional
  int64_t N;
  int M, relu;
  int width;                        // of the stores (store_width)
  int across;                       // the weights lie as [K, M]: y = x W (one input, nothing kept: the input gradient)
};

constexpr int kept_pitch(int ks) { return ks * 64 + 16; }   // bytes of a weight row in LDS: 16 more spread eight rows over the banks

// 32-column steps of a width, as the kernels come: 1, 2, 4 or 8
constexpr int kept_steps(int K) { return K <= 0 ? 0 : K <= 32 ? 1 : K <= 64 ? 2 : K <= 128 ? 4 : 8; }

// Waves per SIMD that the registers are held to: two sets of a tile's rows (one on its way) take 8 per step.
constexpr int kept_waves(int ks1, int ks2) { return ks1 + ks2 > 8 || ks1 == 8 ? 2 : 4; }

constexpr int kept_lds(int M, int ks) {
  return (M + 31) / 32 * 32 * kept_pitch(ks) + kKeptWaves * (int)Patch<bf16_t, 16>::BYTES;
}

// ROWS rows of CHUNKS 16-byte chunks from the wave's patch (128 bytes per row, chunk c of row r at c ^ r) to columns `first` ..
// of their 8-bit rows.
template <int ROWS, int CHUNKS>
__device__ __forceinline__ void leave_bytes(const KeptSeg& s, int64_t N, int64_t r0, int first, int Kp, const char* patch) {
  const int lane = threadIdx.x & 63;
  // rows that leave in one go are joined before the L2 down to 32 bytes (1 M x 96: 84 us past it, 112 through it; in two
  // goes, 1 M x 224: 234 and 185)
  const bool whole = s.ldq % (Kp <= CHUNKS * 16 ? 32 : 64) == 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int c = lane; c < ROWS * CHUNKS; c += 64) {
    const int r = c / CHUNKS, chunk = c % CHUNKS, at = first + chunk * 16;
    const i32x4 v = *reinterpret_cast<const i32x4*>(patch + r * 128 + ((chunk ^ r) & 7) * 16);
    if (r0 + r < N && at < Kp) store_chunk(s.q + (r0 + r) * s.ldq + at, v, whole);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// 16 rows of KS steps in 8 bits: from the operand registers through the wave's patch (2 KiB: 64 columns' results or 128
// columns' bytes) to memory.
template <int KS>
__device__ __forceinline__ void keep_rows(const uint4 (&raw)[KS], const KeptSeg& s, int64_t N, int64_t r0, char* patch) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = (w[j] << 16) & 0x7fffffffu, hi = w[j] & 0x7fff0000u;
      top = lo > top ? lo : top;
      top = hi > top ? hi : top;
    }
  }
  uint32_t o = __shfl_xor(top, 16, 64);
  top = o > top ? o : top;
  o = __shfl_xor(top, 32, 64);
  top = o > top ? o : top;
  const Quant qt = quant_of(top);
  if (g == 0 && r0 + i < N) s.scale[r0 + i] = qt.scale;
  const int Kp = (s.K + 15) & ~15;
  constexpr int PART = KS < 4 ? KS : 4;       // steps that fit the patch: 16 rows x 128 bytes
  constexpr int CHUNKS = PART * 2;            // 16-byte chunks of a row
#pragma unroll
  for (int p = 0; p < KS; p += PART) {
#pragma unroll
    for (int k = 0; k < PART; ++k) {
      const uint32_t w[4] = {raw[p + k].x, raw[p + k].y, raw[p + k].z, raw[p + k].w};
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
      const int chunk = 2 * k + (g >> 1);
      *reinterpret_cast<uint2*>(patch + i * 128 + ((chunk ^ i) & 7) * 16 + (g & 1) * 8) =
          make_uint2(quant_word(v[0], v[1], v[2], v[3], qt), quant_word(v[4], v[5], v[6], v[7], qt));
    }
    leave_bytes<16, CHUNKS>(s, N, r0, p * 32, Kp, patch);
  }
}

template <int KS>
__device__ __forceinline__ void fetch_rows(uint4 (&raw)[KS], const KeptSeg& s, int64_t row, int g) {
  const bf16_t* p = static_cast<const bf16_t*>(s.x) + row * s.ldx;
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int c = 32 * k + 8 * g;   // widths are multiples of 8
    raw[k] = *reinterpret_cast<const uint4*>(p + (c < s.K ? c : 0));
  }
}

template <int KS>
__device__ __forceinline__ void clear_tail(uint4 (&raw)[KS], const KeptSeg& s, int g) {
#pragma unroll
  for (int k = 0; k < KS; ++k)
    if (32 * k + 32 > s.K) {        // uniform
      const uint32_t keep = 32 * k + 8 * g < s.K ? ~0u : 0u;
      raw[k] = make_uint4(raw[k].x & keep, raw[k].y & keep, raw[k].z & keep, raw[k].w & keep);
    }
}

template <int KS1, int KS2>
__global__ void __launch_bounds__(kKeptThreads, kept_waves(KS1, KS2)) k_kept_linear(KeptArgs a) {
  constexpr int KS = KS1 + KS2, PITCH = kept_pitch(KS), N2 = KS2 > 0 ? KS2 : 1;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int m_pad = (a.M + 31) & ~31;
  char* const patch_base = lds + m_pad * PITCH + wave * (int)Patch<bf16_t, 16>::BYTES;
  const Patch<bf16_t, 16> patch{patch_base};

  const int64_t tiles = (a.N + 15) >> 4, step = (int64_t)gridDim.x * kKeptWaves;
  int64_t tile = (int64_t)blockIdx.x * kKeptWaves + wave;
  uint4 raw1[KS1], raw2[N2], next1[KS1], next2[N2];
  auto fetch = [&](int64_t t) __attribute__((always_inline)) {
    const int64_t row = 16 * t + i < a.N ? 16 * t + i : a.N - 1;
    fetch_rows<KS1>(next1, a.a, row, g);
    if constexpr (KS2 > 0) fetch_rows<KS2>(next2, a.b, row, g);
  };
  if (tile < tiles) fetch(tile);

  // weights to LDS: output m of a pair of 16-row tiles t in row 16 t + r with m = 8 (r / 4) + 4 t + r % 4, so that a lane ends
  // with 8 consecutive outputs; zeros behind the widths (the other operand's zeros would not do: 0 * NaN)
  for (int idx = threadIdx.x; idx < m_pad * (KS * 4); idx += kKeptThreads) {
    int pos = idx / (KS * 4), c = idx - pos * (KS * 4);
    if (KS2 == 0 && a.across) {     // neighbours in a row of W
      c = idx / m_pad;
      pos = idx - c * m_pad;
    }
    const int r = pos & 15;
    const int m = (pos & ~31) + 8 * (r >> 2) + 4 * ((pos >> 4) & 1) + (r & 3);
    const bool second = c >= KS1 * 4;
    const int k = (second ? c - KS1 * 4 : c) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (KS2 == 0 && a.across) {
      if (m < a.M && k < a.a.K) {   // widths are multiples of 8
        const bf16_t* w = static_cast<const bf16_t*>(a.w) + (int64_t)k * a.ldw + m;
        uint32_t t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = w[e * a.ldw];
        v = make_uint4(t[0] | t[1] << 16, t[2] | t[3] << 16, t[4] | t[5] << 16, t[6] | t[7] << 16);
      }
    } else if (m < a.M && k < (second ? a.b.K : a.a.K))
      v = *reinterpret_cast<const uint4*>(static_cast<const bf16_t*>(a.w) + (int64_t)m * a.ldw + (second ? a.a.K : 0) + k);
    *reinterpret_cast<uint4*>(lds + pos * PITCH + c * 16) = v;
  }
  __syncthreads();

  for (; tile < tiles; tile += step) {
#pragma unroll
    for (int k = 0; k < KS1; ++k) raw1[k] = next1[k];
    clear_tail<KS1>(raw1, a.a, g);
    if constexpr (KS2 > 0) {
#pragma unroll
      for (int k = 0; k < KS2; ++k) raw2[k] = next2[k];
      clear_tail<KS2>(raw2, a.b, g);
    }
    if (tile + step < tiles) fetch(tile + step);
    const int64_t r0 = 16 * tile;
    for (int b = 0; b < m_pad; b += 32) {
      f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const char* w = lds + (b + i) * PITCH + g * 16;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const bf16x8 x = __builtin_bit_cast(bf16x8, k < KS1 ? raw1[k < KS1 ? k : 0] : raw2[k >= KS1 ? k - KS1 : 0]);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(w + t * 16 * PITCH + k * 64), x, acc[t], 0, 0, 0);
      }
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = acc[e >> 2][e & 3];
        if (a.relu && v[e] <= 0.f) v[e] = 0.f;      // a NaN stays
      }
      patch.put(i, ((b & 32) + 8 * g) / 8, v);
      if (a.bits) {
        uint32_t open = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) open |= (v[e] <= 0.f ? 0u : 1u) << e;
        const int c = b + 8 * g;
        if (r0 + i < a.N) a.bits[(r0 + i) * (m_pad >> 3) + (c >> 3)] = c < a.M ? (uint8_t)open : (uint8_t)0;
      }
      if ((b & 32) || b + 32 >= m_pad) patch.leave(a.y, a.ldy, a.N, r0, b & ~63, a.M, 16);
    }
    if (a.a.q) keep_rows<KS1>(raw1, a.a, a.N, r0, patch_base);
    if constexpr (KS2 > 0) keep_rows<KS2>(raw2, a.b, a.N, r0, patch_base);
  }
}

template <int KS1, int KS2>
int32_t launch_kept(const KeptArgs& a, hipStream_t stream) {
  const int bytes = kept_lds(a.M, KS1 + KS2);
  const int64_t need = (a.N + 16 * kKeptWaves - 1) / (16 * kKeptWaves);
  int per_cu = 160 * 1024 / bytes;
  const int by_regs = kept_waves(KS1, KS2) / 2;
  if (per_cu > by_regs) per_cu = by_regs;
  const int64_t blocks = need < 256 * per_cu ? need : 256 * per_cu;
  if (bytes > 64 * 1024)
    MPNN_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(k_kept_linear<KS1, KS2>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  k_kept_linear<KS1, KS2><<<(unsigned)blocks, kKeptThreads, bytes, stream>>>(a);
  MPNN_LAUNCH_CHECK("k_kept_linear");
  return MPNN_OK;
}

template <int KS1>
int32_t launch_kept1(const KeptArgs& a, hipStream_t stream) {
  switch (kept_steps(a.b.K)) {
    case 0: return launch_kept<KS1, 0>(a, stream);
    case 1: return launch_kept<KS1, 1>(a, stream);
    case 2: return launch_kept<KS1, 2>(a, stream);
    case 4: return launch_kept<KS1, 4>(a, stream);
    default: return launch_kept<KS1, 8>(a, stream);
  }
}

// ------------------------------------------------------------------------------------------------------------ float32
// The layout of v_mfma_f32_32x32x16_bf16: lane (row i, half h) holds columns 16 c + 8 h .. + 7 of chunk c of its row, and of
// the sums 16 outputs of its row.
constexpr int kept_pitch_f32(int ks) { return ks * 192 + 16; }   // three pieces of a weight row, a chunk's pieces side by side
constexpr int kKeptWeightsF32 = 120 * 1024;
// Rows on their way while the ones before are multiplied: as far as the registers go (a step's pieces take 24, rows on their way 16).
constexpr bool kept_ahead_f32(int ks) { return ks <= 4; }

template <int KS>
struct RowsF32 { float v[2 * KS][8]; };

template <int KS>
__device__ __forceinline__ void fetch_rows(RowsF32<KS>& r, const KeptSeg& s, int64_t row, int h) {
  const float* p = static_cast<const float*>(s.x) + row * s.ldx;
#pragma unroll
  for (int k = 0; k < 2 * KS; ++k)
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const int c = 16 * k + 8 * h + e;     // widths are multiples of 4
      const float4 t = *reinterpret_cast<const float4*>(p + (c < s.K ? c : 0));
      r.v[k][e] = t.x; r.v[k][e + 1] = t.y; r.v[k][e + 2] = t.z; r.v[k][e + 3] = t.w;
    }
}

template <int KS>
__device__ __forceinline__ void clear_tail(RowsF32<KS>& r, const KeptSeg& s, int h) {
#pragma unroll
  for (int k = 0; k < 2 * KS; ++k)
    if (16 * k + 16 > s.K)        // uniform
#pragma unroll
      for (int e = 0; e < 8; ++e) r.v[k][e] = 16 * k + 8 * h + e < s.K ? r.v[k][e] : 0.f;
}

template <int KS>
__device__ __forceinline__ void keep_rows(const RowsF32<KS>& x, const KeptSeg& s, int64_t N, int64_t r0, char* patch) {
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 2 * KS; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = magnitude_bits(x.v[k][e]) > top ? magnitude_bits(x.v[k][e]) : top;
  const uint32_t o = __shfl_xor(top, 32, 64);
  top = o > top ? o : top;
  const Quant qt = quant_of(top);
  if (h == 0 && r0 + i < N) s.scale[r0 + i] = qt.scale;
  const int Kp = (s.K + 15) & ~15;
  constexpr int CHUNKS = KS < 4 ? 2 * KS : 8;   // chunks that fit the patch: 32 rows x 128 bytes
#pragma unroll
  for (int p = 0; p < 2 * KS; p += CHUNKS) {
#pragma unroll
    for (int k = 0; k < CHUNKS; ++k) {
      const float* v = x.v[p + k];
      *reinterpret_cast<uint2*>(patch + i * 128 + ((k ^ i) & 7) * 16 + 8 * h) =
          make_uint2(quant_word(v[0], v[1], v[2], v[3], qt), quant_word(v[4], v[5], v[6], v[7], qt));
    }
    leave_bytes<32, CHUNKS>(s, N, r0, p * 16, Kp, patch);
  }
}

// The three pieces of 8 values: each the upper half of what is left.
__device__ __forceinline__ void cut(const float (&v)[8], bf16x8 (&out)[3]) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(__float_as_uint(r[2 * j + 1]), __float_as_uint(r[2 * j]), 0x07060302u);
    out[p] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    if (p < 2)
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] -= __uint_as_float(__float_as_uint(r[e]) & 0xffff0000u);
  }
}

template <int KS1, int KS2>
__global__ void __launch_bounds__(kKeptThreads, 2) k_kept_linear_f32(KeptArgs a, int slice) {
  constexpr int KS = KS1 + KS2, PITCH = kept_pitch_f32(KS), N2 = KS2 > 0 ? KS2 : 1;
  constexpr bool AHEAD = kept_ahead_f32(KS);
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 31, h = lane >> 5;
  const int m_begin = (int)blockIdx.y * slice;
  const int m_count = a.M - m_begin < slice ? a.M - m_begin : slice, m_pad = (m_count + 31) & ~31;
  const int bits_pitch = ((a.M + 31) & ~31) >> 3;
  char* const patch_base = lds + m_pad * PITCH + wave * (int)Patch<float, 32, 32>::BYTES;
  const Patch<float, 32, 32> patch{patch_base};

  const int64_t tiles = (a.N + 31) >> 5, step = (int64_t)gridDim.x * kKeptWaves;
  int64_t tile = (int64_t)blockIdx.x * kKeptWaves + wave;
  RowsF32<KS1> next1;
  RowsF32<N2> next2;
  auto row_of = [&](int64_t t) __attribute__((always_inline)) { return 32 * t + i < a.N ? 32 * t + i : a.N - 1; };
  auto half = [&]() __attribute__((always_inline)) {
    int from = h;
    asm volatile("" : "+v"(from));   // the column offsets are formed anew per tile: kept, they would not fit the registers
    return from;
  };
  auto fetch = [&](int64_t t) __attribute__((always_inline)) {
    fetch_rows<KS1>(next1, a.a, row_of(t), half());
    if constexpr (KS2 > 0) fetch_rows<KS2>(next2, a.b, row_of(t), half());
  };
  if constexpr (AHEAD) fetch(tile);

  // weights to LDS, cut into pieces: output m of 32 in row 8 (m % 16 / 4) + 4 (m / 16) + m % 4, so that a lane ends with 16
  // consecutive outputs; zeros behind the widths
  for (int idx = threadIdx.x; idx < m_pad * (KS * 4); idx += kKeptThreads) {
    int pos = idx / (KS * 4), c = idx - pos * (KS * 4);
    const bool across = KS2 == 0 && a.across;
    if (across) {                   // neighbours in a row of W
      c = idx / m_pad;
      pos = idx - c * m_pad;
    }
    const int k = c >> 1, ch = c & 1;
    const int m = m_begin + (pos & ~31) + 16 * ((pos >> 2) & 1) + 4 * ((pos >> 3) & 3) + (pos & 3);
    const bool second = k >= 2 * KS1;
    const int col = (second ? k - 2 * KS1 : k) * 16 + 8 * ch, K = second ? a.b.K : a.a.K;
    const int64_t along = across ? a.ldw : 1;      // from one contraction index to the next
    const float* w = static_cast<const float*>(a.w) + (m < a.M ? m : 0) * (across ? 1 : a.ldw) + (second ? a.a.K : 0);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = m < a.M && col + e < K ? w[(col + e) * along] : 0.f;
    bf16x8 p[3];
    cut(v, p);
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x8*>(lds + pos * PITCH + k * 96 + q * 32 + ch * 16) = p[q];
  }
  __syncthreads();

  for (; tile < tiles; tile += step) {
    const int64_t r0 = 32 * tile;
    bf16x8 x[2 * KS][3];
    if constexpr (!AHEAD) fetch_rows<KS1>(next1, a.a, row_of(tile), half());
    clear_tail<KS1>(next1, a.a, h);
    if (blockIdx.y == 0 && a.a.q) keep_rows<KS1>(next1, a.a, a.N, r0, patch_base);
#pragma unroll
    for (int k = 0; k < 2 * KS1; ++k) cut(next1.v[k], x[k]);
    if constexpr (KS2 > 0) {
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!AHEAD) fetch_rows<KS2>(next2, a.b, row_of(tile), half());
      clear_tail<KS2>(next2, a.b, h);
      if (blockIdx.y == 0) keep_rows<KS2>(next2, a.b, a.N, r0, patch_base);
#pragma unroll
      for (int k = 0; k < 2 * KS2; ++k) cut(next2.v[k], x[2 * KS1 + k]);
    }
    __builtin_amdgcn_sched_barrier(0);    // the rows on their way take the registers of those just cut
    if constexpr (AHEAD) fetch(tile + step);   // behind the last tile: the last row, for nothing
    for (int b = 0; b < m_pad; b += 32) {
      f32x16 acc;
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = 0.f;
      const char* w = lds + (b + i) * PITCH + h * 16;
      bf16x8 p[2][3];     // a chunk's pieces are read while the one before is multiplied
      auto read = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 3; ++q) p[k & 1][q] = *reinterpret_cast<const bf16x8*>(w + k * 96 + q * 32);
      };
      read(0);
#pragma unroll
      for (int k = 0; k < 2 * KS; ++k) {
        if (k + 1 < 2 * KS) read(k + 1);
        // pieces (weight, x), smallest products first, as k_gemm_nt adds them
        constexpr int PW[6] = {0, 2, 1, 0, 1, 0}, PX[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
        for (int q = 0; q < 6; ++q) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[k & 1][PW[q]], x[k][PX[q]], acc, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);    // further ahead they would not fit the registers
      }
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        v[e] = acc[e];
        if (a.relu && v[e] <= 0.f) v[e] = 0.f;
      }
      const int c = m_begin + b + 16 * h;
      if (a.bits) {
        uint32_t open = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) open |= (v[e] <= 0.f || c + e >= a.M ? 0u : 1u) << e;
        if (r0 + i < a.N) *reinterpret_cast<uint16_t*>(a.bits + (r0 + i) * bits_pitch + (c >> 3)) = (uint16_t)open;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) patch.put(i, 4 * h + e, {v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]});
      patch.leave(a.y, a.ldy, a.N, r0, m_begin + b, m_begin + m_count, a.width);
    }
  }
}

template <int KS1, int KS2>
int32_t launch_kept_f32(const KeptArgs& a, int slices, hipStream_t stream) {
  constexpr int KS = KS1 + KS2, rows = 32 * kKeptWaves;
  const int m32 = (a.M + 31) / 32, per = (m32 + slices - 1) / slices;
  const int bytes = per * 32 * kept_pitch_f32(KS) + kKeptWaves * (int)Patch<float, 32, 32>::BYTES;
  const int64_t need = (a.N + rows - 1) / rows, most = 256 / slices;
  if (bytes > 64 * 1024)
    MPNN_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(k_kept_linear_f32<KS1, KS2>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  k_kept_linear_f32<KS1, KS2><<<dim3((unsigned)(need < most ? need : most), slices), kKeptThreads, bytes, stream>>>(a, per * 32);
  MPNN_LAUNCH_CHECK("k_kept_linear_f32");
  return MPNN_OK;
}

// Slices of the outputs whose weights fit the LDS: 1 or 2, 0 if they do not.  Eight steps fill the registers and some spill:
// in one slice they are still ahead of the separate passes (1 M rows, 128 + 128 -> 64: 430 us and 568; 256 -> 64: 447 and
// 526), in two they are not (128 + 128 -> 128: 757 and 748; 256 -> 128: 771 and 668).
int kept_slices_f32(int K, int K2, int M) {
  const int ks = kept_steps(K) + kept_steps(K2);
  if (ks > 8 || ((K | K2) & 3)) return 0;
  const int m32 = (M + 31) / 32;
  for (int s = 1; s <= (ks > 6 ? 1 : 2); ++s)
    if ((m32 + s - 1) / s * 32 * kept_pitch_f32(ks) <= kKeptWeightsF32) return s;
  return 0;
}

template <int KS1>
int32_t launch_kept1_f32(const KeptArgs& a, hipStream_t stream) {
  const int slices = kept_slices_f32(a.a.K, a.b.K, a.M);
  switch (kept_steps(a.b.K)) {
    case 0: return launch_kept_f32<KS1, 0>(a, slices, stream);
    case 1: if constexpr (KS1 < 8) return launch_kept_f32<KS1, 1>(a, slices, stream); break;
    case 2: if constexpr (KS1 < 8) return launch_kept_f32<KS1, 2>(a, slices, stream); break;
    case 4: if constexpr (KS1 < 8) return launch_kept_f32<KS1, 4>(a, slices, stream); break;
  }
  return fail(MPNN_E_INVALID, "mpnn_kept_linear: no kernel for K=%d K2=%d", a.a.K, a.b.K);
}

int32_t launch_kept_any(KeptArgs& a, int32_t dtype, hipStream_t stream) {
  const int steps = kept_steps(a.a.K);
  if (dtype == MPNN_F32) {
    a.width = store_width(a.y, a.ldy * 4);
    switch (steps) {
      case 1: return launch_kept1_f32<1>(a, stream);
      case 2: return launch_kept1_f32<2>(a, stream);
      case 4: return launch_kept1_f32<4>(a, stream);
      default: return launch_kept1_f32<8>(a, stream);
    }
  }
  switch (steps) {
    case 1: return launch_kept1<1>(a, stream);
    case 2: return launch_kept1<2>(a, stream);
    case 4: return launch_kept1<4>(a, stream);
    default: return launch_kept1<8>(a, stream);
  }
}

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int32_t mpnn_kept_linear_fits(int32_t K, int32_t K2, int32_t M, int32_t dtype) {
  if (K < 1 || K2 < 0 || M < 1 || K > 256 || K2 > 256 || M > 4096) return 0;
  if (dtype == MPNN_F32) {
    const char* form = getenv("MPNN_GEMM");      // "f32" asks for the products on the float32 instructions
    return !(form && (form[0] == 'f' || form[0] == 'F')) && kept_slices_f32(K, K2, M) > 0;
  }
  if (dtype != MPNN_BF16 || ((K | K2 | M) & 7)) return 0;
  return (M + 31) / 32 * 32 * kept_pitch(kept_steps(K) + kept_steps(K2)) <= kKeptWeights;
}

int32_t mpnn_kept_linear(const void* X, int64_t ldx, int32_t K, void* Q, int64_t ldq, float* scale, const void* X2,
                         int64_t ldx2, int32_t K2, void* Q2, int64_t ldq2, float* scale2, const void* W, int64_t ldw,
                         void* Y, int64_t ldy, void* bits, int64_t N, int32_t M, int32_t relu, int32_t dtype,
                         mpnn_stream_t stream) {
  if (N < 0 || !mpnn_kept_linear_fits(K, K2, M, dtype))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear: N=%lld K=%d K2=%d M=%d dtype %d (see mpnn_kept_linear_fits)", (long long)N, K, K2, M, dtype);
  if (ldx < K || ldw < K + K2 || ldy < M || ldq < (K + 15) / 16 * 16 || (K2 > 0 && (ldx2 < K2 || ldq2 < (K2 + 15) / 16 * 16)))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear: leading dimension too small");
  if (N == 0) return MPNN_OK;
  if (!X || !Q || !scale || !W || !Y || (K2 > 0 && (!X2 || !Q2 || !scale2)))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear: null pointer argument");
  const uintptr_t inputs = (uintptr_t)X | (K2 > 0 ? (uintptr_t)X2 : 0), rows8 = (uintptr_t)Q | (K2 > 0 ? (uintptr_t)Q2 : 0);
  if ((rows8 & 15) || (ldq & 15) || (K2 > 0 && (ldq2 & 15)))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear: 8-bit rows must be 16-byte aligned");
  const bool bf16 = dtype == MPNN_BF16;
  if (!bf16 && ((inputs & 15) || ldx % 4 || (K2 > 0 && ldx2 % 4)))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear: float32 inputs must be 16-byte aligned with row strides that keep them so");
  if (bf16 && (((inputs | (uintptr_t)W | (uintptr_t)Y) & 15) || ((ldx | ldw | ldy) & 7) || (K2 > 0 && (ldx2 & 7))))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear: bfloat16 operands must be 16-byte aligned with row strides that keep them so");
  KeptArgs a;
  memset(&a, 0, sizeof a);
  a.a = KeptSeg{X, ldx, static_cast<int8_t*>(Q), ldq, scale, K};
  if (K2 > 0) a.b = KeptSeg{X2, ldx2, static_cast<int8_t*>(Q2), ldq2, scale2, K2};
  a.w = W; a.ldw = ldw;
  a.y = Y; a.ldy = ldy;
  a.bits = static_cast<uint8_t*>(bits);
  a.N = N; a.M = M; a.relu = relu;
  return launch_kept_any(a, dtype, stream);
}

int32_t mpnn_gemm_nn(const void* X, int64_t ldx, const void* W, int64_t ldw, void* Y, int64_t ldy, int64_t N, int32_t K,
                     int32_t M, int32_t dtype, mpnn_stream_t stream) {
  if (N < 0 || !mpnn_kept_linear_fits(K, 0, M, dtype))
    return fail(MPNN_E_INVALID, "mpnn_gemm_nn: N=%lld K=%d M=%d dtype %d (see mpnn_kept_linear_fits)", (long long)N, K, M, dtype);
  if (ldx < K || ldw < M || ldy < M) return fail(MPNN_E_INVALID, "mpnn_gemm_nn: leading dimension too small");
  if (N == 0) return MPNN_OK;
  if (!X || !W || !Y) return fail(MPNN_E_INVALID, "mpnn_gemm_nn: null pointer argument");
  const int vec = dtype == MPNN_BF16 ? 8 : 4;
  if (((uintptr_t)X & 15) || ldx % vec || (dtype == MPNN_BF16 && (((uintptr_t)Y & 15) || ldy % vec)))
    return fail(MPNN_E_INVALID, "mpnn_gemm_nn: rows must be 16-byte aligned with strides that keep them so");
  KeptArgs a;
  memset(&a, 0, sizeof a);
  a.a = KeptSeg{X, ldx, nullptr, 0, nullptr, K};
  a.w = W; a.ldw = ldw;
  a.y = Y; a.ldy = ldy;
  a.N = N; a.M = M; a.across = 1;
  return launch_kept_any(a, dtype, stream);
}

}  // extern "C"
