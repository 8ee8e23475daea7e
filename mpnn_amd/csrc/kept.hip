// A bfloat16 Linear call whose inputs wait for the backward in 8 bits (rows8.hip), in one pass over them:
//
//   y = act(x W1^T [+ x2 W2^T])     and, from the same registers,     q, scale [, q2, scale2] = rows of x [, x2] in 8 bits,
//   bits = one bit per output, set where the relu is open
//
// (models/layers.py:104 and :140 without the concatenation).  Products on v_mfma_f32_16x16x32_bf16, float32 sums, one
// rounding.  The weights, [W1 | W2] of up to 120 KiB, stay in LDS; a wave takes 16 rows at a time as they lie in memory (lane
// (row i, group g) holds columns 32 s + 8 g .. + 7 of every step s, which is the operand's own order), multiplies them
// with every 32 outputs in turn and takes them to 8 bits from the same registers.  Results, 8-bit rows and bits leave
// through LDS as whole row segments.
//
// Bound: memory.  One pass reads x and x2 once and writes y, q, q2; a product, two quantising passes and a pass over y read
// them twice: 4 M rows, 128 + 128 -> 128, in 0.90 ms (4.5 TB/s; a copy reaches 4.9) instead of 0.64 + 0.60 + 0.24 ms.
#include "common.h"
#include "rows8.h"

namespace mpnn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kKeptThreads = 512;
constexpr int kKeptWaves = kKeptThreads / 64;
constexpr int kKeptWeights = 120 * 1024;

struct KeptSeg {
  const bf16_t* x; int64_t ldx;
  int8_t* q; int64_t ldq;
  float* scale;
  int K;
};
struct KeptArgs {
  KeptSeg a, b;                     // b.K = 0: one input
  const bf16_t* w; int64_t ldw;     // [M, K + K2]
  bf16_t* y; int64_t ldy;
  uint8_t* bits;                    // optional
  int64_t N;
  int M, relu;
};

constexpr int kept_pitch(int ks) { return ks * 64 + 16; }   // bytes of a weight row in LDS: 16 more spread eight rows over the banks

// 32-column steps of a width, as the kernels come: 1, 2, 4 or 8
constexpr int kept_steps(int K) { return K <= 0 ? 0 : K <= 32 ? 1 : K <= 64 ? 2 : K <= 128 ? 4 : 8; }

// Waves per SIMD that the registers are held to: two sets of a tile's rows (one on its way) take 8 per step.
constexpr int kept_waves(int ks1, int ks2) { return ks1 + ks2 > 8 || ks1 == 8 ? 2 : 4; }

constexpr int kept_lds(int M, int ks) {
  return (M + 31) / 32 * 32 * kept_pitch(ks) + kKeptWaves * (int)Patch<bf16_t, 16>::BYTES;
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
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = lane; c < 16 * CHUNKS; c += 64) {
      const int r = c / CHUNKS, chunk = c % CHUNKS, at = p * 32 + chunk * 16;
      const i32x4 v = *reinterpret_cast<const i32x4*>(patch + r * 128 + ((chunk ^ r) & 7) * 16);
      if (r0 + r < N && at < Kp) __builtin_nontemporal_store(v, reinterpret_cast<i32x4*>(s.q + (r0 + r) * s.ldq + at));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int KS>
__device__ __forceinline__ void fetch_rows(uint4 (&raw)[KS], const KeptSeg& s, int64_t row, int g) {
  const bf16_t* p = s.x + row * s.ldx;
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
    const int pos = idx / (KS * 4), c = idx - pos * (KS * 4), r = pos & 15;
    const int m = (pos & ~31) + 8 * (r >> 2) + 4 * ((pos >> 4) & 1) + (r & 3);
    const bool second = c >= KS1 * 4;
    const int k = (second ? c - KS1 * 4 : c) * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (m < a.M && k < (second ? a.b.K : a.a.K))
      v = *reinterpret_cast<const uint4*>(a.w + (int64_t)m * a.ldw + (second ? a.a.K : 0) + k);
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
      if ((b & 32) || b + 32 >= m_pad) patch.leave(a.y, a.ldy, a.N, r0, b & ~63, a.M, true);
    }
    keep_rows<KS1>(raw1, a.a, a.N, r0, patch_base);
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

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int32_t mpnn_kept_linear_fits(int32_t K, int32_t K2, int32_t M) {
  if (K < 8 || K2 < 0 || M < 8 || K > 256 || K2 > 256 || M > 4096 || ((K | K2 | M) & 7)) return 0;
  return (M + 31) / 32 * 32 * kept_pitch(kept_steps(K) + kept_steps(K2)) <= kKeptWeights;
}

int32_t mpnn_kept_linear_bf16(const void* X, int64_t ldx, int32_t K, void* Q, int64_t ldq, float* scale, const void* X2,
                              int64_t ldx2, int32_t K2, void* Q2, int64_t ldq2, float* scale2, const void* W, int64_t ldw,
                              void* Y, int64_t ldy, void* bits, int64_t N, int32_t M, int32_t relu, mpnn_stream_t stream) {
  if (N < 0 || !mpnn_kept_linear_fits(K, K2, M))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear_bf16: N=%lld K=%d K2=%d M=%d (see mpnn_kept_linear_fits)", (long long)N, K, K2, M);
  if (ldx < K || ldw < K + K2 || ldy < M || ldq < (K + 15) / 16 * 16 || (K2 > 0 && (ldx2 < K2 || ldq2 < (K2 + 15) / 16 * 16)))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear_bf16: leading dimension too small");
  if (N == 0) return MPNN_OK;
  if (!X || !Q || !scale || !W || !Y || (K2 > 0 && (!X2 || !Q2 || !scale2)))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear_bf16: null pointer argument");
  const uintptr_t ptrs = (uintptr_t)X | (uintptr_t)Q | (uintptr_t)W | (uintptr_t)Y | (K2 > 0 ? (uintptr_t)X2 | (uintptr_t)Q2 : 0);
  if ((ptrs & 15) || ((ldx | ldw | ldy) & 7) || (ldq & 15) || (K2 > 0 && ((ldx2 & 7) || (ldq2 & 15))))
    return fail(MPNN_E_INVALID, "mpnn_kept_linear_bf16: operands must be 16-byte aligned with row strides that keep them so");
  KeptArgs a;
  memset(&a, 0, sizeof a);
  a.a = KeptSeg{static_cast<const bf16_t*>(X), ldx, static_cast<int8_t*>(Q), ldq, scale, K};
  if (K2 > 0) a.b = KeptSeg{static_cast<const bf16_t*>(X2), ldx2, static_cast<int8_t*>(Q2), ldq2, scale2, K2};
  a.w = static_cast<const bf16_t*>(W); a.ldw = ldw;
  a.y = static_cast<bf16_t*>(Y); a.ldy = ldy;
  a.bits = static_cast<uint8_t*>(bits);
  a.N = N; a.M = M; a.relu = relu;
  switch (kept_steps(K)) {
    case 1: return launch_kept1<1>(a, stream);
    case 2: return launch_kept1<2>(a, stream);
    case 4: return launch_kept1<4>(a, stream);
    default: return launch_kept1<8>(a, stream);
  }
}

}  // extern "C"
