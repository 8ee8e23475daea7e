// Rows held in 8 bits (no counterpart in the reference): a row x of K values is kept as whole numbers q in [-127, 127]
// and one float32 scale,
//
//   top = max|x|,  scale = top / 127,  inv = 127 / top   (each one float32 rounding),  q = x * inv to the nearest, ties to even
//
// x * inv is rounded once, to the whole number: fma(x, inv, 1.5 * 2^23) has whole numbers as its last place, so the
// exact product falls to its own side of a border.  A row whose top is below 2^-100 counts as zeros (scale 0); a row
// that holds an infinity or a NaN has scale NaN and zeros: it stands for NaN everywhere.
//
// Rows of q are `ldq` bytes apart, a multiple of 16 of at least K; the bytes behind column K are written as zeros.
//
// Bound: memory, one pass: a row is read once into the registers of LPR lanes, its top found by shuffles, and its bytes
// written from there.
#include "common.h"
#include "rows8.h"

namespace mpnn {
namespace {

constexpr int kRows8MaxK = 8192;
constexpr int kBitsMaxM = 1 << 30;   // a row's columns and their padding count in 32 bits

struct QuantArgs {
  const void* x;
  int64_t ldx;
  int8_t* q;
  int64_t ldq;
  float* scale;
  int64_t N;
  int K, Kp;   // Kp: columns written, K rounded up to 16
};

template <typename T, int VEC, int NV, int LPR>
__global__ void __launch_bounds__(kBlock) k_quantize_rows(QuantArgs a) {
  __shared__ uint32_t red[2][4];
  const int lane = threadIdx.x % LPR;
  const int64_t step = (int64_t)gridDim.x * (kBlock / LPR);
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * (kBlock / LPR) + threadIdx.x / LPR; row < a.N; row += step, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[NV][VEC];
    // magnitudes compare as unsigned integers; infinities and NaN come out above every finite one
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + lane) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[i][k] = 0.f;
      if (c < a.K) RowIO<T, VEC>::load(x + c, v[i]);   // K is a multiple of VEC on the vector path
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < VEC; ++k) top = magnitude_bits(v[i][k]) > top ? magnitude_bits(v[i][k]) : top;
    constexpr int W = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) {
      const uint32_t o = __shfl_xor(top, off, 64);
      top = o > top ? o : top;
    }
    if constexpr (LPR > 64) {   // the block's row: four waves meet, two sets in turn so that one barrier is enough
      if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 4; ++w) top = red[turn][w] > top ? red[turn][w] : top;
    }
    const Quant qt = quant_of(top);
    int8_t* q = a.q + row * a.ldq;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LPR + lane) * VEC;
      if (c >= a.Kp) continue;
      if constexpr (VEC == 1) {
        q[c] = (int8_t)(quant_bits(v[i][0], qt.inv) & qt.keep);
      } else {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int k = 0; k < VEC; k += 4)
          w[k / 4] = quant_word(v[i][k], v[i][k + 1], v[i][k + 2], v[i][k + 3], qt);
        if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(q + c) = w[0];
        else *reinterpret_cast<uint2*>(q + c) = make_uint2(w[0], w[1]);
      }
    }
    if (lane == 0) a.scale[row] = qt.scale;
  }
}

template <typename T, int VEC>
bool launch_quantize(const QuantArgs& a, hipStream_t stream) {
  const int nvec = (a.Kp + VEC - 1) / VEC;
  int lpr, nv;
  if (nvec <= 256) {
    lpr = 8;
    while (lpr < nvec && lpr < 64) lpr *= 2;
    nv = 1;
    while (nv * lpr < nvec) nv *= 2;
  } else {
    lpr = 256;
    nv = 2;
    while (nv * lpr < nvec) nv *= 2;
  }
  int64_t blocks = (a.N + kBlock / lpr - 1) / (kBlock / lpr);
  if (blocks > kMaxBlocks) blocks = kMaxBlocks;
#define MPNN_QUANT(NV, LPR) \
  if (nv == NV && lpr == LPR) { k_quantize_rows<T, VEC, NV, LPR><<<(int)blocks, kBlock, 0, stream>>>(a); return true; }
  MPNN_QUANT(1, 8)
  MPNN_QUANT(1, 16)
  MPNN_QUANT(1, 32)
  MPNN_QUANT(1, 64)
  MPNN_QUANT(2, 64)
  MPNN_QUANT(4, 64)
  MPNN_QUANT(2, 256)
  MPNN_QUANT(4, 256)
  if constexpr (VEC < 8) { MPNN_QUANT(8, 256) }
  if constexpr (VEC == 1) { MPNN_QUANT(16, 256) MPNN_QUANT(32, 256) }
#undef MPNN_QUANT
  return false;
}

// bits[n][b], b < 4 ceil(M / 32): bit i of byte b is the relu of column 8 b + i open: not y <= 0 (NaN counts as open).
// One thread per byte.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kBlock) k_relu_bits(const T* __restrict__ y, int64_t ldy, int64_t N, int M, int pitch,
                                                      uint8_t* __restrict__ bits) {
  const int64_t total = N * pitch;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (int64_t)gridDim.x * kBlock) {
    const int64_t row = i / pitch;
    const int c = (int)(i - row * pitch) * 8;
    const T* p = y + row * ldy + c;
    uint32_t b = 0;
    if (WIDE && c < M) {
      float v[8];
      if constexpr (sizeof(T) == 2) RowIO<T, 8>::load(p, v);
      else {
        float lo[4], hi[4];
        RowIO<T, 4>::load(p, lo);
        RowIO<T, 4>::load(p + 4, hi);
#pragma unroll
        for (int k = 0; k < 4; ++k) { v[k] = lo[k]; v[4 + k] = hi[k]; }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) b |= (v[k] <= 0.f ? 0u : 1u) << k;
    } else {
      for (int k = 0; k < 8 && c + k < M; ++k) b |= (scalar_to_f32(p[k]) <= 0.f ? 0u : 1u) << k;
    }
    bits[i] = (uint8_t)b;
  }
}

// out[n][m] = g[n][m] where bit m of row n's bits is set, zero elsewhere: 8 columns, one byte of bits, per thread.  WIDE: 16-byte
// accesses.  Bound by memory, one pass: 4 M rows of 128 in 435 us (bfloat16, 4.9 TB/s) and 815 us (float32, 5.1); other widths value
// by value, 1 M rows of 100 in bfloat16 in 245 us.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kBlock) k_open_entries(const T* __restrict__ g, int64_t ldg, int64_t N, int M, const uint8_t* __restrict__ bits,
                                                         int pitch, T* __restrict__ out, int64_t ldo) {
  const int per = (M + 7) / 8;
  const int64_t total = N * per;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < total; i += (int64_t)gridDim.x * kBlock) {
    const int64_t row = i / per;
    const int b = (int)(i - row * per);
    const uint32_t open = bits[row * pitch + b];
    const T* p = g + row * ldg + 8 * b;
    T* q = out + row * ldo + 8 * b;
    if constexpr (WIDE) {
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int h = 0; h < 8; h += V) {
        uint4 t = *reinterpret_cast<const uint4*>(p + h);
        uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) {
            w[k] = (open >> (h + k)) & 1u ? w[k] : 0u;
          } else {
            w[k] &= ((open >> (2 * k)) & 1u ? 0x0000ffffu : 0u) | ((open >> (2 * k + 1)) & 1u ? 0xffff0000u : 0u);
          }
        }
        *reinterpret_cast<uint4*>(q + h) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
      for (int k = 0; k < 8 && 8 * b + k < M; ++k) q[k] = (open >> k) & 1u ? p[k] : (T)0;
    }
  }
}

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int32_t mpnn_quantize_rows(const void* x, int64_t ldx, int32_t dtype, int64_t N, int32_t K, void* q, int64_t ldq,
                           float* scale, mpnn_stream_t stream) {
  if (dtype != MPNN_F32 && dtype != MPNN_BF16) return fail(MPNN_E_INVALID, "mpnn_quantize_rows: dtype %d", dtype);
  if (N < 0 || K < 1 || K > kRows8MaxK)
    return fail(MPNN_E_INVALID, "mpnn_quantize_rows: N=%lld K=%d (rows of 1 to %d columns)", (long long)N, K, kRows8MaxK);
  const int Kp = (K + 15) / 16 * 16;
  if (ldx < K || ldq < Kp || (ldq & 15)) return fail(MPNN_E_INVALID, "mpnn_quantize_rows: ldx=%lld ldq=%lld for K=%d", (long long)ldx, (long long)ldq, K);
  if (N == 0) return MPNN_OK;
  if (!x || !q || !scale) return fail(MPNN_E_INVALID, "mpnn_quantize_rows: null pointer argument");
  if ((uintptr_t)q & 15) return fail(MPNN_E_INVALID, "mpnn_quantize_rows: q must be 16-byte aligned");
  const QuantArgs a{x, ldx, static_cast<int8_t*>(q), ldq, scale, N, K, Kp};
  // the widest vectors that width, address and stride allow, one column per lane and step otherwise (1 M bfloat16 rows of
  // 100: 74 us in vectors of 4, 171 by columns)
  const bool bf16 = dtype == MPNN_BF16;
  auto whole = [&](int v) { return K % v == 0 && ldx % v == 0 && (uintptr_t)x % (v * (bf16 ? 2 : 4)) == 0; };
  bool known;
  if (!bf16) known = whole(4) ? launch_quantize<float, 4>(a, stream) : launch_quantize<float, 1>(a, stream);
  else if (whole(8)) known = launch_quantize<bf16_t, 8>(a, stream);
  else known = whole(4) ? launch_quantize<bf16_t, 4>(a, stream) : launch_quantize<bf16_t, 1>(a, stream);
  if (!known) return fail(MPNN_E_INVALID, "mpnn_quantize_rows: no kernel for K=%d", K);
  MPNN_LAUNCH_CHECK("k_quantize_rows");
  return MPNN_OK;
}

int32_t mpnn_relu_bits(const void* y, int64_t ldy, int32_t dtype, int64_t N, int32_t M, void* bits, mpnn_stream_t stream) {
  if (dtype != MPNN_F32 && dtype != MPNN_BF16) return fail(MPNN_E_INVALID, "mpnn_relu_bits: dtype %d", dtype);
  if (N < 0 || M < 1 || M > kBitsMaxM || ldy < M) return fail(MPNN_E_INVALID, "mpnn_relu_bits: N=%lld M=%d ldy=%lld", (long long)N, M, (long long)ldy);
  if (N == 0) return MPNN_OK;
  if (!y || !bits) return fail(MPNN_E_INVALID, "mpnn_relu_bits: null pointer argument");
  const int pitch = (M + 31) / 32 * 4;
  const bool wide = M % 8 == 0 && ((uintptr_t)y & 15) == 0 && ldy % (dtype == MPNN_BF16 ? 8 : 4) == 0;
  int64_t blocks = (N * pitch + kBlock - 1) / kBlock;
  if (blocks > 4 * kMaxBlocks) blocks = 4 * kMaxBlocks;
  uint8_t* b = static_cast<uint8_t*>(bits);
  if (dtype == MPNN_BF16) {
    if (wide) k_relu_bits<bf16_t, true><<<(int)blocks, kBlock, 0, stream>>>((const bf16_t*)y, ldy, N, M, pitch, b);
    else k_relu_bits<bf16_t, false><<<(int)blocks, kBlock, 0, stream>>>((const bf16_t*)y, ldy, N, M, pitch, b);
  } else {
    if (wide) k_relu_bits<float, true><<<(int)blocks, kBlock, 0, stream>>>((const float*)y, ldy, N, M, pitch, b);
    else k_relu_bits<float, false><<<(int)blocks, kBlock, 0, stream>>>((const float*)y, ldy, N, M, pitch, b);
  }
  MPNN_LAUNCH_CHECK("k_relu_bits");
  return MPNN_OK;
}

int32_t mpnn_open_entries(const void* g, int64_t ldg, int32_t dtype, const void* bits, void* out, int64_t ldo, int64_t N, int32_t M,
                          mpnn_stream_t stream) {
  if (dtype != MPNN_F32 && dtype != MPNN_BF16) return fail(MPNN_E_INVALID, "mpnn_open_entries: dtype %d", dtype);
  if (N < 0 || M < 1 || M > kBitsMaxM || ldg < M || ldo < M)
    return fail(MPNN_E_INVALID, "mpnn_open_entries: N=%lld M=%d ldg=%lld ldo=%lld", (long long)N, M, (long long)ldg, (long long)ldo);
  if (N == 0) return MPNN_OK;
  if (!g || !bits || !out) return fail(MPNN_E_INVALID, "mpnn_open_entries: null pointer argument");
  const int pitch = (M + 31) / 32 * 4;
  const int vec = dtype == MPNN_BF16 ? 8 : 4;
  const bool wide = M % 8 == 0 && (((uintptr_t)g | (uintptr_t)out) & 15) == 0 && ldg % vec == 0 && ldo % vec == 0;
  int64_t blocks = (N * ((M + 7) / 8) + kBlock - 1) / kBlock;
  if (blocks > 4 * kMaxBlocks) blocks = 4 * kMaxBlocks;
  auto launch = [&](auto kernel, auto t) {
    typedef decltype(t) T;
    kernel<<<(int)blocks, kBlock, 0, stream>>>(static_cast<const T*>(g), ldg, N, M, static_cast<const uint8_t*>(bits), pitch,
                                               static_cast<T*>(out), ldo);
  };
  if (dtype == MPNN_BF16) wide ? launch(k_open_entries<bf16_t, true>, bf16_t()) : launch(k_open_entries<bf16_t, false>, bf16_t());
  else wide ? launch(k_open_entries<float, true>, float()) : launch(k_open_entries<float, false>, float());
  MPNN_LAUNCH_CHECK("k_open_entries");
  return MPNN_OK;
}

}  // extern "C"
