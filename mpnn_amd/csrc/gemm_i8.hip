// Product of 8-bit rows with 8-bit weights (rows8.hip holds the format):
//
//   y[n, m] = act( (sum_k xq[n, k] * wq[m, k]) * (xs[n] * ws[m]) + bias[m] )
//
// the forward of a Linear call (models/layers.py:104,140, models/mpnn.py:101) of a trained model, with one scale per
// row of x and one per output channel.  The sum is exact (32-bit integers: 127 * 127 * K stays below 2^31 for
// K <= 8192), the scales are applied in float32 and the result is rounded once to the output type.
#include "common.h"
#include "rowio.h"

namespace mpnn {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

constexpr int kI8MaxK = 8192;

struct I8Args {
  const int8_t* x; int64_t ldx;
  const float* xs;
  const int8_t* w; int64_t ldw;
  const float* ws;
  const void* bias;
  void* y; int64_t ldy;
  int64_t N;
  int K, M, relu;
};

template <typename T>
__device__ __forceinline__ void store_quad(T* p, const float (&v)[4], int left, bool wide) {
  if (wide && left >= 4) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else
      *reinterpret_cast<uint2*>(p) = make_uint2((uint32_t)f32_to_bf16(v[0]) | ((uint32_t)f32_to_bf16(v[1]) << 16),
                                                (uint32_t)f32_to_bf16(v[2]) | ((uint32_t)f32_to_bf16(v[3]) << 16));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = f32_to_scalar<T>(v[j]);
  }
}

// A wave owns 32 rows x 128 output columns (four 32 x 32 tiles, the weights as the first operand so that a lane holds
// four consecutive outputs of one row); operands come from memory as they lie.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_linear_i8(I8Args a, bool wide) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i32 = lane & 31, half = lane >> 5;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * 32;
  const int m0 = (int)blockIdx.y * 128;
  if (n0 >= a.N) return;
  const int64_t row = n0 + i32 < a.N ? n0 + i32 : a.N - 1;
  const int Kp = (a.K + 15) & ~15;
  const int8_t* xp = a.x + row * a.ldx;
  const int8_t* wp[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int m = m0 + 32 * t + i32;
    wp[t] = a.w + (int64_t)(m < a.M ? m : 0) * a.ldw;
  }
  i32x16 acc[4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0;
  for (int k0 = 0; k0 < Kp; k0 += 32) {
    const int k = k0 + 16 * half;
    const int off = k < Kp ? k : 0;
    i32x4 x = *reinterpret_cast<const i32x4*>(xp + off);
    const int left = a.K - k;   // bytes of this lane that are columns; the others count as zeros
    if (left < 16)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int l = left - 4 * j;
        x[j] = l >= 4 ? x[j] : (l <= 0 ? 0 : (int32_t)((uint32_t)x[j] & ((1u << (8 * l)) - 1u)));
      }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      acc[t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(*reinterpret_cast<const i32x4*>(wp[t] + off), x, acc[t], 0, 0, 0);
  }
  if (n0 + i32 >= a.N) return;
  const float xs = a.xs[row];
  T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = m0 + 32 * t + 8 * q + 4 * half;
      if (m >= a.M) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int mj = m + j < a.M ? m + j : a.M - 1;
        v[j] = (float)acc[t][4 * q + j] * (xs * a.ws[mj]);
        if (a.bias) v[j] += scalar_to_f32(static_cast<const T*>(a.bias)[mj]);
        if (a.relu) v[j] = v[j] <= 0.f ? 0.f : v[j];   // a NaN stays
      }
      store_quad(y + m, v, a.M - m, wide);
    }
}

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int64_t mpnn_linear_int8_workspace_bytes(int64_t N, int32_t K, int32_t M, int32_t x_dtype) {
  if (N < 0 || K < 1 || K > kI8MaxK || M < 1) return -1;
  if (x_dtype == MPNN_I8) return 0;
  return N * ((K + 15) / 16 * 16) + align_up(N * 4, 16);
}

int32_t mpnn_linear_int8(const void* X, int64_t ldx, int32_t x_dtype, const float* x_scale, const void* W, int64_t ldw,
                         const float* w_scale, const void* bias, void* Y, int64_t ldy, int32_t y_dtype, int64_t N,
                         int32_t K, int32_t M, int32_t relu, void* workspace, mpnn_stream_t stream) {
  if ((x_dtype != MPNN_F32 && x_dtype != MPNN_BF16 && x_dtype != MPNN_I8) || (y_dtype != MPNN_F32 && y_dtype != MPNN_BF16))
    return fail(MPNN_E_INVALID, "mpnn_linear_int8: dtypes %d, %d", x_dtype, y_dtype);
  if (N < 0 || K < 1 || K > kI8MaxK || M < 1) return fail(MPNN_E_INVALID, "mpnn_linear_int8: N=%lld K=%d M=%d (K up to %d)", (long long)N, K, M, kI8MaxK);
  const int Kp = (K + 15) / 16 * 16;
  if (ldx < (x_dtype == MPNN_I8 ? Kp : K) || ldw < Kp || ldy < M) return fail(MPNN_E_INVALID, "mpnn_linear_int8: leading dimension too small");
  if (N == 0) return MPNN_OK;
  if (!X || !W || !w_scale || !Y || (x_dtype == MPNN_I8 ? !x_scale : !workspace)) return fail(MPNN_E_INVALID, "mpnn_linear_int8: null pointer argument");
  if (((uintptr_t)W & 15) || (ldw & 15) || (x_dtype == MPNN_I8 && (((uintptr_t)X & 15) || (ldx & 15))) || ((uintptr_t)workspace & 15))
    return fail(MPNN_E_INVALID, "mpnn_linear_int8: 8-bit rows and the workspace must be 16-byte aligned");
  I8Args a{static_cast<const int8_t*>(X), ldx, x_scale, static_cast<const int8_t*>(W), ldw, w_scale, bias, Y, ldy, N, K, M, relu};
  if (x_dtype != MPNN_I8) {
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + N * Kp);
    const int32_t rc = mpnn_quantize_rows(X, ldx, x_dtype, N, K, q, Kp, s, stream);
    if (rc != MPNN_OK) return rc;
    a.x = q; a.ldx = Kp; a.xs = s;
  }
  if ((N + 127) / 128 > INT32_MAX || (M + 127) / 128 > 65535) return fail(MPNN_E_INVALID, "mpnn_linear_int8: N=%lld M=%d", (long long)N, M);
  const dim3 grid((unsigned)((N + 127) / 128), (unsigned)((M + 127) / 128));
  const int quad = y_dtype == MPNN_BF16 ? 8 : 16;
  const bool wide = ((uintptr_t)Y % quad) == 0 && ldy % 4 == 0;
  if (y_dtype == MPNN_BF16) k_linear_i8<bf16_t><<<grid, kBlock, 0, stream>>>(a, wide);
  else k_linear_i8<float><<<grid, kBlock, 0, stream>>>(a, wide);
  MPNN_LAUNCH_CHECK("k_linear_i8");
  return MPNN_OK;
}

}  // extern "C"
