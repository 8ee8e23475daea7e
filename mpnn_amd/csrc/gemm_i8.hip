// Product of 8-bit rows with 8-bit weights (rows8.hip holds the format):
//
//   y[n, m] = act( (sum_k xq[n, k] * wq[m, k]) * xs[n] * ws[m] + bias[m] )
//
// the forward of a Linear call (models/layers.py:104,140, models/mpnn.py:101) of a trained model, with one scale per
// row of x and one per output channel.  The sum is exact (32-bit integers: 127 * 127 * K stays below 2^31 for
// K <= 8192), the scales are applied in float32 and the result is rounded once to the output type, in the same steps
// by every kernel here.  Weights are the first matrix operand, rows of x the second, so that a lane's results are
// consecutive outputs of one row.  Bytes behind column K count as zeros on x's side, whatever the weights hold there.
//
// Two kernels:
//   rows    K <= 512, weights resident in LDS: x is read once as it lies, taken to 8 bits in registers and multiplied
//           from there.  Bound by memory: 4 M rows of 128 -> 256 in 0.60 to 0.67 ms (bfloat16, 4.6 to 5.1 TB/s) and 1.20 ms
//           (float32, 5.1 TB/s; a copy reaches 4.9), Flickr's 89,250 of 500 -> 192 in 57 us (float32, 4.3 TB/s).
//   tiles   both sides staged through LDS in steps of 128 bytes by asynchronous copies.  65,536 x 1024 -> 2048 to
//           bfloat16 in 178 us (1540 TOP/s), 4096^3 in 74 us (1860 TOP/s; a large library product reaches 1990).  What bounds
//           it: operand reads from LDS (192 KiB per step of 128 and CU, three quarters of the matrix cores' time) and, for
//           short K, the results.
#include "common.h"
#include "rows8.h"

namespace mpnn {
namespace {

typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

constexpr int kI8MaxK = 8192;
constexpr int kI8MaxM = 1 << 20;

constexpr int kI8MaxTileLd = 1 << 22;   // bytes from row to row: a tile's rows are reached by 32-bit offsets

struct I8Args {
  const void* x; int64_t ldx;      // 8-bit rows, or float rows (rows kernel)
  const float* xs;                 // of 8-bit rows
  const int8_t* w; int64_t ldw;
  const float* ws;
  const void* bias;
  void* y; int64_t ldy;
  int64_t N;
  int K, M, relu;
  int width;                       // of the stores (store_width)
};

// A row's scale, as the factor the sum meets before the weight's scale and the one it meets after it.  The sum is a whole number
// below 2^28 and scales of rows are at least 2^-107: with a scale of at most 1 first, or one above 1 last, no product on the way
// leaves float32's range unless the result does (scale times scale would: 2^120 and 2^10 leave no zero of a sum of 0).
struct RowScale { float before, after; };
__device__ __forceinline__ RowScale row_scale(float xs) {
  const bool small = xs <= 1.f;           // a NaN goes last
  return RowScale{small ? xs : 1.f, small ? 1.f : xs};
}

__device__ __forceinline__ float finish(int32_t acc, RowScale x, float ws, float bias, int relu) {
  const float v = fmaf((float)acc * x.before * ws, x.after, bias);
  return relu && v <= 0.f ? 0.f : v;      // a NaN stays
}

// 16 bytes of which the first `left` are columns; the others count as zeros.
__device__ __forceinline__ i32x4 keep_bytes(i32x4 v, int left) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int l = left - 4 * j;
    v[j] = l >= 4 ? v[j] : (l <= 0 ? 0 : (int32_t)((uint32_t)v[j] & ((1u << (8 * l)) - 1u)));
  }
  return v;
}

// ------------------------------------------------------------------------------------------------------------- rows
// A wave owns 16 rows at a time.  Lane (row i = lane % 16, group g = lane / 16) holds 16 values of every step of 64
// columns.  Which 16 is free as long as both operands agree, so they are the ones that make the loads whole: in float32
// columns 16 p + 4 g .. + 3 (a row's four groups read 64 consecutive bytes per load), in bfloat16 32 p + 8 g .. + 7, in
// 8 bits 16 g .. + 15; the weights are brought into that order on their way to LDS, once per block.
// A result tile leaves lane (row, g) with the tile's weight rows 4 g .. 4 g + 3; the weight rows of a pair of tiles t are
// laid so that a lane ends with 8 consecutive outputs: column 8 (i / 4) + 4 t + i % 4 of the pair in row 16 t + i.
constexpr int kI8RowsThreads = 512;
constexpr int kI8RowsLds = 120 * 1024;   // for weights, their scales and biases; the result patches come on top

template <typename X> struct XRaw;
template <> struct XRaw<float> { float v[16]; };
template <> struct XRaw<bf16_t> { uint32_t v[8]; };
template <> struct XRaw<int8_t> { i32x4 v; };

// V elements of a row per load: the widest that the width, the address and the stride allow (89,250 bfloat16 rows of 500 -> 192:
// 39 us in vectors of 4, 86 one by one).
template <typename X, int V>
__device__ __forceinline__ void load_x(const X* p, int s, int g, int K, XRaw<X>& r) {
  if constexpr (sizeof(X) == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = 64 * s + 16 * q + 4 * g;
      if constexpr (V == 4) {   // K is a multiple of 4
        const float4 t = *reinterpret_cast<const float4*>(p + (k < K ? k : 0));
        r.v[4 * q] = t.x; r.v[4 * q + 1] = t.y; r.v[4 * q + 2] = t.z; r.v[4 * q + 3] = t.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[4 * q + e] = p[k + e < K ? k + e : 0];
      }
    }
  } else if constexpr (sizeof(X) == 2) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = 64 * s + 32 * q + 8 * g;
      if constexpr (V == 8) {   // K is a multiple of 8
        const uint4 t = *reinterpret_cast<const uint4*>(p + (k < K ? k : 0));
        r.v[4 * q] = t.x; r.v[4 * q + 1] = t.y; r.v[4 * q + 2] = t.z; r.v[4 * q + 3] = t.w;
      } else if constexpr (V == 4) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const uint2 t = *reinterpret_cast<const uint2*>(p + (k + e < K ? k + e : 0));
          r.v[4 * q + e / 2] = t.x; r.v[4 * q + e / 2 + 1] = t.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          r.v[4 * q + e / 2] = (uint32_t)p[k + e < K ? k + e : 0] | ((uint32_t)p[k + e + 1 < K ? k + e + 1 : 0] << 16);
      }
    }
  } else {
    const int k = 64 * s + 16 * g;
    r.v = *reinterpret_cast<const i32x4*>(p + (k < K ? k : 0));   // rows are readable up to K rounded up to 16
  }
}

// The step's 16 values in operand order, zeros for columns from K on.
template <typename X>
__device__ __forceinline__ void values_of(const XRaw<X>& r, int s, int g, int K, float (&v)[16]) {
  if constexpr (sizeof(X) == 4) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = r.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[2 * e] = __uint_as_float(r.v[e] << 16);
      v[2 * e + 1] = __uint_as_float(r.v[e] & 0xffff0000u);
    }
  }
  if (64 * s + 64 > K)   // uniform
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int k = sizeof(X) == 4 ? 64 * s + 16 * (e / 4) + 4 * g + e % 4 : 64 * s + 32 * (e / 8) + 8 * g + e % 8;
      v[e] = k < K ? v[e] : 0.f;
    }
}

// Waves per SIMD that the registers are held to: 16 waves per CU, 8 where a tile's raw rows take more than half of them.
template <typename X>
constexpr int rows_waves(int ks) { return ks == 8 || ks * sizeof(X) * 4 > 48 ? 2 : 4; }

template <typename X, typename Y, int KS, int V>
__global__ void __launch_bounds__(kI8RowsThreads, rows_waves<X>(KS)) k_linear_i8_rows(I8Args a, int slice) {
  extern __shared__ __align__(16) char lds[];
  constexpr int PITCH = KS * 64 + 16;   // 16 bytes more: eight consecutive rows start in different banks
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int m_begin = (int)blockIdx.y * slice;
  const int m_count = a.M - m_begin < slice ? a.M - m_begin : slice;
  const int m_pad = (m_count + 31) & ~31;
  const int Kp = (a.K + 15) & ~15, steps = (a.K + 63) >> 6;
  float* const s_ws = reinterpret_cast<float*>(lds + m_pad * PITCH);
  float* const s_bias = s_ws + m_pad;
  const Patch<Y, 16> patch{reinterpret_cast<char*>(s_bias + m_pad) + wave * (int)Patch<Y, 16>::BYTES};
  const X* const x = static_cast<const X*>(a.x);

  const int64_t tiles = (a.N + 15) >> 4, step = (int64_t)gridDim.x * (kI8RowsThreads / 64);
  int64_t tile = (int64_t)blockIdx.x * (kI8RowsThreads / 64) + wave;
  XRaw<X> raw[KS];
  float held = 0.f;
  auto fetch = [&](int64_t t) __attribute__((always_inline)) {
    const int64_t row = 16 * t + i < a.N ? 16 * t + i : a.N - 1;
    if constexpr (sizeof(X) == 1) held = a.xs[row];
    int from = g;
    asm volatile("" : "+v"(from));   // the column offsets are formed anew per tile: kept, they would not fit the registers
#pragma unroll
    for (int s = 0; s < KS; ++s)
      if (s < steps) load_x<X, V>(x + row * a.ldx, s, from, a.K, raw[s]);
  };
  if (tile < tiles) fetch(tile);

  for (int idx = threadIdx.x; idx < m_pad * (KS * 4); idx += kI8RowsThreads) {
    const int pos = idx / (KS * 4), c = idx - pos * (KS * 4);
    if (16 * c >= Kp) continue;         // never multiplied by anything but zeros
    const int r = pos & 15;
    const int m = m_begin + (pos & ~31) + 8 * (r >> 2) + 4 * ((pos >> 4) & 1) + (r & 3);
    const i32x4 v = *reinterpret_cast<const i32x4*>(a.w + (int64_t)(m < a.M ? m : a.M - 1) * a.ldw + 16 * c);
    char* d = lds + pos * PITCH + (c >> 2) * 64;
    const int cc = c & 3;
    if constexpr (sizeof(X) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<int32_t*>(d + j * 16 + cc * 4) = v[j];
    } else if constexpr (sizeof(X) == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int u = 2 * cc + h;
        *reinterpret_cast<int2*>(d + (2 * (u & 3) + (u >> 2)) * 8) = make_int2(v[2 * h], v[2 * h + 1]);
      }
    } else {
      *reinterpret_cast<i32x4*>(d + cc * 16) = v;
    }
  }
  for (int j = threadIdx.x; j < m_pad; j += kI8RowsThreads) {
    const int m = m_begin + j < a.M ? m_begin + j : a.M - 1;
    s_ws[j] = a.ws[m];
    s_bias[j] = a.bias ? scalar_to_f32(static_cast<const Y*>(a.bias)[m]) : 0.f;
  }
  __syncthreads();

  for (; tile < tiles; tile += step) {
    i32x4 q[KS];
    float xs;
    if constexpr (sizeof(X) == 1) {
      xs = held;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = 64 * s + 64 > a.K ? keep_bytes(raw[s].v, a.K - 64 * s - 16 * g) : raw[s].v;
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (s < steps) {
          float v[16];
          values_of<X>(raw[s], s, g, a.K, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) top = magnitude_bits(v[e]) > top ? magnitude_bits(v[e]) : top;
        }
      {   // the row's other three groups
        uint32_t o = __shfl_xor(top, 16, 64);
        top = o > top ? o : top;
        o = __shfl_xor(top, 32, 64);
        top = o > top ? o : top;
      }
      const Quant qt = quant_of(top);
      xs = qt.scale;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (s < steps) {
          float v[16];
          values_of<X>(raw[s], s, g, a.K, v);
#pragma unroll
          for (int j = 0; j < 4; ++j) q[s][j] = (int32_t)quant_word(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], qt);
        }
    }
    if (tile + step < tiles) fetch(tile + step);
    const RowScale scale = row_scale(xs);
    for (int b = 0; b < m_pad; b += 32) {
      i32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      const char* w = lds + (b + i) * PITCH + g * 16;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        if (s < steps)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(w + t * 16 * PITCH + s * 64), q[s], acc[t], 0, 0, 0);
      float v[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float4 ws = *reinterpret_cast<const float4*>(s_ws + b + 8 * g + 4 * t);
        const float4 bs = *reinterpret_cast<const float4*>(s_bias + b + 8 * g + 4 * t);
        v[4 * t] = finish(acc[t][0], scale, ws.x, bs.x, a.relu);
        v[4 * t + 1] = finish(acc[t][1], scale, ws.y, bs.y, a.relu);
        v[4 * t + 2] = finish(acc[t][2], scale, ws.z, bs.z, a.relu);
        v[4 * t + 3] = finish(acc[t][3], scale, ws.w, bs.w, a.relu);
      }
      const int chunk = ((b & 32) + 8 * g) / patch.VEC;
      if constexpr (sizeof(Y) == 4) {
        patch.put(i, chunk, {v[0], v[1], v[2], v[3]});
        patch.put(i, chunk + 1, {v[4], v[5], v[6], v[7]});
      } else {
        patch.put(i, chunk, v);
      }
      if ((b & 32) || b + 32 >= m_pad) patch.leave(a.y, a.ldy, a.N, 16 * tile, m_begin + (b & ~63), m_begin + m_count, a.width);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ tiles
// A block of WN x WM waves owns WN * 32 TN rows x WM * 64 outputs; a wave TN x 2 tiles of 32 x 32.  Steps of PC 16-byte
// pieces of K (8 or 4): rows lie in LDS PC pieces apart, their pieces in an order that depends on the row, so that the 8
// lanes of a read group reach 8 different bank groups; the copies go straight to LDS in that order because a lane
// chooses where it reads, not where it writes.  The next step's copies run under this step's products.
// Output column m of a wave lies in row 32 t + i of its weight tiles with m = 32 ((i / 4) % 2) + 16 t + 4 (i / 8) + i % 4:
// a lane ends with 32 consecutive outputs.
__device__ const i32x4 kZeroPiece = {0, 0, 0, 0};

template <int WN, int WM, int TN, int PC>
constexpr int tiles_lds() { return 2 * (WN * TN * 32 + WM * 64) * 16 * PC + 2 * WM * 64 * 4; }   // + scales and biases

// Piece c of row r lies at this place of the row.
template <int PC>
__device__ __forceinline__ int piece_at(int r, int c) { return PC == 8 ? c ^ (r & 7) : c ^ ((r >> 1) & 3); }

template <typename Y, int WN, int WM, int TN, int PC>
__global__ void __launch_bounds__(WN * WM * 64, 2) k_linear_i8_tiles(I8Args a, int n_tiles, int m_tiles) {
  constexpr int BN = WN * TN * 32, BM = WM * 64, WAVES = WN * WM;
  constexpr int ROW = 16 * PC, STAGE = (BN + BM) * ROW;
  // results leave through the buffer that was read last
  static_assert(WAVES * Patch<Y, 32>::BYTES <= STAGE, "result patches fit a buffer");
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i32 = lane & 31, half = lane >> 5;
  const int wn = wave / WM, wm = wave % WM;
  // Blocks stay and go round the tiles, those of one XCD (block index mod 8) through all column tiles of a row tile one
  // after the other, so that a row tile is fetched into one L2 only.  A tile's last step already copies the next tile's
  // first, under its products; the barrier before the results waits for that copy.
  const int xcd = blockIdx.x & 7, turn = gridDim.x >> 3;
  const int Kp = (a.K + 15) & ~15, pieces = Kp >> 4;

  // copies: one instruction of a wave fills 64 / PC rows (1 KiB); rows 0 .. BN - 1 are x's, the others weights
  constexpr int COPIES = (BN + BM) * PC / 64 / WAVES, COPIES_X = BN * PC / 64 / WAVES;
  static_assert(COPIES_X * WAVES * 64 == BN * PC, "a copy is x's or the weights'");
  const int8_t *x0 = nullptr, *w0 = nullptr;   // the tile's first rows, and the lane's rows from there
  uint32_t from[COPIES];
  auto take = [&](int t) __attribute__((always_inline)) {   // false: no such tile
    const int nt = (t / m_tiles) * 8 + xcd;
    if (nt >= n_tiles) return false;
    const int64_t n0 = (int64_t)nt * BN;
    const int m0 = t % m_tiles * BM;
    x0 = static_cast<const int8_t*>(a.x) + n0 * a.ldx;
    w0 = a.w + (int64_t)m0 * a.ldw;
    const int n_last = a.N - n0 < BN ? (int)(a.N - n0) - 1 : BN - 1, m_last = a.M - m0 < BM ? a.M - m0 - 1 : BM - 1;
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      const int r = (c * WAVES + wave) * (64 / PC) + lane / PC;
      if (c < COPIES_X) {
        from[c] = (uint32_t)(r < n_last ? r : n_last) * (uint32_t)a.ldx;
      } else {
        const int p = r - BN, i = p & 31;
        const int m = (p & ~63) + 32 * ((i >> 2) & 1) + 16 * ((p >> 5) & 1) + 4 * (i >> 3) + (i & 3);
        from[c] = (uint32_t)(m < m_last ? m : m_last) * (uint32_t)a.ldw;
      }
    }
    return true;
  };
  const int piece = piece_at<PC>(lane / PC, lane % PC);   // (the copy's first row is a multiple of 8)
  auto stage = [&](int buf, int p0) __attribute__((always_inline)) {
    const int at = p0 + piece;
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      const int8_t* p = at < pieces ? (c < COPIES_X ? x0 : w0) + (from[c] + 16 * at) : reinterpret_cast<const int8_t*>(&kZeroPiece);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                       (__attribute__((address_space(3))) void*)(lds + buf * STAGE + (c * WAVES + wave) * 1024), 16, 0, 0);
    }
  };

  int tile = blockIdx.x >> 3, buf = 0;
  bool more = take(tile);
  if (more) stage(0, 0);
  while (more) {
    const int64_t n0 = (int64_t)((tile / m_tiles) * 8 + xcd) * BN;
    const int m0 = tile % m_tiles * BM;
    tile += turn;
    // what the results need besides the sums, ahead of a wait that is due anyway
    float xs[TN], ws = 0.f, bs = 0.f;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t row = n0 + (wn * TN + j) * 32 + i32;
      xs[j] = a.xs[row < a.N ? row : a.N - 1];
    }
    if (threadIdx.x < BM) {
      const int m = m0 + (int)threadIdx.x < a.M ? m0 + (int)threadIdx.x : a.M - 1;
      ws = a.ws[m];
      if (a.bias) bs = scalar_to_f32(static_cast<const Y*>(a.bias)[m]);
    }
    i32x16 acc[TN][2];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[j][t][r] = 0;
    for (int p0 = 0; p0 < pieces; p0 += PC, buf ^= 1) {
      copies_landed();
      __syncthreads();                     // this step's rows are here, the other buffer is read no more
      if (p0 + PC < pieces) stage(buf ^ 1, p0 + PC);
      else if ((more = take(tile))) stage(buf ^ 1, 0);
      const char* const xb = lds + buf * STAGE + (wn * TN * 32 + i32) * ROW;
      const char* const wb = lds + buf * STAGE + (BN + wm * 64 + i32) * ROW;
      if ((a.K & 15) && p0 + PC >= pieces) {   // the last piece holds bytes that are no columns
        for (int r = threadIdx.x; r < BN; r += WAVES * 64) {
          i32x4* const p = reinterpret_cast<i32x4*>(lds + buf * STAGE + r * ROW + piece_at<PC>(r, pieces - 1 - p0) * 16);
          *p = keep_bytes(*p, a.K & 15);
        }
        copies_landed();                   // (no copy is on its way across a barrier)
        __syncthreads();
      }
      i32x4 w[2][2], v[2][TN];                 // the operands of one product are on their way while the one before runs
      auto read = [&](auto kk) __attribute__((always_inline)) {
        const int slot = piece_at<PC>(lane, 2 * kk + half) * 16;
#pragma unroll
        for (int t = 0; t < 2; ++t) w[kk % 2][t] = *reinterpret_cast<const i32x4*>(wb + t * 32 * ROW + slot);
#pragma unroll
        for (int j = 0; j < TN; ++j) v[kk % 2][j] = *reinterpret_cast<const i32x4*>(xb + j * 32 * ROW + slot);
      };
      read(std::integral_constant<int, 0>{});
      each<PC / 2>([&](auto kk) __attribute__((always_inline)) {
        if constexpr (kk + 1 < PC / 2) read(std::integral_constant<int, kk + 1>{});
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int t = 0; t < 2; ++t) acc[j][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[kk % 2][t], v[kk % 2][j], acc[j][t], 0, 0, 0);
      });
    }
    float* const s_ws = reinterpret_cast<float*>(lds + 2 * STAGE);
    float* const s_bs = s_ws + BM;
    if (threadIdx.x < BM) {
      s_ws[threadIdx.x] = ws;
      s_bs[threadIdx.x] = bs;
    }
    const int mw = m0 + wm * 64;
    copies_landed();
    __syncthreads();                       // every wave has read its operands: the buffer may take results
    const Patch<Y, 32> patch{lds + (buf ^ 1) * STAGE + wave * (int)Patch<Y, 32>::BYTES};
    constexpr int VEC = Patch<Y, 32>::VEC;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const RowScale scale = row_scale(xs[j]);
#pragma unroll
      for (int c = 0; c < 32 / VEC; ++c) {
        float v[VEC], sw[VEC], sb[VEC];
        const int first = wm * 64 + 32 * half + c * VEC;
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          const float4 t = *reinterpret_cast<const float4*>(s_ws + first + e), u = *reinterpret_cast<const float4*>(s_bs + first + e);
          sw[e] = t.x; sw[e + 1] = t.y; sw[e + 2] = t.z; sw[e + 3] = t.w;
          sb[e] = u.x; sb[e + 1] = u.y; sb[e + 2] = u.z; sb[e + 3] = u.w;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int o = c * VEC + e;
          v[e] = finish(acc[j][o >> 4][o & 15], scale, sw[e], sb[e], a.relu);
        }
        patch.put(i32, half * (32 / VEC) + c, v);
      }
      patch.leave(a.y, a.ldy, a.N, n0 + (wn * TN + j) * 32, mw, a.M, a.width);
    }
  }
}

// --------------------------------------------------------------------------------------------------------- dispatch
// Steps of 64 columns of a width, as the rows kernel comes.
int rows_steps(int K) { return K <= 64 ? 1 : K <= 128 ? 2 : K <= 256 ? 4 : 8; }

// LDS bytes of 32 output columns in the rows kernel: weights, scales, biases.
constexpr int rows_per32(int ks) { return 32 * (ks * 64 + 16 + 8); }

// Rows or tiles (whose x is taken to 8 bits by a pass of its own first).  The rows kernel reads x once per slice of weights
// that fits the LDS.  Up to 256 columns it wins with one or two slices, or with few rows: 64 -> 2048 (two slices) takes 4 us
// for 18 rows and 231 for 262,144, tiles 7.5 and 264; 256 -> 512 (two) 5.3 and 115 against 8.2 and 116.  Wider rows leave it
// 8 waves per CU: it wins with one slice (1 M rows of 512 -> 128: 252 us, the quantising pass alone 300) and with very few
// rows (512 -> 2048: 7.7 against 10.0 us for 18), and loses with more (65,536 rows of 512 -> 512, three slices: 69 against 49).
bool i8_by_rows(int64_t N, int K, int M) {
  if (K > 512) return false;
  const int ks = rows_steps(K);
  const int64_t bytes = (int64_t)((M + 31) / 32) * rows_per32(ks);
  return ks < 8 ? bytes <= 2 * kI8RowsLds || N <= 4096 : bytes <= kI8RowsLds || N <= 32;
}

// What a launch of the rows kernel asks for: groups of 32 outputs per slice, slices, and LDS bytes of a block.
struct RowsPlan { int per, slices, bytes; };
constexpr int kI8Lds = 160 * 1024;       // of a CU

template <typename Y>
RowsPlan rows_plan(int64_t N, int M, int ks) {
  constexpr int patches = kI8RowsThreads / 64 * (int)Patch<Y, 16>::BYTES;
  const int m32 = (M + 31) / 32, per32 = rows_per32(ks);
  const int most = (kI8Lds - patches) / per32;      // groups of a slice that fit next to the result patches
  const int64_t row_blocks = (N + 127) / 128;       // 8 waves of 16 rows
  // as few slices as fit the room for weights, more of them when the rows alone would leave CUs without work
  int slices = (m32 * per32 + kI8RowsLds - 1) / kI8RowsLds;
  while (slices < m32 && row_blocks * slices < 256) ++slices;
  int per = (m32 + slices - 1) / slices;
  if (per > most) per = most;                       // (the share was rounded up to whole groups)
  slices = (m32 + per - 1) / per;
  return RowsPlan{per, slices, per * per32 + patches};
}

template <typename X, typename Y, int KS, int V>
int32_t launch_rows(const I8Args& a, hipStream_t stream) {
  const RowsPlan p = rows_plan<Y>(a.N, a.M, KS);
  const int64_t row_blocks = (a.N + 127) / 128;
  int per_cu = kI8Lds / p.bytes;
  const int by_regs = rows_waves<X>(KS) / 2;
  if (per_cu > by_regs) per_cu = by_regs;
  int64_t blocks = 256 * per_cu / p.slices;
  if (blocks < 1) blocks = 1;
  if (blocks > row_blocks) blocks = row_blocks;
  if (p.bytes > 64 * 1024)
    MPNN_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(k_linear_i8_rows<X, Y, KS, V>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, p.bytes));
  k_linear_i8_rows<X, Y, KS, V><<<dim3((unsigned)blocks, p.slices), kI8RowsThreads, p.bytes, stream>>>(a, p.per * 32);
  MPNN_LAUNCH_CHECK("k_linear_i8_rows");
  return MPNN_OK;
}

template <typename X, typename Y, int V>
int32_t rows_of(const I8Args& a, hipStream_t stream) {
  switch (rows_steps(a.K)) {
    case 1: return launch_rows<X, Y, 1, V>(a, stream);
    case 2: return launch_rows<X, Y, 2, V>(a, stream);
    case 4: return launch_rows<X, Y, 4, V>(a, stream);
    default: return launch_rows<X, Y, 8, V>(a, stream);
  }
}

template <typename Y, int WN, int WM, int TN, int PC>
int32_t launch_tiles(const I8Args& a, hipStream_t stream) {
  constexpr int BN = WN * TN * 32, BM = WM * 64, bytes = tiles_lds<WN, WM, TN, PC>();
  const int64_t nt = (a.N + BN - 1) / BN, mt = (a.M + BM - 1) / BM;
  if (a.ldx > kI8MaxTileLd || a.ldw > kI8MaxTileLd) return fail(MPNN_E_INVALID, "mpnn_linear_int8: row strides above %d", kI8MaxTileLd);
  const int64_t all = (nt + 7) / 8 * 8 * mt;
  const int64_t resident = 256 * (160 * 1024 / bytes);
  const int64_t grid = all < resident ? all : resident;
  if (all > INT32_MAX) return fail(MPNN_E_INVALID, "mpnn_linear_int8: N=%lld M=%d", (long long)a.N, a.M);
  const void* const f = reinterpret_cast<const void*>(k_linear_i8_tiles<Y, WN, WM, TN, PC>);
  MPNN_HIP_CHECK(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  k_linear_i8_tiles<Y, WN, WM, TN, PC><<<(unsigned)grid, WN * WM * 64, bytes, stream>>>(a, (int)nt, (int)mt);
  MPNN_LAUNCH_CHECK("k_linear_i8_tiles");
  return MPNN_OK;
}

// Tiles of 256 x 256 where they fill the CUs (16,384 rows of 500 -> 1024, 256 tiles: 30 us, with tiles of 128 x 128 32) and
// are not half empty; of 128 x 128 otherwise (16,384 of 512 -> 512, 128 large tiles: 18 us against 23; 65,536 of 2048 -> 64:
// 103 against 112).
bool i8_large_tiles(int64_t N, int M) { return M > 128 && ((N + 255) / 256) * ((M + 255) / 256) >= 256; }

template <typename Y>
int32_t launch_i8(const I8Args& a, bool rows, int x_dtype, int vec_in, hipStream_t stream) {
  if (rows) {
    if (x_dtype == MPNN_I8) return rows_of<int8_t, Y, 16>(a, stream);
    if (x_dtype == MPNN_F32) return vec_in == 4 ? rows_of<float, Y, 4>(a, stream) : rows_of<float, Y, 1>(a, stream);
    if (vec_in == 8) return rows_of<bf16_t, Y, 8>(a, stream);
    return vec_in == 4 ? rows_of<bf16_t, Y, 4>(a, stream) : rows_of<bf16_t, Y, 1>(a, stream);
  }
  return i8_large_tiles(a.N, a.M) ? launch_tiles<Y, 2, 4, 4, 8>(a, stream) : launch_tiles<Y, 2, 2, 2, 8>(a, stream);
}

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int64_t mpnn_linear_int8_workspace_bytes(int64_t N, int32_t K, int32_t M, int32_t x_dtype) {
  if (N < 0 || K < 1 || K > kI8MaxK || M < 1 || M > kI8MaxM) return -1;
  if (x_dtype == MPNN_I8 || i8_by_rows(N, K, M)) return 0;
  return N * ((K + 15) / 16 * 16) + align_up(N * 4, 16);
}

int64_t mpnn_linear_int8_lds_bytes(int64_t N, int32_t K, int32_t M, int32_t y_dtype) {
  if (N < 0 || K < 1 || K > kI8MaxK || M < 1 || M > kI8MaxM || (y_dtype != MPNN_F32 && y_dtype != MPNN_BF16)) return -1;
  if (i8_by_rows(N, K, M))
    return y_dtype == MPNN_BF16 ? rows_plan<bf16_t>(N, M, rows_steps(K)).bytes : rows_plan<float>(N, M, rows_steps(K)).bytes;
  return i8_large_tiles(N, M) ? tiles_lds<2, 4, 4, 8>() : tiles_lds<2, 2, 2, 8>();
}

int32_t mpnn_linear_int8(const void* X, int64_t ldx, int32_t x_dtype, const float* x_scale, const void* W, int64_t ldw,
                         const float* w_scale, const void* bias, void* Y, int64_t ldy, int32_t y_dtype, int64_t N,
                         int32_t K, int32_t M, int32_t relu, void* workspace, mpnn_stream_t stream) {
  if ((x_dtype != MPNN_F32 && x_dtype != MPNN_BF16 && x_dtype != MPNN_I8) || (y_dtype != MPNN_F32 && y_dtype != MPNN_BF16))
    return fail(MPNN_E_INVALID, "mpnn_linear_int8: dtypes %d, %d", x_dtype, y_dtype);
  if (N < 0 || K < 1 || K > kI8MaxK || M < 1 || M > kI8MaxM)
    return fail(MPNN_E_INVALID, "mpnn_linear_int8: N=%lld K=%d M=%d (K up to %d, M up to %d)", (long long)N, K, M, kI8MaxK, kI8MaxM);
  const int Kp = (K + 15) / 16 * 16;
  if (ldx < (x_dtype == MPNN_I8 ? Kp : K) || ldw < Kp || ldy < M) return fail(MPNN_E_INVALID, "mpnn_linear_int8: leading dimension too small");
  if (N == 0) return MPNN_OK;
  const bool rows = i8_by_rows(N, K, M), take = x_dtype != MPNN_I8 && !rows;     // to 8 bits in a pass of its own
  if (!X || !W || !w_scale || !Y || (x_dtype == MPNN_I8 && !x_scale) || (take && !workspace))
    return fail(MPNN_E_INVALID, "mpnn_linear_int8: null pointer argument");
  if (((uintptr_t)W & 15) || (ldw & 15) || (x_dtype == MPNN_I8 && (((uintptr_t)X & 15) || (ldx & 15))) || ((uintptr_t)workspace & 15))
    return fail(MPNN_E_INVALID, "mpnn_linear_int8: 8-bit rows and the workspace must be 16-byte aligned");
  const int width = store_width(Y, ldy * (y_dtype == MPNN_BF16 ? 2 : 4));
  I8Args a{X, ldx, x_scale, static_cast<const int8_t*>(W), ldw, w_scale, bias, Y, ldy, N, K, M, relu, width};
  if (take) {
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + N * Kp);
    const int32_t rc = mpnn_quantize_rows(X, ldx, x_dtype, N, K, q, Kp, s, stream);
    if (rc != MPNN_OK) return rc;
    a.x = q; a.ldx = Kp; a.xs = s;
  }
  int vec_in = x_dtype == MPNN_BF16 ? 8 : 4;
  auto whole = [&](int v) { return K % v == 0 && ldx % v == 0 && (uintptr_t)X % (v * (x_dtype == MPNN_BF16 ? 2 : 4)) == 0; };
  while (vec_in > 1 && !whole(vec_in)) vec_in = vec_in == 8 ? 4 : 1;
  return y_dtype == MPNN_BF16 ? launch_i8<bf16_t>(a, rows, x_dtype, vec_in, stream)
                              : launch_i8<float>(a, rows, x_dtype, vec_in, stream);
}

}  // extern "C"
