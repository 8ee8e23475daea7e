// Weight gradient from inputs that were kept in 8 bits (rows8.hip):
//
//   dW[m, k] = sum over rows n of  g[n, m] * open[n, m] * (scale[n] * q[n, k])        [q | q2] side by side as columns
//
// which for y = x W^T is the gradient of W with x replaced by the values its 8-bit rows stand for (the gradients of
// models/layers.py:104,140's Linear calls).  The scale belongs to the row, the contraction index, so it goes to g's
// side: p = g * scale in float32, cut into bfloat16 pieces of 8 bits each - three for float32 (exact), two for bfloat16
// g (16 of p's bits) - against q, whose whole numbers bfloat16 holds exactly.  v_mfma_f32_32x32x16_bf16, float32 sums.
//
// Bound: memory, if g is read once: a block of 8 waves owns up to 8 strips of g's columns (32 in float32, 64 in
// bfloat16) and one or two tiles of 128 columns of q, and walks row slabs.
//   g      goes from memory into the matrix operand directly: a lane's 8 contraction values are one column's 8 rows, so
//          32 lanes load 128 consecutive bytes of a row per instruction and nothing of g passes the LDS.
//   q      a thread loads 4 columns x 8 rows as 8 words, turns the bytes into four 8-value bfloat16 operands in
//          registers and leaves them in LDS in operand order (16-byte writes and reads, consecutive over lanes): every
//          value is converted once per block.  Column 4 i + t of a tile is column i of matrix tile t.
//   strips x tiles < 8: the waves left over share the rows of a slab; their sums meet in LDS at the end, in wave order.
// One partial tile per block, added in block order by a second launch: no atomics, the same bits on every run.
// Measured on 4 M rows: float32 256 x 128 0.97 ms = 4.8 TB/s, 128 x [128 | 128] with the relu's bits and g * open
// written 1.13 ms = 4.6 TB/s; bfloat16 256 x 128 0.65 ms = 4.0 TB/s, 128 x [128 | 128] with both 0.87 to 0.93 ms = 3.4 to
// 3.6 TB/s (a copy reaches 4.9).  What bounds bfloat16 there: the pieces are made once per matrix of q for half the bytes of g.
// Slabs of 64 rows instead of 128 for two column tiles took 1.13 ms, row clamps instead of whole slabs 20 % more.
#include "common.h"
#include "rowio.h"

namespace mpnn {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kTn8Threads = 512;
constexpr int kTn8MaxLd = 1 << 21;     // row strides: 24-bit byte offsets times a row of the slab fit 32 bits
constexpr int kTn8Rows = 128;           // rows per slab
constexpr int kTn8Tile = kTn8Rows * 256;   // bytes of a column tile of a slab: 128 columns in bfloat16
constexpr int tn8_lds(int wk) { return 2 * wk * kTn8Tile + 2 * wk * kTn8Rows * 4; }

struct Tn8Args {
  const void* g;
  int64_t ldg;
  const uint32_t* bits;          // optional [N][bits_pitch]
  int bits_pitch;                // words
  const int8_t *q, *q2;
  int64_t ldq, ldq2;
  const float *scale, *scale2;
  int K, K2;
  void* gout;                    // optional [N, M]: g * open
  int64_t ldgo;
  float* partial;                // [gridDim.x][M][K + K2]
  int64_t N;
  int M;
  int ktiles;                    // column tiles of both matrices
  int slabs;                     // of all rows
};

// 4 bytes of one row each from 8 rows -> the 8 values of column t as bfloat16, packed.
__device__ __forceinline__ u32x4 column_of(const uint32_t (&w)[8], int t) {
  u32x4 r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float lo = (float)((int32_t)(w[2 * p] << (24 - 8 * t)) >> 24);
    const float hi = (float)((int32_t)(w[2 * p + 1] << (24 - 8 * t)) >> 24);
    // whole numbers of 7 bits: the upper half of the float32 word is the bfloat16 value
    r[p] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
  return r;
}

// The pieces of 8 products.  Three: each is the upper half of what is left, so that the differences are exact and the
// third takes the rest whole.  Two: the nearest bfloat16 and the nearest to the exact difference, 2^-17 of the product.
template <int P>
__device__ __forceinline__ void pieces_of(const float (&v)[8], bf16x8 (&out)[P]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = v[j];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = P == 2 ? pack_bf16(r[2 * j], r[2 * j + 1])
                    : __builtin_amdgcn_perm(__float_as_uint(r[2 * j + 1]), __float_as_uint(r[2 * j]), 0x07060302u);
    out[p] = __builtin_bit_cast(bf16x8, w);
    if (p + 1 < P)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[2 * j] -= __uint_as_float(P == 2 ? w[j] << 16 : __float_as_uint(r[2 * j]) & 0xffff0000u);
        r[2 * j + 1] -= __uint_as_float(P == 2 ? w[j] & 0xffff0000u : __float_as_uint(r[2 * j + 1]) & 0xffff0000u);
      }
  }
}

// T: float (strips of 32 columns, one matrix tile per wave and column tile) or bf16_t (64 columns: a lane loads columns
// 2 i and 2 i + 1, matrix tiles of the even and the odd ones).  WM strips x WK column tiles x WN row shares = 8 waves.
template <typename T, int WM, int WK, int WN, bool BITS>
__global__ void __launch_bounds__(kTn8Threads, 2) k_gemm_tn8(Tn8Args a) {
  constexpr bool BF = sizeof(T) == 2;
  constexpr int U = BF ? 2 : 1;              // matrix tiles of g's columns per wave
  constexpr int P = BF ? 2 : 3;              // pieces
  constexpr int SN = kTn8Rows;
  constexpr int STEPS = SN / 16 / WN;        // of this wave per slab
  constexpr int D = STEPS < 4 ? STEPS : 4;   // steps of g in flight, 2 KiB per wave each
  static_assert(WM * WK * WN == 8 && STEPS >= 1, "8 waves");
  extern __shared__ __align__(16) char smem[];
  float* const s_scale = reinterpret_cast<float*>(smem + 2 * WK * kTn8Tile);   // [2][WK][SN]
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);   // uniform: what hangs on it stays in scalar registers
  const int i32 = lane & 31, half = lane >> 5;
  const int wm = wave % WM, wk = (wave / WM) % WK, wn = wave / (WM * WK);

  const int z0 = (a.K + 127) / 128;
  const int strip = (int)blockIdx.y * WM + wm;
  const int m0 = strip * 32 * U;
  const bool live = m0 < a.M && (int)blockIdx.z * WK + wk < a.ktiles;   // uniform in a wave

  f32x16 acc[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[u][t][r] = 0.f;

  // In float32 the sums of 1024 rows at a time are added to a second set: one chain over all of a block's rows would lose
  // two digits on millions of rows (a product's rounding to bfloat16 hides that).
  constexpr int CHAIN = 8;                   // slabs
  f32x16 whole[BF ? 1 : U][BF ? 1 : 4];
  int chain = 0;
  if constexpr (!BF)
#pragma unroll
    for (int t = 0; t < 4; ++t) whole[0][t] = acc[0][t];

  // staging: thread -> (octet of rows, word of 4 columns), 16 x 32 for each of the block's tiles
  const int st_oct = tid >> 5, st_word = tid & 31;
  const int8_t* st_q[WK];
  const float* st_scale[WK];
  int64_t st_ld[WK];
  uint32_t st_col[WK], q_off[WK];
#pragma unroll
  for (int w = 0; w < WK; ++w) {
    const int t = (int)blockIdx.z * WK + w < a.ktiles ? (int)blockIdx.z * WK + w : 0;
    const bool second = t >= z0;
    st_q[w] = second ? a.q2 : a.q;
    st_ld[w] = second ? a.ldq2 : a.ldq;
    st_scale[w] = second ? a.scale2 : a.scale;
    const int col = (second ? t - z0 : t) * 128 + 4 * st_word;
    st_col[w] = col < ((second ? a.K2 : a.K) + 15) / 16 * 16 ? col : 0;   // past the row: any bytes, never stored
    q_off[w] = __umul24(8 * st_oct, (uint32_t)st_ld[w]) + st_col[w];
  }
  uint32_t qw[WK][8];
  float sc = 0.f;
  // Every slab is whole: the last one starts SN rows before the end, and its rows that belong to the slab before count
  // with scale 0 (finite values add nothing then; an infinity or a NaN has made its sums NaN in its own slab already).
  // Addresses: a uniform base per row and 32-bit offsets from it (row strides are bounded by the host).
  auto first_of = [&](int slab) { return (int64_t)slab * SN < a.N - SN ? (int64_t)slab * SN : a.N - SN; };
  auto fetch_q = [&](int slab) __attribute__((always_inline)) {
    const int64_t n0 = first_of(slab);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const int8_t* base = st_q[w] + n0 * st_ld[w];
      each<8>([&](auto j) __attribute__((always_inline)) { qw[w][j] = *reinterpret_cast<const uint32_t*>(base + j * st_ld[w] + q_off[w]); });
    }
    // the scales of the slab's rows: tile 0's by the first 128 threads, tile 1's by the next
    if (tid < WK * SN) {
      const int64_t row = n0 + (tid & (SN - 1));
      sc = row >= (int64_t)slab * SN ? (WK == 2 && tid >= SN ? st_scale[WK - 1] : st_scale[0])[row] : 0.f;
    }
  };
  auto stash_q = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      char* base = smem + (buf * WK + w) * kTn8Tile;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        *reinterpret_cast<u32x4*>(base + ((((st_oct >> 1) * 4 + t) * 64) + (st_oct & 1) * 32 + st_word) * 16) = column_of(qw[w], t);
    }
    if (tid < WK * SN) s_scale[buf * WK * SN + tid] = sc;
  };

  // g: the lane's columns, 8 rows per step
  const int col = m0 + i32 * U;
  const int gcol = col < a.M ? col : 0;
  const int wbit = m0 / 32 + (BF ? i32 >> 4 : 0);
  const int wbit_in = wbit < a.bits_pitch ? wbit : 0;
  const int bshift = BF ? (2 * i32) & 31 : i32;
  const bool emit = a.gout && blockIdx.z == 0 && wk == 0 && live;
  uint32_t gr[D][8], br[D];
  const int64_t ldg = a.ldg * (int64_t)sizeof(T);
  const uint32_t g_off = __umul24(8 * half, (uint32_t)ldg) + gcol * sizeof(T);
  const uint32_t b_off = __umul24(8 * half + (lane & 7), (uint32_t)a.bits_pitch) + wbit_in;
  auto fetch_g = [&](int slab, auto s) __attribute__((always_inline)) {
    const int64_t r0 = first_of(slab) + (wn + s * WN) * 16;
    const char* base = static_cast<const char*>(a.g) + r0 * ldg;
    each<8>([&](auto j) __attribute__((always_inline)) { gr[s % D][j] = *reinterpret_cast<const uint32_t*>(base + j * ldg + g_off); });
    // lane l of 8 holds the word of row l; the lanes trade them when they are used
    if constexpr (BITS) br[s % D] = (a.bits + r0 * a.bits_pitch)[b_off];
  };

  const int64_t ldgo = a.ldgo * (int64_t)sizeof(T);
  const uint32_t o_off = __umul24(8 * half, (uint32_t)ldgo) + gcol * sizeof(T);
  int slab = blockIdx.x;
  int buf = 0;
  if (slab < a.slabs) {
    fetch_q(slab);
    if (live) each<D>([&](auto s) __attribute__((always_inline)) { fetch_g(slab, s); });
    stash_q(0);
  }
  __syncthreads();
  for (; slab < a.slabs; slab += gridDim.x, buf ^= 1) {
    const int next = slab + (int)gridDim.x;
    const bool more = next < a.slabs;
    if (more) fetch_q(next);
    if (live) {
      const char* base = smem + (buf * WK + wk) * kTn8Tile;
      const float* const scales = s_scale + (buf * WK + wk) * SN;
      each<STEPS>([&](auto s) __attribute__((always_inline)) {
        const int step = wn + s * WN;
        uint32_t w[8];
        each<8>([&](auto j) __attribute__((always_inline)) {
          w[j] = gr[s % D][j];
          if constexpr (BITS) {
            // one bit sign-extended is the mask of its entry
            const int word = __builtin_amdgcn_ds_swizzle((int)br[s % D], (j << 5) | 0x18);
            const uint32_t lo = (uint32_t)__builtin_amdgcn_sbfe(word, bshift, 1);
            if constexpr (BF) w[j] &= (lo & 0x0000ffffu) | ((uint32_t)__builtin_amdgcn_sbfe(word, bshift + 1, 1) & 0xffff0000u);
            else w[j] &= lo;
          }
        });
        if (emit && col < a.M) {
          char* out = static_cast<char*>(a.gout) + (first_of(slab) + step * 16) * ldgo;
          each<8>([&](auto j) __attribute__((always_inline)) { *reinterpret_cast<uint32_t*>(out + j * ldgo + o_off) = w[j]; });
        }
        if constexpr (s + D < STEPS) fetch_g(slab, std::integral_constant<int, s + D>{});
        else if (more) fetch_g(next, std::integral_constant<int, s + D - STEPS>{});
        float sv[8];
        {
          const float4 lo = *reinterpret_cast<const float4*>(scales + step * 16 + 8 * half);
          const float4 hi = *reinterpret_cast<const float4*>(scales + step * 16 + 8 * half + 4);
          sv[0] = lo.x; sv[1] = lo.y; sv[2] = lo.z; sv[3] = lo.w;
          sv[4] = hi.x; sv[5] = hi.y; sv[6] = hi.z; sv[7] = hi.w;
        }
        bf16x8 b[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          b[t] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(base + ((step * 4 + t) * 64 + lane) * 16));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t x = !BF ? w[j] : (u == 0 ? w[j] << 16 : w[j] & 0xffff0000u);
            v[j] = __uint_as_float(x) * sv[j];
          }
          bf16x8 p[P];
          pieces_of<P>(v, p);
#pragma unroll
          for (int q = P - 1; q >= 0; --q)   // the smallest pieces first
#pragma unroll
            for (int t = 0; t < 4; ++t) acc[u][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[q], b[t], acc[u][t], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);   // steps are not mixed: their operands would not fit the registers
      });
    }
    if constexpr (!BF) {
      if (++chain == CHAIN || !more) {
        chain = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            whole[0][t][r] += acc[0][t][r];
            acc[0][t][r] = 0.f;
          }
      }
    }
    if (more) stash_q(buf ^ 1);
    __syncthreads();
  }
  if constexpr (!BF)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[0][t] = whole[0][t];
  // the row shares meet in LDS: share 1, 2, .. are added to share 0 in that order, 16 values per lane at a time
  if constexpr (WN > 1) {
    float* meet = reinterpret_cast<float*>(smem);      // [wave][16][64] floats: 4 KiB per wave
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (wn > 0)
#pragma unroll
          for (int r = 0; r < 16; ++r) meet[(wave * 16 + r) * 64 + lane] = acc[u][t][r];
        __syncthreads();
        if (wn == 0)
#pragma unroll
          for (int o = 1; o < WN; ++o)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[u][t][r] += meet[((wave + o * WM * WK) * 16 + r) * 64 + lane];
        __syncthreads();
      }
  }
  if (!live || wn != 0) return;
  const int my_t = (int)blockIdx.z * WK + wk;
  const bool second = my_t >= z0;
  const int k0 = (second ? my_t - z0 : my_t) * 128, km = second ? a.K2 : a.K, ktot = a.K + a.K2;
  float* out = a.partial + (int64_t)blockIdx.x * a.M * ktot + (second ? a.K : 0);
  const int m_lane = m0 + 4 * half * U, k_lane = k0 + 4 * i32;
  const uint32_t o_lane = (uint32_t)m_lane * (uint32_t)ktot + k_lane;   // M * ktot is bounded by the host
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int i = ((r & 3) + 8 * (r >> 2)) * U + u;   // + 4 U half: the tile's row
      if (m_lane + i < a.M)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (k_lane + t < km) (out + (int64_t)i * ktot)[o_lane + t] = acc[u][t][r];
    }
}

// dW[m, k] = sum over blocks of partial[b][m][k]: wave w of a block adds blocks w, w + 4, .. for 64 consecutive
// outputs, then the four wave sums are added in wave order.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_tn8_sums(const float* __restrict__ partial, int blocks, int M, int K,
                                                     T* __restrict__ dW, int64_t ldw) {
  __shared__ float red[kBlock];
  const int64_t count = (int64_t)M * K;
  const int o = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + o;
  float s = 0.f;
  if (i < count) {
#pragma unroll 8
    for (int b = g; b < blocks; b += kBlock / 64) s += partial[(int64_t)b * count + i];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (g == 0 && i < count)
    dW[(i / K) * ldw + (i % K)] = f32_to_scalar<T>((red[o] + red[64 + o]) + (red[128 + o] + red[192 + o]));
}

// Fewer rows than a slab: a thread per output, 64 consecutive columns of [q | q2] by 4 rows of dW to a block; float32
// throughout.  Bound by latency.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_gemm_tn8_few(Tn8Args a, T* __restrict__ dW, int64_t ldw) {
  const int ktot = a.K + a.K2;
  const int c = (int)blockIdx.y * 64 + (threadIdx.x & 63), m = (int)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= a.M) return;
  const bool second = c >= a.K;
  const int8_t* q = second ? a.q2 : a.q;
  const int64_t ldq = second ? a.ldq2 : a.ldq;
  const float* scale = second ? a.scale2 : a.scale;
  const int k = c < ktot ? (second ? c - a.K : c) : 0;
  float sum = 0.f;
#pragma unroll 8
  for (int n = 0; n < (int)a.N; ++n) {
    float g = scalar_to_f32(static_cast<const T*>(a.g)[(int64_t)n * a.ldg + m]);
    if (a.bits && !((a.bits[(int64_t)n * a.bits_pitch + (m >> 5)] >> (m & 31)) & 1u)) g = 0.f;
    if (a.gout && c == 0) static_cast<T*>(a.gout)[n * a.ldgo + m] = f32_to_scalar<T>(g);
    if (c < ktot) sum = fmaf(g * scale[n], (float)q[n * ldq + k], sum);
  }
  if (c < ktot) dW[m * ldw + c] = f32_to_scalar<T>(sum);
}

struct Tn8Plan {
  int wm, wk, wn, strips, ktiles, slab_rows, blocks;
};

// Strips first (g is read once if all of them sit in one block), then column tiles, the rest of the waves over rows.
Tn8Plan tn8_plan(int64_t N, int M, int K, int K2, bool bf16) {
  Tn8Plan p;
  const int width = bf16 ? 64 : 32;
  p.strips = (M + width - 1) / width;
  p.ktiles = (K + 127) / 128 + (K2 + 127) / 128;
  p.wm = p.strips > 4 ? 8 : (p.strips > 2 ? 4 : p.strips);
  p.wk = (p.ktiles > 1 && p.wm < 8) ? 2 : 1;
  p.wn = 8 / (p.wm * p.wk);
  p.slab_rows = kTn8Rows;
  // one block per CU over all output tiles, as many as there are slabs (two slabs each at least: 18,432 rows, 64 x [64 | 64]
  // float32 18.5 us instead of 16.3, no faster with more rows)
  const int tiles = ((p.strips + p.wm - 1) / p.wm) * ((p.ktiles + p.wk - 1) / p.wk);
  int64_t blocks = 256 / tiles;
  const int64_t slabs = (N + p.slab_rows - 1) / p.slab_rows;
  if (blocks > slabs) blocks = slabs;
  if (blocks < 1) blocks = 1;
  p.blocks = (int)blocks;
  return p;
}

int32_t launch_one(void (*kernel)(Tn8Args), const Tn8Args& a, dim3 grid, int wk, hipStream_t stream) {
  const int bytes = tn8_lds(wk);
  MPNN_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  kernel<<<grid, kTn8Threads, bytes, stream>>>(a);
  MPNN_LAUNCH_CHECK("k_gemm_tn8");
  return MPNN_OK;
}

template <typename T>
int32_t launch_tn8(const Tn8Args& a, const Tn8Plan& p, hipStream_t stream) {
  const dim3 grid(p.blocks, (p.strips + p.wm - 1) / p.wm, (p.ktiles + p.wk - 1) / p.wk);
#define MPNN_TN8(WM, WK, WN)                                                              \
  if (p.wm == WM && p.wk == WK)                                                           \
    return a.bits ? launch_one(k_gemm_tn8<T, WM, WK, WN, true>, a, grid, WK, stream)      \
                  : launch_one(k_gemm_tn8<T, WM, WK, WN, false>, a, grid, WK, stream);
  MPNN_TN8(8, 1, 1)
  MPNN_TN8(4, 1, 2)
  MPNN_TN8(4, 2, 1)
  MPNN_TN8(2, 1, 4)
  MPNN_TN8(2, 2, 2)
  MPNN_TN8(1, 1, 8)
  MPNN_TN8(1, 2, 4)
#undef MPNN_TN8
  return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: no kernel for M=%d K=%d", a.M, a.K);
}

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int64_t mpnn_gemm_tn8_scratch_floats(int64_t N, int32_t M, int32_t K, int32_t K2, int32_t dtype) {
  if (N < 0 || M < 1 || K < 1 || K2 < 0) return -1;
  if (N < kTn8Rows) return 0;
  return (int64_t)tn8_plan(N, M, K, K2, dtype == MPNN_BF16).blocks * M * ((int64_t)K + K2);
}

int32_t mpnn_gemm_tn8(const void* G, int64_t ldg, int32_t dtype, const void* bits, const void* Q, int64_t ldq,
                      const float* scale, int32_t K, const void* Q2, int64_t ldq2, const float* scale2, int32_t K2,
                      void* dW, int64_t lddw, float* scratch, void* Gout, int64_t ldgo, int64_t N, int32_t M,
                      mpnn_stream_t stream) {
  const bool bf16 = dtype == MPNN_BF16;
  if (!bf16 && dtype != MPNN_F32) return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: dtype %d", dtype);
  if (N < 0 || M < 1 || K < 1 || K2 < 0 || M > kTn8MaxLd || K > kTn8MaxLd || K2 > kTn8MaxLd)
    return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: N=%lld M=%d K=%d K2=%d", (long long)N, M, K, K2);
  const int64_t ktot = (int64_t)K + K2;
  if (M * ktot > (1 << 30) || (ktot + 63) / 64 > 65535) return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: M=%d x %lld outputs", M, (long long)ktot);
  if (!dW || lddw < ktot) return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: dW is null or lddw below K + K2");
  const Tn8Plan p = tn8_plan(N, M, K, K2, bf16);
  if (N > 0) {
    if (!G || !Q || !scale || (N >= kTn8Rows && !scratch) || (K2 > 0 && (!Q2 || !scale2))) return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: null pointer argument");
    if (ldg < M || ldq < (K + 15) / 16 * 16 || (K2 > 0 && ldq2 < (K2 + 15) / 16 * 16) || (Gout && ldgo < M))
      return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: leading dimension too small");
    if (ldg > kTn8MaxLd || ldq > kTn8MaxLd || ldq2 > kTn8MaxLd || ldgo > kTn8MaxLd)
      return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: row strides above %d", kTn8MaxLd);
    // q moves as words of 4 columns, bfloat16 g as pairs
    if ((((uintptr_t)Q | (uintptr_t)Q2) & 3) || (ldq & 3) || (K2 > 0 && (ldq2 & 3)))
      return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: 8-bit rows must be 4-byte aligned");
    if (bf16 && ((M & 1) || (ldg & 1) || (Gout && (ldgo & 1)) || (((uintptr_t)G | (uintptr_t)Gout) & 3)))
      return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: bfloat16 rows must hold whole pairs of columns");
    if ((N + p.slab_rows - 1) / p.slab_rows > INT32_MAX / 2) return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: too many rows");
    Tn8Args a;
    memset(&a, 0, sizeof a);
    a.g = G; a.ldg = ldg;
    a.bits = static_cast<const uint32_t*>(bits); a.bits_pitch = (M + 31) / 32;
    a.q = static_cast<const int8_t*>(Q); a.ldq = ldq; a.scale = scale; a.K = K;
    if (K2 > 0) { a.q2 = static_cast<const int8_t*>(Q2); a.ldq2 = ldq2; a.scale2 = scale2; a.K2 = K2; }
    a.gout = Gout; a.ldgo = ldgo; a.partial = scratch; a.N = N; a.M = M;
    a.ktiles = p.ktiles;
    a.slabs = (int)((N + p.slab_rows - 1) / p.slab_rows);
    if (N < kTn8Rows) {
      const dim3 grid((unsigned)((M + 3) / 4), (unsigned)((ktot + 63) / 64));
      if (bf16) k_gemm_tn8_few<bf16_t><<<grid, kBlock, 0, stream>>>(a, static_cast<bf16_t*>(dW), lddw);
      else k_gemm_tn8_few<float><<<grid, kBlock, 0, stream>>>(a, static_cast<float*>(dW), lddw);
      MPNN_LAUNCH_CHECK("k_gemm_tn8_few");
      return MPNN_OK;
    }
    const int32_t rc = bf16 ? launch_tn8<bf16_t>(a, p, stream) : launch_tn8<float>(a, p, stream);
    if (rc != MPNN_OK) return rc;
  }
  const int64_t count = (int64_t)M * ktot;
  const int64_t grid = (count + 63) / 64;
  if (grid > INT32_MAX) return fail(MPNN_E_INVALID, "mpnn_gemm_tn8: M=%d x %lld outputs", M, (long long)ktot);
  const int blocks = N > 0 ? p.blocks : 0;
  if (bf16) k_tn8_sums<bf16_t><<<(int)grid, kBlock, 0, stream>>>(scratch, blocks, M, (int)ktot, static_cast<bf16_t*>(dW), lddw);
  else k_tn8_sums<float><<<(int)grid, kBlock, 0, stream>>>(scratch, blocks, M, (int)ktot, static_cast<float*>(dW), lddw);
  MPNN_LAUNCH_CHECK("k_tn8_sums");
  return MPNN_OK;
}

}  // extern "C"
