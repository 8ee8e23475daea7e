// Residual join with the norms around it (no counterpart in the reference, whose stacks are two layers deep; it stands
// between the layers of a deep stack built from models/layers.py:11-140).  Per row of H columns, in float32:
//
//   n      = post ? norm(block) * post_w + post_b : block        norm(v) = v / sqrt(mean(v^2) + eps)            (RMS)
//   stream = residual_scale * residual + branch_scale * gate * n  norm(v) = (v - mean) / sqrt(var(v) + eps)    (LAYER)
//   normed = norm(stream) * w + b                                 gate: none, [H], one per row, or [N, H]
//
// Backward of y = hat * w + b with hat = norm(v), inv = 1 / sqrt(.. + eps):  gh = gy * w,
//   gv = inv * (gh - hat * mean(gh * hat) [- mean(gh), LAYER]),  gw = sum over rows gy * hat,  gb = sum over rows gy.
// The backward reads the forward's INPUTS and forms the rows again in registers (two or four sums over a row more):
// nothing but the inputs is kept between the passes, and the recomputed rows are the forward's before rounding.
//
// Bound: memory.  Forward 2 rows read and 2 written (3 read with a full gate), backward 4 read and 2 written, no
// value touched twice.  A row lies in LPR lanes (8 to 512, a power of two) with four columns each, so that two dozen
// registers hold a row's streams, the parameters and the column sums and 16 waves per CU keep the next row of every
// stream on its way (eight columns per lane halved the waves: 2.13 instead of 1.17 ms for the backward of 4 M rows
// of 128 in bfloat16).  Sums over a row are lane exchanges on the vector unit, across waves (LPR > 64) through LDS.
// Sums over rows (gradients of weights, biases and a channel gate) stay in registers while a block walks its rows,
// leave one slab per block and are added by a second launch in block order: no atomics, the same bits on every run.
// Measured on 4 M rows of 128 in bfloat16 (RMS, norms on both sides, channel gate): forward 0.82 ms = 5.0 TB/s, backward
// 1.17 ms = 5.2 TB/s; a copy of 2 GiB reaches 4.9 TB/s.
#include "common.h"
#include "rowio.h"

namespace mpnn {
namespace {

constexpr int kNormMaxH = 2048;
constexpr int kNormSums = 5;            // post_w, post_b, w, b, channel gate
// Waves per SIMD that the register budget of each direction is held to, and the blocks launched for them: a block more
// would run after the others.
constexpr int kNormFwdWaves = 6;
constexpr int kNormBwdWaves = 4;

constexpr int norm_threads(int lpr) { return lpr > kBlock ? lpr : kBlock; }

struct NormArgs {
  const void *block, *residual, *gate, *post_w, *post_b, *w, *b;
  int64_t ldb, ldr, ldg;
  void *stream, *normed;
  int64_t lds, ldn;
  const void *g_stream, *g_normed;
  int64_t ldgs, ldgn;
  void *g_block, *g_residual, *g_gate;   // g_gate: rows for ROW / FULL
  int64_t ldgb, ldgr, ldgg;
  float* partial;                        // [gridDim.x][n_sums][H]
  int32_t slot[kNormSums];               // where a column sum lies in a slab, -1: not wanted
  int32_t n_sums;
  int64_t N;
  int32_t H, gate_kind, layer, post;
  float eps, rs, bs;
};

// Lane exchanges inside a row without the LDS crossbar: v of the lane that differs in the given bits of the lane index
// (1 and 2: within a quad; 4 and 8: mirrored within 8 and 16 lanes, which is as good where quads already hold equal
// sums).
template <int CTRL>
__device__ __forceinline__ float dpp_of(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}

// Sums of K values over the LPR lanes of a row.  LPR > 64: the row's waves meet in `red` (two sets used in turn, so that
// one barrier per call is enough; every row of the block is at the same call).
template <int LPR, int K>
struct RowSum {
  float* red;
  int turn;
  __device__ __forceinline__ void operator()(float (&v)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] += dpp_of<0xb1>(v[k]);    // quad_perm [1, 0, 3, 2]
      v[k] += dpp_of<0x4e>(v[k]);    // quad_perm [2, 3, 0, 1]
      v[k] += dpp_of<0x141>(v[k]);   // row_half_mirror
      if constexpr (LPR >= 16) v[k] += dpp_of<0x140>(v[k]);   // row_mirror
      if constexpr (LPR >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[k]), __float_as_uint(v[k]), false, false);
        v[k] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
      }
      if constexpr (LPR >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[k]), __float_as_uint(v[k]), false, false);
        v[k] = __uint_as_float(p[0]) + __uint_as_float(p[1]);
      }
    }
    if constexpr (LPR > 64) {
      constexpr int W = LPR / 64;                    // waves of a row
      float* r = red + turn * (K * 8);
      const int wave = threadIdx.x >> 6;             // at most 8 in the block
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) r[k * 8 + wave] = v[k];
      __syncthreads();
      const int first = wave / W * W;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float t = r[k * 8 + first];
#pragma unroll
        for (int w = 1; w < W; ++w) t += r[k * 8 + first + w];
        v[k] = t;
      }
      turn ^= 1;
    }
  }
};

// VEC columns of T at a time: 16 bytes in float32, 8 in bfloat16, or one column.  The columns a lane owns: vector v of NV
// covers columns (v * LPR + lane) * VEC and the VEC - 1 after it.  Raw: the lane's share of a row as it lies in memory,
// which a row that is on its way takes less registers for.
template <typename T, int VEC, int NV, int LPR>
struct Lane {
  static constexpr int C = VEC * NV;
  typedef RowIO<T, VEC> IO;
  struct Raw { typename IO::Raw v[NV]; };
  int col[NV];
  bool in[NV];
  __device__ __forceinline__ void init(int lane, int H) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LPR + lane) * VEC;
      in[v] = c < H;              // widths are multiples of VEC on this path: a vector is in or out
      col[v] = in[v] ? c : 0;     // lanes past the row load its first vector and count it as zeros
    }
  }
  __device__ __forceinline__ void fetch(const void* base, int64_t off, Raw& r) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) r.v[v] = IO::load_raw(static_cast<const T*>(base) + off + col[v]);
  }
  __device__ __forceinline__ void unpack(const Raw& r, float (&x)[C]) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float t[VEC];
      IO::unpack(r.v[v], t);
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[v * VEC + k] = in[v] ? t[k] : 0.f;
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t off, const float (&x)[C]) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!in[v]) continue;
      T* p = static_cast<T*>(base) + off + col[v];
      float t[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) t[k] = x[v * VEC + k];
      IO::store(p, t);
    }
  }
  // a column vector, `other` where there is none
  __device__ __forceinline__ void vector(const void* base, float other, float (&x)[C]) const {
    if (base) {
      Raw r;
      fetch(base, 0, r);
      unpack(r, x);
    } else
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = other;
  }
};

// What a row's tensors hold, on its way from memory.  One row of each stream is always in flight while the one before
// it is worked on.
template <typename L, typename T, bool BACKWARD>
struct RowData {
  typename L::Raw block, residual, gate, g_stream, g_normed;
  T row_gate;
  __device__ __forceinline__ void fetch(const NormArgs& a, const L& lane, int64_t row) {
    lane.fetch(a.block, row * a.ldb, block);
    if (a.residual) lane.fetch(a.residual, row * a.ldr, residual);
    if (a.gate_kind == MPNN_GATE_FULL) lane.fetch(a.gate, row * a.ldg, gate);
    if (a.gate_kind == MPNN_GATE_ROW) row_gate = static_cast<const T*>(a.gate)[row * a.ldg];
    if constexpr (BACKWARD) {
      if (a.g_stream) lane.fetch(a.g_stream, row * a.ldgs, g_stream);
      if (a.g_normed) lane.fetch(a.g_normed, row * a.ldgn, g_normed);
    }
  }
};

// The gate of a row times branch_scale; gch holds the channel gate (ones without one).
template <typename L, typename T, int C, typename D>
__device__ __forceinline__ void gate_of(const NormArgs& a, const L& lane, const D& d, const float (&gch)[C], float (&g)[C]) {
  if (a.gate_kind == MPNN_GATE_FULL) {
    lane.unpack(d.gate, g);
#pragma unroll
    for (int c = 0; c < C; ++c) g[c] *= a.bs;
  } else {
    const float one = a.gate_kind == MPNN_GATE_ROW ? a.bs * scalar_to_f32(d.row_gate) : a.bs;
#pragma unroll
    for (int c = 0; c < C; ++c) g[c] = gch[c] * one;
  }
}

// v -> hat in place, returns inv.  Columns past H hold zeros before and after.
template <typename L, int LPR, int C, int VEC>
__device__ __forceinline__ float normalize(float (&v)[C], const L& lane, bool layer, float inv_h, float eps,
                                           RowSum<LPR, 1>& sum) {
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) s[0] += v[c];
    sum(s);
    const float mean = s[0] * inv_h;
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = lane.in[c / VEC] ? v[c] - mean : 0.f;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int c = 0; c < C; ++c) q[0] = fmaf(v[c], v[c], q[0]);
  sum(q);
  const float inv = rsqrtf(q[0] * inv_h + eps);
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] *= inv;
  return inv;
}

// FORM: bit 0 the layer norm, bit 1 a norm of the block too; -1: as the arguments say (the column-by-column shapes)
template <int FORM>
__device__ __forceinline__ bool is_layer(const NormArgs& a) { return FORM < 0 ? a.layer != 0 : (FORM & 1) != 0; }
template <int FORM>
__device__ __forceinline__ bool is_post(const NormArgs& a) { return FORM < 0 ? a.post != 0 : (FORM & 2) != 0; }

template <typename T, int VEC, int NV, int LPR, int FORM>
__global__ void __launch_bounds__(norm_threads(LPR), kNormFwdWaves) k_block_norm_fwd(NormArgs a) {
  typedef Lane<T, VEC, NV, LPR> L;
  constexpr int C = L::C, THREADS = norm_threads(LPR), ROWS = THREADS / LPR;   // rows of a block at a time
  __shared__ float red[16];
  L lane;
  lane.init(threadIdx.x % LPR, a.H);
  RowSum<LPR, 1> sum{red, 0};
  const float inv_h = 1.f / (float)a.H;
  const bool layer = is_layer<FORM>(a), post = is_post<FORM>(a);
  float pw[C], pb[C], w[C], b[C], gch[C];
  lane.vector(a.post_w, 1.f, pw);
  lane.vector(a.post_b, 0.f, pb);
  lane.vector(a.w, 1.f, w);
  lane.vector(a.b, 0.f, b);
  lane.vector(a.gate_kind == MPNN_GATE_CHANNEL ? a.gate : nullptr, 1.f, gch);
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  // rows of several waves meet at barriers: a row past the end goes along, reads the last row and leaves nothing
  int64_t turns = a.N > row ? (a.N - row + step - 1) / step : 0;
  if constexpr (LPR > 64) turns = (a.N - (int64_t)blockIdx.x * ROWS + step - 1) / step;
  RowData<L, T, false> next, now;
  if (turns > 0) next.fetch(a, lane, row < a.N ? row : a.N - 1);
  for (; turns > 0; --turns, row += step) {
    now = next;
    const bool live = LPR <= 64 || row < a.N;
    if (turns > 1) next.fetch(a, lane, row + step < a.N ? row + step : a.N - 1);
    float n[C], s[C], g[C];
    lane.unpack(now.block, n);
    gate_of<L, T, C>(a, lane, now, gch, g);
    if (post) {
      normalize<L, LPR, C, VEC>(n, lane, layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) n[c] = fmaf(n[c], pw[c], pb[c]);
    }
    if (a.residual) {
      lane.unpack(now.residual, s);
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = fmaf(g[c], n[c], a.rs * s[c]);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = g[c] * n[c];
    }
    if (a.stream && live) lane.store(a.stream, row * a.lds, s);
    if (a.normed) {
      normalize<L, LPR, C, VEC>(s, lane, layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = fmaf(s[c], w[c], b[c]);
      if (live) lane.store(a.normed, row * a.ldn, s);
    }
  }
}

// Gradient of v from gh = gy * w and hat, inv of the forward.
template <typename L, int LPR, int C, int VEC>
__device__ __forceinline__ void norm_backward(float (&gh)[C], const float (&hat)[C], float inv, bool layer, float inv_h,
                                              RowSum<LPR, 1>& sum, RowSum<LPR, 2>& sum2) {
  float m0 = 0.f, m1;
  if (layer) {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) {       // columns past H hold zeros
      s[0] += gh[c];
      s[1] = fmaf(gh[c], hat[c], s[1]);
    }
    sum2(s);
    m0 = s[0] * inv_h;
    m1 = s[1] * inv_h;
  } else {
    float s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < C; ++c) s[0] = fmaf(gh[c], hat[c], s[0]);
    sum(s);
    m1 = s[0] * inv_h;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) gh[c] = inv * ((layer ? gh[c] - m0 : gh[c]) - hat[c] * m1);
}

template <typename T, int VEC, int NV, int LPR, int FORM>
__global__ void __launch_bounds__(norm_threads(LPR), kNormBwdWaves) k_block_norm_bwd(NormArgs a) {
  typedef Lane<T, VEC, NV, LPR> L;
  constexpr int C = L::C, THREADS = norm_threads(LPR), ROWS = THREADS / LPR;   // rows of a block at a time
  __shared__ float red[16];
  __shared__ float red2[32];
  __shared__ float col[THREADS * C];
  L lane;
  lane.init(threadIdx.x % LPR, a.H);
  RowSum<LPR, 1> sum{red, 0};
  RowSum<LPR, 2> sum2{red2, 0};
  const float inv_h = 1.f / (float)a.H;
  const bool layer = is_layer<FORM>(a), post = is_post<FORM>(a);
  float pw[C], pb[C], w[C], gch[C];
  lane.vector(a.post_w, 1.f, pw);
  lane.vector(a.post_b, 0.f, pb);
  lane.vector(a.w, 1.f, w);
  lane.vector(a.gate_kind == MPNN_GATE_CHANNEL ? a.gate : nullptr, 1.f, gch);
  float acc[kNormSums][C];
#pragma unroll
  for (int k = 0; k < kNormSums; ++k)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[k][c] = 0.f;
  const bool biases = a.slot[1] >= 0 || a.slot[3] >= 0;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LPR;
  // rows of several waves meet at barriers: a row past the end goes along, reads the last row and leaves nothing
  int64_t turns = a.N > row ? (a.N - row + step - 1) / step : 0;
  if constexpr (LPR > 64) turns = (a.N - (int64_t)blockIdx.x * ROWS + step - 1) / step;
  RowData<L, T, true> next, now;
  if (turns > 0) next.fetch(a, lane, row < a.N ? row : a.N - 1);
  for (; turns > 0; --turns, row += step) {
    now = next;
    const bool live = LPR <= 64 || row < a.N;
    if (turns > 1) next.fetch(a, lane, row + step < a.N ? row + step : a.N - 1);
    float n[C], s[C], gs[C], gu[C], g[C], hat1[C], inv1 = 0.f;
    lane.unpack(now.block, n);
    gate_of<L, T, C>(a, lane, now, gch, g);
    if (post) {
      inv1 = normalize<L, LPR, C, VEC>(n, lane, layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        hat1[c] = n[c];
        n[c] = fmaf(n[c], pw[c], pb[c]);
      }
    }
    if (a.g_stream) lane.unpack(now.g_stream, gs);
    else
#pragma unroll
      for (int c = 0; c < C; ++c) gs[c] = 0.f;
    if constexpr (LPR > 64) {
      if (!live)
#pragma unroll
        for (int c = 0; c < C; ++c) gs[c] = 0.f;
    }
    if (a.g_normed) {
      if (a.residual) {
        lane.unpack(now.residual, s);
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = fmaf(g[c], n[c], a.rs * s[c]);
      } else {
#pragma unroll
        for (int c = 0; c < C; ++c) s[c] = g[c] * n[c];
      }
      const float inv2 = normalize<L, LPR, C, VEC>(s, lane, layer, inv_h, a.eps, sum);
      lane.unpack(now.g_normed, gu);
      if constexpr (LPR > 64) {
        if (!live)
#pragma unroll
          for (int c = 0; c < C; ++c) gu[c] = 0.f;
      }
      if (biases)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[3][c] += gu[c];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        acc[2][c] = fmaf(gu[c], s[c], acc[2][c]);
        gu[c] *= w[c];
      }
      norm_backward<L, LPR, C, VEC>(gu, s, inv2, layer, inv_h, sum, sum2);
#pragma unroll
      for (int c = 0; c < C; ++c) gs[c] += lane.in[c / VEC] ? gu[c] : 0.f;
    }
    // gs: gradient of the stream
    if (a.g_residual) {
#pragma unroll
      for (int c = 0; c < C; ++c) gu[c] = a.rs * gs[c];
      if (live) lane.store(a.g_residual, row * a.ldgr, gu);
    }
    if (a.gate_kind != MPNN_GATE_NONE) {   // gradient of the gate
#pragma unroll
      for (int c = 0; c < C; ++c) gu[c] = gs[c] * (a.bs * n[c]);
      if (a.gate_kind == MPNN_GATE_CHANNEL) {
#pragma unroll
        for (int c = 0; c < C; ++c) acc[4][c] += gu[c];
      } else if (a.g_gate && a.gate_kind == MPNN_GATE_FULL) {
        if (live) lane.store(a.g_gate, row * a.ldgg, gu);
      } else if (a.g_gate) {
        float t[1] = {0.f};
#pragma unroll
        for (int c = 0; c < C; ++c) t[0] += lane.in[c / VEC] ? gu[c] : 0.f;
        sum(t);
        if (threadIdx.x % LPR == 0 && live) static_cast<T*>(a.g_gate)[row * a.ldgg] = f32_to_scalar<T>(t[0]);
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) gs[c] *= g[c];   // gradient of n
    if (post) {
      if (biases)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[1][c] += gs[c];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        acc[0][c] = fmaf(gs[c], hat1[c], acc[0][c]);
        gs[c] *= pw[c];
      }
      if (a.g_block) norm_backward<L, LPR, C, VEC>(gs, hat1, inv1, layer, inv_h, sum, sum2);
    }
    if (a.g_block && live) lane.store(a.g_block, row * a.ldgb, gs);
  }
  // column sums of the block: the row groups meet in LDS, group 0 first
#pragma unroll
  for (int k = 0; k < kNormSums; ++k) {
    if (a.slot[k] < 0) continue;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c) col[threadIdx.x * C + c] = acc[k][c];
    __syncthreads();
    float* out = a.partial + ((int64_t)blockIdx.x * a.n_sums + a.slot[k]) * a.H;
    for (int j = threadIdx.x; j < a.H; j += THREADS) {
      const int vec = j / VEC, v = vec / LPR, l = vec - v * LPR;
      float t = 0.f;
      for (int g = 0; g < ROWS; ++g) t += col[(g * LPR + l) * C + v * VEC + (j - vec * VEC)];
      out[j] = t;
    }
  }
}

struct NormSumArgs {
  const float* partial;
  void* out[kNormSums];      // by slot
  int32_t n_sums, H, blocks;
};

// out[slot][j] = sum over blocks of partial[block][slot][j].  A block takes 16 consecutive sums, 16 threads each: thread
// t of a sum adds blocks t, t + 16, .., then the 16 meet in LDS in that order (a wave per 64 sums walked the 768 slabs
// in 13 to 19 us).
template <typename T>
__global__ void __launch_bounds__(kBlock) k_block_norm_sums(NormSumArgs a) {
  __shared__ float red[kBlock];
  const int total = a.n_sums * a.H;
  const int o = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int i = blockIdx.x * 16 + o;
  float s = 0.f;
  if (i < total) {
#pragma unroll 16
    for (int b = g; b < a.blocks; b += 16) s += a.partial[(int64_t)b * total + i];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (g == 0 && i < total) {
    float t = red[o];
#pragma unroll
    for (int k = 1; k < 16; ++k) t += red[k * 16 + o];
    const int k = i / a.H;
    static_cast<T*>(a.out[k])[i - k * a.H] = f32_to_scalar<T>(t);
  }
}

// Lanes of a row: the smallest power of two that holds it with four columns per lane, in one vector (`wide`: width,
// addresses and strides allow 16 bytes in float32, 8 in bfloat16) or column by column.
int norm_lanes(int H, bool wide) {
  int lpr = wide ? 8 : 16;
  while (lpr * 4 < H) lpr *= 2;
  return !wide && lpr == 32 ? 64 : lpr;
}

// Blocks of the backward: at least four rows per row group, so that the slabs of column sums stay small next to the
// rows.
int norm_bwd_blocks(int64_t N, int lpr) {
  const int64_t per = 4 * (norm_threads(lpr) / lpr);
  const int64_t b = (N + per - 1) / per;
  const int most = 256 * 4 * kNormBwdWaves / (norm_threads(lpr) / 64);
  return (int)(b > most ? most : b);
}

template <typename T, int VEC, int NV, int LPR, int FORM>
void launch_form(const NormArgs& a, bool backward, int blocks, hipStream_t stream) {
  if (backward) k_block_norm_bwd<T, VEC, NV, LPR, FORM><<<blocks, norm_threads(LPR), 0, stream>>>(a);
  else k_block_norm_fwd<T, VEC, NV, LPR, FORM><<<blocks, norm_threads(LPR), 0, stream>>>(a);
}

template <typename T, int VEC, int NV, int LPR>
void launch_norm(const NormArgs& a, bool backward, int blocks, hipStream_t stream) {
  if constexpr (VEC == 1) {
    launch_form<T, VEC, NV, LPR, -1>(a, backward, blocks, stream);
  } else {
    const int form = (a.layer ? 1 : 0) | (a.post ? 2 : 0);
    if (form == 0) launch_form<T, VEC, NV, LPR, 0>(a, backward, blocks, stream);
    else if (form == 1) launch_form<T, VEC, NV, LPR, 1>(a, backward, blocks, stream);
    else if (form == 2) launch_form<T, VEC, NV, LPR, 2>(a, backward, blocks, stream);
    else launch_form<T, VEC, NV, LPR, 3>(a, backward, blocks, stream);
  }
}

template <typename T>
bool dispatch_norm(const NormArgs& a, bool wide, int lpr, bool backward, int blocks, hipStream_t stream) {
#define MPNN_NORM(LPR)                                                          \
  if (lpr == LPR) {                                                             \
    if (wide) launch_norm<T, 4, 1, LPR>(a, backward, blocks, stream);           \
    else if constexpr (LPR != 8 && LPR != 32) launch_norm<T, 1, 4, LPR>(a, backward, blocks, stream); \
    else return false;                                                          \
    return true;                                                                \
  }
  MPNN_NORM(8)
  MPNN_NORM(16)
  MPNN_NORM(32)
  MPNN_NORM(64)
  MPNN_NORM(128)
  MPNN_NORM(256)
  MPNN_NORM(512)
#undef MPNN_NORM
  return false;
}

// Checks what both directions share and fills the kernel's arguments; `wide`: every row of every operand can move four
// columns at a time, 16 bytes in float32 and 8 in bfloat16.
int32_t norm_args(const char* who, const mpnn_block_norm* d, bool backward, NormArgs& a, bool& wide) {
  if (!d) return fail(MPNN_E_INVALID, "%s: null descriptor", who);
  if (d->N < 0 || d->H < 1 || d->H > kNormMaxH)
    return fail(MPNN_E_INVALID, "%s: N=%lld H=%d (rows of 1 to %d columns)", who, (long long)d->N, d->H, kNormMaxH);
  if (d->dtype != MPNN_F32 && d->dtype != MPNN_BF16) return fail(MPNN_E_INVALID, "%s: dtype %d", who, d->dtype);
  if (d->norm != MPNN_NORM_RMS && d->norm != MPNN_NORM_LAYER) return fail(MPNN_E_INVALID, "%s: norm %d", who, d->norm);
  if (d->gate_kind < MPNN_GATE_NONE || d->gate_kind > MPNN_GATE_FULL) return fail(MPNN_E_INVALID, "%s: gate kind %d", who, d->gate_kind);
  if (!(d->eps >= 0.f)) return fail(MPNN_E_INVALID, "%s: eps must not be negative", who);
  const bool rows = d->N > 0;
  if (rows && !d->block) return fail(MPNN_E_INVALID, "%s: null pointer argument", who);
  if ((d->gate_kind != MPNN_GATE_NONE) != (d->gate != nullptr) && (rows || d->gate))
    return fail(MPNN_E_INVALID, "%s: gate and its kind disagree", who);
  const int H = d->H, vec_bytes = d->dtype == MPNN_BF16 ? 8 : 16;
  wide = H % 4 == 0;
  bool ok = true;
  auto row = [&](const void* p, int64_t ld) {
    if (!p) return;
    if (ld < H) ok = false;
    if ((uintptr_t)p % vec_bytes || ld % 4) wide = false;
  };
  auto vector = [&](const void* p) {
    if (p && (uintptr_t)p % vec_bytes) wide = false;
  };
  row(d->block, d->ldb);
  row(d->residual, d->ldr);
  if (d->gate_kind == MPNN_GATE_FULL) row(d->gate, d->ldg);
  if (d->gate_kind == MPNN_GATE_CHANNEL) vector(d->gate);
  if (d->gate_kind == MPNN_GATE_ROW && d->gate && d->ldg < 1) ok = false;
  vector(d->post_w);
  vector(d->post_b);
  vector(d->w);
  vector(d->b);
  if (!backward) {
    row(d->stream, d->lds);
    row(d->normed, d->ldn);
  } else {
    row(d->g_stream, d->ldgs);
    row(d->g_normed, d->ldgn);
    row(d->g_block, d->ldgb);
    row(d->g_residual, d->ldgr);
    if (d->gate_kind == MPNN_GATE_FULL) row(d->g_gate, d->ldgg);
    if (d->gate_kind == MPNN_GATE_ROW && d->g_gate && d->ldgg < 1) ok = false;
  }
  if (!ok) return fail(MPNN_E_INVALID, "%s: leading dimension too small", who);
  memset(&a, 0, sizeof a);
  a.block = d->block; a.residual = d->residual; a.gate = d->gate;
  a.post_w = d->post_w; a.post_b = d->post_b; a.w = d->w; a.b = d->b;
  a.ldb = d->ldb; a.ldr = d->ldr; a.ldg = d->ldg;
  a.N = d->N; a.H = H; a.gate_kind = d->gate_kind; a.layer = d->norm == MPNN_NORM_LAYER; a.post = d->post != 0;
  a.eps = d->eps; a.rs = d->residual_scale; a.bs = d->branch_scale;
  return MPNN_OK;
}

}  // namespace
}  // namespace mpnn

using namespace mpnn;

extern "C" {

int32_t mpnn_block_norm_fwd(const mpnn_block_norm* d, mpnn_stream_t stream) {
  NormArgs a;
  bool wide;
  const int32_t rc = norm_args("mpnn_block_norm_fwd", d, false, a, wide);
  if (rc != MPNN_OK) return rc;
  if (d->N == 0) return MPNN_OK;
  if (!d->stream && !d->normed) return fail(MPNN_E_INVALID, "mpnn_block_norm_fwd: no output");
  a.stream = d->stream; a.lds = d->lds; a.normed = d->normed; a.ldn = d->ldn;
  const bool bf16 = d->dtype == MPNN_BF16;
  const int lpr = norm_lanes(d->H, wide), rows = norm_threads(lpr) / lpr;
  const int64_t need = (d->N + rows - 1) / rows, most = 256 * 4 * kNormFwdWaves / (norm_threads(lpr) / 64);
  const int blocks = (int)(need > most ? most : need);
  const bool known = bf16 ? dispatch_norm<bf16_t>(a, wide, lpr, false, blocks, stream)
                          : dispatch_norm<float>(a, wide, lpr, false, blocks, stream);
  if (!known) return fail(MPNN_E_INVALID, "mpnn_block_norm_fwd: no kernel for H=%d", d->H);
  MPNN_LAUNCH_CHECK("k_block_norm_fwd");
  return MPNN_OK;
}

int64_t mpnn_block_norm_partial_floats(int64_t N, int32_t H, int32_t dtype) {
  (void)dtype;   // the slabs are float whatever the rows are
  if (N < 0 || H < 1 || H > kNormMaxH) return -1;
  int blocks = norm_bwd_blocks(N, norm_lanes(H, false));
  if (H % 4 == 0) {
    const int b = norm_bwd_blocks(N, norm_lanes(H, true));
    if (b > blocks) blocks = b;
  }
  return (int64_t)blocks * kNormSums * H;
}

int32_t mpnn_block_norm_bwd(const mpnn_block_norm* d, mpnn_stream_t stream) {
  NormArgs a;
  bool wide;
  const int32_t rc = norm_args("mpnn_block_norm_bwd", d, true, a, wide);
  if (rc != MPNN_OK) return rc;
  if (!d->post && (d->g_post_w || d->g_post_b)) return fail(MPNN_E_INVALID, "mpnn_block_norm_bwd: gradients of a norm that is not there");
  a.g_stream = d->g_stream; a.ldgs = d->ldgs; a.g_normed = d->g_normed; a.ldgn = d->ldgn;
  a.g_block = d->g_block; a.ldgb = d->ldgb; a.g_residual = d->g_residual; a.ldgr = d->ldgr;
  if (d->gate_kind == MPNN_GATE_ROW || d->gate_kind == MPNN_GATE_FULL) { a.g_gate = d->g_gate; a.ldgg = d->ldgg; }
  NormSumArgs f;
  memset(&f, 0, sizeof f);
  void* const sums[kNormSums] = {d->g_post_w, d->g_post_b, d->g_w, d->g_b,
                                 d->gate_kind == MPNN_GATE_CHANNEL ? d->g_gate : nullptr};
  int n = 0;
  for (int k = 0; k < kNormSums; ++k) {
    a.slot[k] = sums[k] ? n : -1;
    if (sums[k]) f.out[n++] = sums[k];
  }
  a.n_sums = n;
  if (n > 0 && d->N > 0 && !d->partial) return fail(MPNN_E_INVALID, "mpnn_block_norm_bwd: null pointer argument");
  a.partial = d->partial;
  const bool bf16 = d->dtype == MPNN_BF16;
  const int lpr = norm_lanes(d->H, wide);
  const int blocks = norm_bwd_blocks(d->N, lpr);
  if (d->N > 0) {
    const bool known = bf16 ? dispatch_norm<bf16_t>(a, wide, lpr, true, blocks, stream)
                            : dispatch_norm<float>(a, wide, lpr, true, blocks, stream);
    if (!known) return fail(MPNN_E_INVALID, "mpnn_block_norm_bwd: no kernel for H=%d", d->H);
    MPNN_LAUNCH_CHECK("k_block_norm_bwd");
  }
  if (n > 0) {
    f.partial = d->partial; f.n_sums = n; f.H = d->H; f.blocks = d->N > 0 ? blocks : 0;
    const int grid = (n * d->H + 15) / 16;
    if (bf16) k_block_norm_sums<bf16_t><<<grid, kBlock, 0, stream>>>(f);
    else k_block_norm_sums<float><<<grid, kBlock, 0, stream>>>(f);
    MPNN_LAUNCH_CHECK("k_block_norm_sums");
  }
  return MPNN_OK;
}

}  // extern "C"
