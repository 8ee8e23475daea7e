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
// value touched twice; the sums over a row are shuffles inside the LPR lanes that hold it (a power of two from 8 to
// 64 lanes, or the 256 of a block for wide rows), so a row never leaves registers between load and store.  Sums over
// rows (gradients of weights, biases and a channel gate) stay in registers while a block walks its rows, leave one
// slab per block and are added by a second launch in block order: no atomics, the same bits on every run.
#include "common.h"
#include "rowio.h"

namespace mpnn {
namespace {

constexpr int kNormMaxH = 2048;
constexpr int kNormSums = 5;            // post_w, post_b, w, b, channel gate
constexpr int kNormBwdBlocks = 1024;    // 4 blocks of 256 threads per CU

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

// Sums of K values over the LPR lanes of a row.  LPR = 256: the block's four waves meet in `red` (K floats per wave,
// two sets used in turn, so that one barrier per call is enough).
template <int LPR, int K>
struct RowSum {
  float* red;
  int turn;
  __device__ __forceinline__ void operator()(float (&v)[K]) {
    constexpr int W = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], off, 64);
    if constexpr (LPR > 64) {
      float* r = red + turn * (K * 4);
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) r[k * 4 + wave] = v[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = (r[k * 4] + r[k * 4 + 1]) + (r[k * 4 + 2] + r[k * 4 + 3]);
      turn ^= 1;
    }
  }
};

// The columns a lane owns: vector v of NV covers columns (v * LPR + lane) * VEC and the VEC - 1 after it.
template <typename T, int VEC, int NV, int LPR>
struct Lane {
  static constexpr int C = VEC * NV;
  int col[NV];
  bool in[NV];
  __device__ __forceinline__ void init(int lane, int H) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * LPR + lane) * VEC;
      in[v] = c < H;              // widths are multiples of VEC on this path: a vector is in or out
      col[v] = in[v] ? c : 0;
    }
  }
  __device__ __forceinline__ void load(const void* base, int64_t off, float (&x)[C]) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float t[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) t[k] = 0.f;
      if (in[v]) RowIO<T, VEC>::load(static_cast<const T*>(base) + off + col[v], t);
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[v * VEC + k] = t[k];
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t off, const float (&x)[C]) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float t[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) t[k] = x[v * VEC + k];
      if (in[v]) RowIO<T, VEC>::store(static_cast<T*>(base) + off + col[v], t);
    }
  }
  // a column vector, `other` where there is none
  __device__ __forceinline__ void vector(const void* base, float other, float (&x)[C]) const {
    if (base) load(base, 0, x);
    else
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = other;
  }
};

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
  const float inv = 1.f / sqrtf(q[0] * inv_h + eps);
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] *= inv;
  return inv;
}

template <typename T, int VEC, int NV, int LPR>
__global__ void __launch_bounds__(kBlock) k_block_norm_fwd(NormArgs a) {
  typedef Lane<T, VEC, NV, LPR> L;
  constexpr int C = L::C;
  __shared__ float red[8];
  L lane;
  lane.init(threadIdx.x % LPR, a.H);
  RowSum<LPR, 1> sum{red, 0};
  const float inv_h = 1.f / (float)a.H;
  float pw[C], pb[C], w[C], b[C], gch[C];
  lane.vector(a.post_w, 1.f, pw);
  lane.vector(a.post_b, 0.f, pb);
  lane.vector(a.w, 1.f, w);
  lane.vector(a.b, 0.f, b);
  lane.vector(a.gate_kind == MPNN_GATE_CHANNEL ? a.gate : nullptr, 1.f, gch);
  const int64_t step = (int64_t)gridDim.x * (kBlock / LPR);
  for (int64_t row = (int64_t)blockIdx.x * (kBlock / LPR) + threadIdx.x / LPR; row < a.N; row += step) {
    float n[C], s[C];
    lane.load(a.block, row * a.ldb, n);
    if (a.residual) lane.load(a.residual, row * a.ldr, s);
    else
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = 0.f;
    float g[C];
    if (a.gate_kind == MPNN_GATE_FULL) lane.load(a.gate, row * a.ldg, g);
    else {
      const float one = a.gate_kind == MPNN_GATE_ROW ? scalar_to_f32(static_cast<const T*>(a.gate)[row * a.ldg]) : 1.f;
#pragma unroll
      for (int c = 0; c < C; ++c) g[c] = gch[c] * one;
    }
    if (a.post) {
      normalize<L, LPR, C, VEC>(n, lane, a.layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) n[c] = fmaf(n[c], pw[c], pb[c]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) s[c] = fmaf(a.bs * g[c], n[c], a.rs * s[c]);
    if (a.stream) lane.store(a.stream, row * a.lds, s);
    if (a.normed) {
      normalize<L, LPR, C, VEC>(s, lane, a.layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = fmaf(s[c], w[c], b[c]);
      lane.store(a.normed, row * a.ldn, s);
    }
  }
}

// Gradient of v from gh = gy * w and hat, inv of the forward.
template <typename L, int LPR, int C, int VEC>
__device__ __forceinline__ void norm_backward(float (&gh)[C], const float (&hat)[C], float inv, const L& lane, bool layer,
                                              float inv_h, RowSum<LPR, 2>& sum) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < C; ++c) {
    s[0] += gh[c];                      // columns past H hold zeros
    s[1] = fmaf(gh[c], hat[c], s[1]);
  }
  sum(s);
  const float m0 = layer ? s[0] * inv_h : 0.f, m1 = s[1] * inv_h;
#pragma unroll
  for (int c = 0; c < C; ++c) gh[c] = inv * (gh[c] - m0 - hat[c] * m1);
}

template <typename T, int VEC, int NV, int LPR>
__global__ void __launch_bounds__(kBlock) k_block_norm_bwd(NormArgs a) {
  typedef Lane<T, VEC, NV, LPR> L;
  constexpr int C = L::C;
  __shared__ float red[8];
  __shared__ float red2[16];
  __shared__ float col[kBlock * C];
  L lane;
  lane.init(threadIdx.x % LPR, a.H);
  RowSum<LPR, 1> sum{red, 0};
  RowSum<LPR, 2> sum2{red2, 0};
  const float inv_h = 1.f / (float)a.H;
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
  const int64_t step = (int64_t)gridDim.x * (kBlock / LPR);
  for (int64_t row = (int64_t)blockIdx.x * (kBlock / LPR) + threadIdx.x / LPR; row < a.N; row += step) {
    float n[C], s[C], gs[C], gu[C], g[C];
    lane.load(a.block, row * a.ldb, n);
    if (a.residual) lane.load(a.residual, row * a.ldr, s);
    else
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = 0.f;
    if (a.gate_kind == MPNN_GATE_FULL) lane.load(a.gate, row * a.ldg, g);
    else {
      const float one = a.gate_kind == MPNN_GATE_ROW ? scalar_to_f32(static_cast<const T*>(a.gate)[row * a.ldg]) : 1.f;
#pragma unroll
      for (int c = 0; c < C; ++c) g[c] = gch[c] * one;
    }
    if (a.g_stream) lane.load(a.g_stream, row * a.ldgs, gs);
    else
#pragma unroll
      for (int c = 0; c < C; ++c) gs[c] = 0.f;
    float hat1[C], inv1 = 0.f;
    if (a.post) {
      inv1 = normalize<L, LPR, C, VEC>(n, lane, a.layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        hat1[c] = n[c];
        n[c] = fmaf(n[c], pw[c], pb[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) hat1[c] = 0.f;
    }
    if (a.g_normed) {
      lane.load(a.g_normed, row * a.ldgn, gu);
#pragma unroll
      for (int c = 0; c < C; ++c) s[c] = fmaf(a.bs * g[c], n[c], a.rs * s[c]);
      const float inv2 = normalize<L, LPR, C, VEC>(s, lane, a.layer, inv_h, a.eps, sum);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        acc[2][c] = fmaf(gu[c], s[c], acc[2][c]);
        acc[3][c] += gu[c];
        gu[c] *= w[c];
      }
      norm_backward<L, LPR, C, VEC>(gu, s, inv2, lane, a.layer, inv_h, sum2);
#pragma unroll
      for (int c = 0; c < C; ++c) gs[c] += lane.in[c / VEC] ? gu[c] : 0.f;
    }
    // gs: gradient of the stream
    if (a.g_residual) {
#pragma unroll
      for (int c = 0; c < C; ++c) gu[c] = a.rs * gs[c];
      lane.store(a.g_residual, row * a.ldgr, gu);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      gs[c] *= a.bs;
      gu[c] = gs[c] * n[c];            // gradient of the gate
      gs[c] *= g[c];                   // gradient of n
      acc[4][c] += gu[c];
    }
    if (a.g_gate && a.gate_kind == MPNN_GATE_FULL) lane.store(a.g_gate, row * a.ldgg, gu);
    if (a.g_gate && a.gate_kind == MPNN_GATE_ROW) {
      float t[1] = {0.f};
#pragma unroll
      for (int c = 0; c < C; ++c) t[0] += lane.in[c / VEC] ? gu[c] : 0.f;
      sum(t);
      if (threadIdx.x % LPR == 0) static_cast<T*>(a.g_gate)[row * a.ldgg] = f32_to_scalar<T>(t[0]);
    }
    if (a.post) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        acc[0][c] = fmaf(gs[c], hat1[c], acc[0][c]);
        acc[1][c] += gs[c];
        gs[c] *= pw[c];
      }
      if (a.g_block) norm_backward<L, LPR, C, VEC>(gs, hat1, inv1, lane, a.layer, inv_h, sum2);
    }
    if (a.g_block) lane.store(a.g_block, row * a.ldgb, gs);
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
    for (int j = threadIdx.x; j < a.H; j += kBlock) {
      const int vec = j / VEC, v = vec / LPR, l = vec - v * LPR;
      float t = 0.f;
      for (int g = 0; g < kBlock / LPR; ++g) t += col[(g * LPR + l) * C + v * VEC + (j - vec * VEC)];
      out[j] = t;
    }
  }
}

struct NormSumArgs {
  const float* partial;
  void* out[kNormSums];      // by slot
  int32_t n_sums, H, blocks;
};

// out[slot][j] = sum over blocks of partial[block][slot][j]: wave w of a block adds blocks w, w + 4, .. for 64
// consecutive sums, then the four wave sums are added in wave order.
template <typename T>
__global__ void __launch_bounds__(kBlock) k_block_norm_sums(NormSumArgs a) {
  __shared__ float red[kBlock];
  const int total = a.n_sums * a.H;
  const int o = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int i = blockIdx.x * 64 + o;
  float s = 0.f;
  if (i < total) {
#pragma unroll 8
    for (int b = g; b < a.blocks; b += kBlock / 64) s += a.partial[(int64_t)b * total + i];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (g == 0 && i < total) {
    const float t = (red[o] + red[64 + o]) + (red[128 + o] + red[192 + o]);
    const int k = i / a.H;
    static_cast<T*>(a.out[k])[i - k * a.H] = f32_to_scalar<T>(t);
  }
}

// How a row is spread: LPR lanes with NV vectors of VEC columns each.
struct NormShape { int vec, nv, lpr; };

// Whole 16-byte vectors: the smallest power of two of lanes that holds the row once; rows of more than 64 vectors
// take two per lane in float32 and a block of 256 lanes beyond that.  Other widths and alignments: one column per
// vector, up to 8 per lane.
NormShape norm_shape(int H, bool wide, bool bf16) {
  const int vec = wide ? (bf16 ? 8 : 4) : 1;
  const int nvec = H / vec;
  if (wide) {
    for (int lpr = 8; lpr <= 64; lpr *= 2)
      if (nvec <= lpr) return {vec, 1, lpr};
    if (!bf16 && nvec <= 128) return {vec, 2, 64};
    return {vec, nvec <= 256 ? 1 : 2, 256};
  }
  if (nvec <= 16) return {1, 1, 16};
  for (int nv = 1; nv <= 8; nv *= 2)
    if (nvec <= 64 * nv) return {1, nv, 64};
  return {1, nvec <= 1024 ? 4 : 8, 256};
}

// Blocks of the backward: at least four rows per row group, so that the slabs of column sums stay small next to the
// rows.
int norm_bwd_blocks(int64_t N, const NormShape& s) {
  const int64_t per = 4 * (kBlock / s.lpr);
  const int64_t b = (N + per - 1) / per;
  return (int)(b > kNormBwdBlocks ? kNormBwdBlocks : b);
}

template <typename T, int VEC, int NV, int LPR>
void launch_norm(const NormArgs& a, bool backward, int blocks, hipStream_t stream) {
  if (backward) k_block_norm_bwd<T, VEC, NV, LPR><<<blocks, kBlock, 0, stream>>>(a);
  else k_block_norm_fwd<T, VEC, NV, LPR><<<blocks, kBlock, 0, stream>>>(a);
}

template <typename T>
bool dispatch_norm(const NormArgs& a, const NormShape& s, bool backward, int blocks, hipStream_t stream) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  if (s.vec == V) {
    if (s.nv == 1 && s.lpr == 8) launch_norm<T, V, 1, 8>(a, backward, blocks, stream);
    else if (s.nv == 1 && s.lpr == 16) launch_norm<T, V, 1, 16>(a, backward, blocks, stream);
    else if (s.nv == 1 && s.lpr == 32) launch_norm<T, V, 1, 32>(a, backward, blocks, stream);
    else if (s.nv == 1 && s.lpr == 64) launch_norm<T, V, 1, 64>(a, backward, blocks, stream);
    else if (s.nv == 1 && s.lpr == 256) launch_norm<T, V, 1, 256>(a, backward, blocks, stream);
    else if constexpr (V == 4) {
      if (s.nv == 2 && s.lpr == 64) launch_norm<T, V, 2, 64>(a, backward, blocks, stream);
      else if (s.nv == 2 && s.lpr == 256) launch_norm<T, V, 2, 256>(a, backward, blocks, stream);
      else return false;
    } else return false;
    return true;
  }
  if (s.lpr == 16 && s.nv == 1) launch_norm<T, 1, 1, 16>(a, backward, blocks, stream);
  else if (s.lpr == 64 && s.nv == 1) launch_norm<T, 1, 1, 64>(a, backward, blocks, stream);
  else if (s.lpr == 64 && s.nv == 2) launch_norm<T, 1, 2, 64>(a, backward, blocks, stream);
  else if (s.lpr == 64 && s.nv == 4) launch_norm<T, 1, 4, 64>(a, backward, blocks, stream);
  else if (s.lpr == 64 && s.nv == 8) launch_norm<T, 1, 8, 64>(a, backward, blocks, stream);
  else if (s.lpr == 256 && s.nv == 4) launch_norm<T, 1, 4, 256>(a, backward, blocks, stream);
  else if (s.lpr == 256 && s.nv == 8) launch_norm<T, 1, 8, 256>(a, backward, blocks, stream);
  else return false;
  return true;
}

// Checks what both directions share and fills the kernel's arguments; `wide`: every row of every operand can move as
// 16-byte vectors.
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
  const int H = d->H, vec = d->dtype == MPNN_BF16 ? 8 : 4;
  wide = H % vec == 0;
  bool ok = true;
  auto row = [&](const void* p, int64_t ld) {
    if (!p) return;
    if (ld < H) ok = false;
    if (((uintptr_t)p & 15) || ld % vec) wide = false;
  };
  auto vector = [&](const void* p) {
    if (p && ((uintptr_t)p & 15)) wide = false;
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
  const NormShape s = norm_shape(d->H, wide, bf16);
  const int64_t need = (d->N + kBlock / s.lpr - 1) / (kBlock / s.lpr);
  const int blocks = (int)(need > kMaxBlocks ? kMaxBlocks : need);
  const bool known = bf16 ? dispatch_norm<bf16_t>(a, s, false, blocks, stream) : dispatch_norm<float>(a, s, false, blocks, stream);
  if (!known) return fail(MPNN_E_INVALID, "mpnn_block_norm_fwd: no kernel for H=%d", d->H);
  MPNN_LAUNCH_CHECK("k_block_norm_fwd");
  return MPNN_OK;
}

int64_t mpnn_block_norm_partial_floats(int64_t N, int32_t H, int32_t dtype) {
  if (N < 0 || H < 1 || H > kNormMaxH) return -1;
  const bool bf16 = dtype == MPNN_BF16;
  const int v = bf16 ? 8 : 4;
  int blocks = norm_bwd_blocks(N, norm_shape(H, false, bf16));
  if (H % v == 0) {
    const int b = norm_bwd_blocks(N, norm_shape(H, true, bf16));
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
  const NormShape s = norm_shape(d->H, wide, bf16);
  const int blocks = norm_bwd_blocks(d->N, s);
  if (d->N > 0) {
    const bool known = bf16 ? dispatch_norm<bf16_t>(a, s, true, blocks, stream) : dispatch_norm<float>(a, s, true, blocks, stream);
    if (!known) return fail(MPNN_E_INVALID, "mpnn_block_norm_bwd: no kernel for H=%d", d->H);
    MPNN_LAUNCH_CHECK("k_block_norm_bwd");
  }
  if (n > 0) {
    f.partial = d->partial; f.n_sums = n; f.H = d->H; f.blocks = d->N > 0 ? blocks : 0;
    const int grid = (n * d->H + 63) / 64;
    if (bf16) k_block_norm_sums<bf16_t><<<grid, kBlock, 0, stream>>>(f);
    else k_block_norm_sums<float><<<grid, kBlock, 0, stream>>>(f);
    MPNN_LAUNCH_CHECK("k_block_norm_sums");
  }
  return MPNN_OK;
}

}  // extern "C"
