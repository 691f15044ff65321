// Linear classifier + softmax cross entropy in pieces of the vocabulary, without keeping the logits.
//
//   l[n][v] = x[n] . w[v] + b[v],   lse[n] = log sum_v exp(l[n][v])
//   loss[n] = lse[n] - (1 - e) l[n][y] - e mean_v l[n][v]           (e: label smoothing)
//   d[n][v] = exp(l[n][v] - lse[n]) - e / V - (1 - e) [v = y],  s[n]: the row's upstream gradient
//   dx = s . d w,  dw = (s . d)' x,  db = sum_n s . d
//
// Bound by the matrix cores: 2 N V D operations for the loss, 8 N V D with the gradients, because the
// backward pass computes the logits again instead of reading N V of them from memory.
//
//  * forward: one product whose epilogue leaves (max, sum of exponentials) of every row over the
//    columns of one wave; a second launch joins them.
//  * backward, for each piece of the vocabulary: the product again, its epilogue writes d in bf16; then
//    dx += d w and dw = d' x, whose sums run over the classes and over the rows. Both operands whose sum index
//    is not the contiguous one, w and d, are read k by k as they lie (gemm_tile.h); d written both ways round and
//    w' laid out cost 8192 x 65536 x 2048 7.41 ms against 7.02, 2048 x 21841 x 1024 418 us against 392. x'
//    is laid out once a call, since rows that do not count have to be zeros in it.
//  * d is rounded to bf16 before it is scaled (and divided by 1 - e): a label's entry p - 1 then rounds the
//    same whatever the batch size, and the scale is applied to the fp32 sums. Only an upstream gradient for
//    each row goes into d, since the sum over n cannot apply it.
//  * a row whose label is ignored (or lies outside [0, V)) takes no part: its d is zero and so is its
//    row of x', whatever x holds there.
//  * sums that split an axis go through fp32 slabs added in a fixed order: no atomics, the same bits
//    every time.
//
// Measured, bf16 weight and no bias: 8192 rows x 65536 classes x 2048 wide 6.9 to 7.1 ms from machine to machine: the statistics
// 1.73 (1.27 PFLOP/s), d 1.92 (1.14: its 1 GB of stores is not hidden), dx and dw 3.21 (1.37). 771 x 20011 x 1021
// 245 us: packing 16, statistics 52, d 62, dx and dw 94 + 7 (670 TFLOP/s, 128 x 128 tiles). 256 x 1000 x 2048: 9 + 5, 12,
// 12 us in 32 x 32 and 64 x 64. An fp32 parameter whose gradient is added into its buffer: 7.1 ms, 253 us; a bias costs
// 8192 x 65536 another 0.3 ms.
#include "gemm_tile.h"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

namespace {
using Big = GemmTile<256, 256, 2, 4>;
using Mid = GemmTile<128, 128, 2, 2>;
using Small = GemmTile<64, 64, 2, 2>;
using Thin = ThinTile;

constexpr int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
constexpr int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// tile (row block, column block) of a grid: consecutive ids share an XCD and walk groups of 16 row
// blocks, so that the tiles in flight there reuse both operands from its L2
struct TileAt { int m, n; };
DV_DEVICE TileAt tile_at(int id, int grid, int tm, int tn) {
  id = xcd_remap(id, grid);
  const int per = 16 * tn, g = id / per, r = id - g * per, gs = min(16, tm - g * 16);
  return {g * 16 + r % gs, r / gs};
}

// this wave's LDS writes before, and reads after, stay on their side (the LDS itself works in order)
DV_DEVICE void wave_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

DV_DEVICE bool counted(int64_t label, const DvXent& a) { return label != a.ignore && label >= 0 && label < a.V; }
// d is held divided by this, so that a label's entry is -1 plus a probability and rounds to a step of 1: all
// entries at -0.9 would round the same way
DV_DEVICE float unit(const DvXent& a) { return a.smooth < 1.f ? 1.f - a.smooth : 1.f; }
// the factor of every row's gradient that does not depend on the row
DV_DEVICE float common_scale(const DvXent& a) {
  const float s = a.reduction == DV_XENT_NONE ? 1.f : a.reduction == DV_XENT_SUM ? a.go[0] : a.go[0] / fmaxf(a.total[1], 1.f);
  return s * unit(a);
}

// exp(a - b) as exp2((a - b) * LOG2E): subtracted first, since a class ruled out by the type's lowest
// value leaves the type's range where the product comes first
constexpr float LOG2E = 1.44269504f;
DV_DEVICE float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// acc + bias, -inf behind the last class
template <class T, int BM>
DV_DEVICE void add_bias(T& t, const DvXent& a, int v0) {
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float b = a.bias[min(v0 + t.row(i, r), a.V - 1)];
#pragma unroll
        for (int j = 0; j < T::TN; ++j) t.acc[i][j][r] += b;
      }
      __builtin_amdgcn_sched_barrier(0);  // 16 loads at a time: all of them at once spill
    }
  }
  if (v0 + BM > a.V) {
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) t.acc[i][j][r] = v0 + t.row(i, r) < a.V ? t.acc[i][j][r] : -INFINITY;
  }
}

// ---------------------------------------------------------------------------------------- forward
template <class T, int BM, int BN, int WM>
__global__ __launch_bounds__(T::NTHREADS, T::NTHREADS / 256) void stats_kernel(DvXent a, float2* __restrict__ part,
                                                                               float* __restrict__ psum,
                                                                               float* __restrict__ at_label) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tm = (a.V + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
  const TileAt at = tile_at(blockIdx.x, gridDim.x, tm, tn);
  const int v0 = at.m * BM, n0 = at.n * BN;
  T t;
  t.run({a.w + (int64_t)v0 * a.ldw, a.ldw, a.V - v0}, {a.x + (int64_t)n0 * a.ldx, a.ldx, a.N - n0}, a.D / 64, smem);
  if (!t.active()) return;
  add_bias<T, BM>(t, a, v0);
  const int vw = v0 + t.wm * T::TM * 32;  // the wave's columns: [vw, vw + 32 TM)
#pragma unroll
  for (int j = 0; j < T::TN; ++j) {
    const int n = n0 + t.col(j);
    const int64_t label = n < a.N ? a.labels[n] : -1;
    const bool here = counted(label, a) && label >= vw && label < vw + T::TM * 32;
    if (__any(here)) {  // few of many pieces of the vocabulary hold a label of the wave's rows
      const int rel = here ? (int)label - vw - 4 * (t.lane >> 5) : -1;
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (rel == i * 32 + (r & 3) + 8 * (r >> 2)) at_label[n] = t.acc[i][j][r];
    }
    float top = -INFINITY, s = 0.f;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, t.acc[i][j][r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s += exp2_fast((t.acc[i][j][r] - ref) * LOG2E);
    s += __shfl_xor(s, 32, 64);
    float sum = 0.f;
    if (psum) {
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += v0 + t.row(i, r) < a.V ? t.acc[i][j][r] - ref : 0.f;
      sum += __shfl_xor(sum, 32, 64);
    }
    if (t.lane < 32 && n < a.N) {
      const int64_t o = (int64_t)(at.m * WM + t.wm) * a.N + n;
      part[o] = {top, s};
      if (psum) psum[o] = sum;
    }
  }
}

// ROWS rows a block, 1024 / ROWS strips of the parts: (largest logit, log2 of the sum of exponentials
// above it) of each row, kept apart so that a large common offset costs no precision, and its loss; the
// block's (sum, count), or where one block holds every row the result itself
template <int ROWS>
__global__ __launch_bounds__(1024) void join_kernel(DvXent a, const float2* __restrict__ part, const float* __restrict__ psum,
                                                    const float* __restrict__ at_label, int parts, int cols_a_part,
                                                    float2* __restrict__ lse, float* __restrict__ loss,
                                                    float2* __restrict__ blocks, float* __restrict__ out,
                                                    float* __restrict__ total) {
  constexpr int STRIPS = 1024 / ROWS, GROUPS = ROWS < 64 ? 16 : STRIPS;  // a wave joins its own strips first
  __shared__ float sh[3][GROUPS][ROWS];
  __shared__ float red[2][ROWS < 64 ? 1 : ROWS / 64];
  const int j = threadIdx.x % ROWS, k = threadIdx.x / ROWS, group = ROWS < 64 ? threadIdx.x >> 6 : k;
  const int64_t n = (int64_t)blockIdx.x * ROWS + j;
  float top = -INFINITY;
  if (n < a.N)
#pragma unroll 8
    for (int p = k; p < parts; p += STRIPS) top = fmaxf(top, part[(int64_t)p * a.N + n].x);
#pragma unroll
  for (int o = ROWS; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  sh[0][group][j] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) top = fmaxf(top, sh[0][i][j]);
  float s = 0.f, sum = 0.f;  // of exp(l - top), of l - top
  if (n < a.N)
#pragma unroll 8
    for (int p = k; p < parts; p += STRIPS) {
      const float2 q = part[(int64_t)p * a.N + n];
      s += q.x == -INFINITY ? q.y : q.y * exp2_fast((q.x - top) * LOG2E);  // (-inf: 0, or NaN)
      if (psum) {
        const int cols = min(a.V - p * cols_a_part, cols_a_part);
        if (cols > 0) sum += psum[(int64_t)p * a.N + n] + (q.x == -INFINITY ? 0.f : cols * (q.x - top));
      }
    }
#pragma unroll
  for (int o = ROWS; o < 64; o <<= 1) {
    s += __shfl_xor(s, o, 64);
    sum += __shfl_xor(sum, o, 64);
  }
  sh[1][group][j] = s;
  sh[2][group][j] = sum;
  __syncthreads();
  float l = 0.f, one = 0.f;
  if (k == 0) {
    float tot = 0.f, all = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) { tot += sh[1][i][j]; all += sh[2][i][j]; }
    if (n < a.N) {
      if (counted(a.labels[n], a)) {
        one = 1.f;
        l = logf(tot) + (1.f - a.smooth) * (top - at_label[n]);
        if (psum) l -= a.smooth * (all / a.V);
      }
      if (lse) lse[n] = {top, log2f(tot)};
      if (loss) loss[n] = l;
    }
  }
  if (!out) return;
  l = wave_sum(l);
  one = wave_sum(one);
  if (threadIdx.x < (ROWS < 64 ? 64 : ROWS) && (threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = l;
    red[1][threadIdx.x >> 6] = one;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    l = one = 0.f;
#pragma unroll
    for (int i = 0; i < (ROWS < 64 ? 1 : ROWS / 64); ++i) { l += red[0][i]; one += red[1][i]; }
    if (gridDim.x > 1) {
      blocks[blockIdx.x] = {l, one};
    } else {
      total[0] = l;
      total[1] = one;
      *out = a.reduction == DV_XENT_MEAN ? l / fmaxf(one, 1.f) : l;
    }
  }
}

// out = the loss, total = (sum, count)
__global__ __launch_bounds__(256) void total_kernel(const float2* __restrict__ blocks, int n, int mean,
                                                    float* __restrict__ out, float* __restrict__ total) {
  __shared__ float sh[4];
  float s = 0.f, c = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) { s += blocks[i].x; c += blocks[i].y; }
  s = block_sum<256>(s, sh);
  c = block_sum<256>(c, sh);
  if (threadIdx.x == 0) {
    total[0] = s;
    total[1] = c;
    *out = mean ? s / fmaxf(c, 1.f) : s;
  }
}

// --------------------------------------------------------------------------------------- backward
// x' [width][ldt] of the rows that count, 0 in the others and up to ldt; 64 x 64 by 256 threads. 16-byte
// loads and stores; a column of the LDS image is gathered by 2 bytes.
struct Transpose {
  u16* to;
  int64_t ldt;
  int blocks;  // (ldt / 64) x ceil(width / 64)
};
constexpr int TRANSPOSE_LDS = 64 * 74 * 2;  // 37 banks a row: gathers of 8 rows apart do not meet
DV_DEVICE void transpose_block(const DvXent& x, const Transpose& t, int id, int tid, char* smem) {
  u16(*sh)[74] = reinterpret_cast<u16(*)[74]>(smem);
  const bool any = id < t.blocks;
  const int across = any ? (int)(t.ldt / 64) : 1, r0 = id % across * 64, c0 = id / across * 64;
  if (any) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // rows of x hold whole 64-column blocks (zeros from `width` on)
      const int r = e * 32 + (tid >> 3), c = (tid & 7) * 8;
      uint4 d{0, 0, 0, 0};
      if (r0 + r < x.N && counted(x.labels[r0 + r], x))
        d = *reinterpret_cast<const uint4*>(x.x + (int64_t)(r0 + r) * x.ldx + c0 + c);
      uint32_t* to = reinterpret_cast<uint32_t*>(&sh[r][c]);
      to[0] = d.x; to[1] = d.y; to[2] = d.z; to[3] = d.w;
    }
  }
  __syncthreads();
  if (!any) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int c = e * 32 + (tid >> 3), r = (tid & 7) * 8;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)sh[r + 2 * k][c] | (uint32_t)sh[r + 2 * k + 1][c] << 16;
    if (c0 + c < x.width) *reinterpret_cast<uint4*>(t.to + (int64_t)(c0 + c) * t.ldt + r0 + r) = uint4{w[0], w[1], w[2], w[3]};
  }
}
__global__ __launch_bounds__(256) void transpose_kernel(DvXent x, Transpose t) {
  __shared__ __attribute__((aligned(16))) char smem[TRANSPOSE_LDS];
  transpose_block(x, t, blockIdx.x, threadIdx.x, smem);
}

// d (times its gradient, where each row has one of its own) of the piece [p0, p0 + pv) of the vocabulary:
// P [ldt][pvp], zero from N and from pv on; db partial sums [n block and wave][pv]
template <class T, int BM, int BN, int WN>
__global__ __launch_bounds__(T::NTHREADS, T::NTHREADS / 256) void grad_kernel(DvXent a, const float2* __restrict__ lse, int p0,
                                                                              int pv, int pvp, u16* __restrict__ P, int ldt,
                                                                              float* __restrict__ pbias, int tiles,
                                                                              Transpose xt) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if ((int)blockIdx.x >= tiles) {  // the blocks behind the tiles lay out x', which the next launch reads
    const int sub = threadIdx.x >> 8;
    transpose_block(a, xt, (blockIdx.x - tiles) * (T::NTHREADS / 256) + sub, threadIdx.x & 255, smem + sub * TRANSPOSE_LDS);
    return;
  }
  constexpr int PITCH = 144;  // bytes: 64 bf16 + 16, without bank conflicts
  constexpr int MG = T::TM < 2 ? 1 : 2, MW = 32 * MG, NW = 32 * T::TN;
  // tiles up to pvp and ldt: where a tile is half of 64 the last one may hold nothing but zeros
  const int tm = (pvp + BM - 1) / BM, tn = (ldt + BN - 1) / BN;
  const TileAt at = tile_at(blockIdx.x, tiles, tm, tn);
  const int v0 = at.m * BM, n0 = at.n * BN;  // v: within the piece
  T t;
  t.run({a.w + (int64_t)(p0 + min(v0, pv - 1)) * a.ldw, a.ldw, max(pv - v0, 1)},
        {a.x + (int64_t)min(n0, a.N - 1) * a.ldx, a.ldx, max(a.N - n0, 1)}, a.D / 64, smem);
  if (!t.active()) return;
  add_bias<T, BM>(t, a, p0 + v0);
  const float inv = 1.f / unit(a), off = a.smooth / a.V * inv, hot = a.smooth < 1.f ? 1.f : 0.f;
  const int vw0 = p0 + v0 + t.wm * T::TM * 32;
#pragma unroll
  for (int j = 0; j < T::TN; ++j) {
    const int n = n0 + t.col(j);
    const int64_t label = n < a.N ? a.labels[n] : -1;
    const bool use = n < a.N && counted(label, a);
    const float2 z = use ? lse[n] : float2{0.f, 0.f};
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) t.acc[i][j][r] = fmaf(exp2_fast(fmaf(t.acc[i][j][r] - z.x, LOG2E, -z.y)), inv, -off);
    const bool here = use && label >= vw0 && label < vw0 + T::TM * 32;
    if (__any(here)) {
      const int rel = here ? (int)label - vw0 - 4 * (t.lane >> 5) : -1;
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) t.acc[i][j][r] -= rel == i * 32 + (r & 3) + 8 * (r >> 2) ? hot : 0.f;
    }
    if (a.reduction == DV_XENT_NONE) {
      const float row = use ? a.go[n] : 0.f;
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) t.acc[i][j][r] *= row;
    }
    if (__any(!use)) {  // whatever x holds in rows that do not count
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) t.acc[i][j][r] = use ? t.acc[i][j][r] : 0.f;
    }
    if (v0 + BM > pv) {  // behind the piece's end
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) t.acc[i][j][r] = v0 + t.row(i, r) < pv ? t.acc[i][j][r] : 0.f;
    }
  }
  if (pbias) {  // over the wave's rows n: in registers, then over the 32 lanes of a column of blocks
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < T::TN; ++j) s += t.acc[i][j][r];
        s = row16_sum(s);
        s += __shfl_xor(s, 16, 64);
        const int v = v0 + t.row(i, r);
        if ((t.lane & 31) == 0 && v < pv) pbias[(int64_t)(at.n * WN + t.wn) * pv + v] = s;
      }
  }
  // rows of P through this wave's own part of LDS, MW columns of the vocabulary at a time
  char* mine = smem + t.wave * NW * PITCH;
#pragma unroll
  for (int h = 0; h < T::TM / MG; ++h) {
    const int vw = v0 + (t.wm * T::TM + h * MG) * 32, nw = n0 + t.wn * T::TN * 32;
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int i = 0; i < MG; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x16& c = t.acc[h * MG + i][j];
          *reinterpret_cast<uint2*>(mine + (j * 32 + (t.lane & 31)) * PITCH + (i * 32 + 8 * q + 4 * (t.lane >> 5)) * 2) =
              uint2{pack2bf(c[4 * q], c[4 * q + 1]), pack2bf(c[4 * q + 2], c[4 * q + 3])};
        }
    wave_sync();
#pragma unroll
    for (int e = 0; e < NW * MW / 512; ++e) {
      const int w = e * 64 + t.lane, n = w / (MW / 8), c = w % (MW / 8) * 8;
      const uint4 d = *reinterpret_cast<const uint4*>(mine + n * PITCH + c * 2);
      if (nw + n < ldt && vw + c < pvp) *reinterpret_cast<uint4*>(P + (int64_t)(nw + n) * pvp + vw + c) = d;
    }
    wave_sync();
  }
}

// out[n][m] = scale * sum_k A[m][k] B[n][k] over this split's K-tiles. dx: A = w' and B = d; dw: A = x' and
// B = d'. w and d are read as they lie, k by k for A and for B.
struct OutArgs {
  const u16 *a, *b;
  int64_t lda, ldb;
  int M, N, ktiles, splits;
  float* slab;       // [split][N][M], added to where slab_add; or null: `out` itself
  int slab_add;
  void* out;         // [N][M], bf16 or fp32
  int out_f32, out_add;
  int by_row;        // 0 in rows n whose label does not count
  int deep;          // valid k
};
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

DV_DEVICE float out_scale(const DvXent& x, bool by_row, int64_t n, float common) {
  return !by_row || counted(x.labels[n], x) ? common : 0.f;
}
DV_DEVICE void put4(void* out, int f32, int add, int64_t o, int left, f32x4 v) {
  if (f32) {
    float* p = reinterpret_cast<float*>(out) + o;
    if (left >= 4) {
      if (add) v += *reinterpret_cast<const f32x4_a4*>(p);
      *reinterpret_cast<f32x4_a4*>(p) = v;
    } else {
      for (int e = 0; e < left; ++e) p[e] = add ? p[e] + v[e] : v[e];
    }
  } else {
    u16* p = reinterpret_cast<u16*>(out) + o;
    if (left >= 4) *reinterpret_cast<u32x2_a2*>(p) = u32x2_a2{pack2bf(v[0], v[1]), pack2bf(v[2], v[3])};
    else
      for (int e = 0; e < left; ++e) p[e] = f2bf(v[e]);
  }
}

// db[v] (+)= scale * sum of the partial rows, 64 columns a block
struct BiasArgs {
  const float* part;
  int parts, pv;
  float* db;
  int add;
};
DV_DEVICE void fold_bias(const DvXent& x, const BiasArgs& b, int block, float* sh) {
  const int j = threadIdx.x & 63, k = threadIdx.x >> 6, v = block * 64 + j;
  float s = 0.f;
  if (v < b.pv && k < 4)
    for (int p = k; p < b.parts; p += 4) s += b.part[(int64_t)p * b.pv + v];
  if (k < 4) sh[k * 64 + j] = s;
  __syncthreads();
  if (k == 0 && v < b.pv) {
    s = ((sh[j] + sh[64 + j]) + (sh[128 + j] + sh[192 + j])) * common_scale(x);
    b.db[v] = b.add ? b.db[v] + s : s;
  }
}

// tile `id` of g
template <class T, int BM, int BN, bool DX>
DV_DEVICE void out_tile(const DvXent& x, const OutArgs& g, int id, char* smem) {
  constexpr int PITCH = 144, NW = 32 * T::TN;
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  const int tiles = tm * tn, split = id / tiles;
  const TileAt at = tile_at(id - split * tiles, tiles, tm, tn);
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int k0 = (int)((int64_t)g.ktiles * split / g.splits), k1 = (int)((int64_t)g.ktiles * (split + 1) / g.splits);
  const int64_t k = (int64_t)k0 * 64;
  const int deep = g.deep - k0 * 64;
  const GemmOperand a{g.a + (DX ? k * g.lda + m0 : m0 * g.lda + k), g.lda, g.M - m0, deep};
  const GemmOperand b{g.b + (DX ? n0 * g.ldb + k : k * g.ldb + n0), g.ldb, g.N - n0, deep};
  T t;
  t.run(a, b, k1 - k0, smem);
  const float common = g.slab ? 1.f : common_scale(x);
  char* mine = smem + t.wave * NW * PITCH;
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    const int mw = m0 + (t.wm * T::TM + i) * 32, nw = n0 + t.wn * NW;
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x16& c = t.acc[i][j];
        *reinterpret_cast<f32x4*>(mine + (j * 32 + (t.lane & 31)) * PITCH + (8 * q + 4 * (t.lane >> 5)) * 4) =
            f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]};
      }
    wave_sync();
#pragma unroll
    for (int e = 0; e < NW / 8; ++e) {
      const int n = nw + e * 8 + (t.lane >> 3), m = mw + (t.lane & 7) * 4;
      f32x4 v = *reinterpret_cast<const f32x4*>(mine + (e * 8 + (t.lane >> 3)) * PITCH + (t.lane & 7) * 16);
      if (n >= g.N || m >= g.M) continue;
      const int64_t o = (int64_t)n * g.M + m;
      if (g.slab) {
        put4(g.slab + (int64_t)split * g.N * g.M, 1, g.slab_add, o, g.M - m, v);
      } else {
        const float s = out_scale(x, g.by_row, n, common);
        put4(g.out, g.out_f32, g.out_add, o, g.M - m, s == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v * s);
      }
    }
    wave_sync();
  }
}

// The products behind a piece's d, and the fold of its bias gradient, in one launch: blocks [0, b0) compute
// dx, [b0, b0 + b1) dw, the rest the bias.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, WM * WN / 4) void out_kernel(DvXent x, OutArgs gx, OutArgs gw, BiasArgs bias, int b0,
                                                                        int b1) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int id = blockIdx.x;
  if (id < b0) out_tile<GemmTile<BM, BN, WM, WN, true, false>, BM, BN, true>(x, gx, id, smem);
  else if (id < b0 + b1) out_tile<GemmTile<BM, BN, WM, WN, false, true>, BM, BN, false>(x, gw, id - b0, smem);
  else fold_bias(x, bias, id - b0 - b1, reinterpret_cast<float*>(smem));
}

// out[n][m] = scale * sum over splits of the slab
__global__ __launch_bounds__(256) void reduce_kernel(DvXent x, OutArgs g) {
  const int64_t all = (int64_t)g.N * g.M;
  const float common = common_scale(x);
  const int per = (g.M + 3) / 4;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < (int64_t)g.N * per; u += (int64_t)gridDim.x * 256) {
    const int64_t n = u / per;
    const int m = (int)(u - n * per) * 4, left = g.M - m;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < g.splits; ++s) {
      const float* p = g.slab + s * all + n * g.M + m;
      if (left >= 4) v += *reinterpret_cast<const f32x4_a4*>(p);
      else
        for (int e = 0; e < left; ++e) v[e] += p[e];
    }
    const float s = out_scale(x, g.by_row, n, common);
    put4(g.out, g.out_f32, g.out_add, n * g.M + m, left, s == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v * s);
  }
}

// dst [rows][ldd] bf16 = src [rows][cols] (bf16 or fp32), zero behind cols; one or two matrices a launch
template <class S>
DV_DEVICE uint4 pack8(const S* p, int left) {
  uint32_t w[4] = {};
  if (left >= 8) {  // rows start at any element
    if constexpr (sizeof(S) == 2) {
      const u32x4_a2 q = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = q[e];
    } else {
      const f32x4_a4 q0 = *reinterpret_cast<const f32x4_a4*>(p), q1 = *reinterpret_cast<const f32x4_a4*>(p + 4);
      w[0] = pack2bf(q0[0], q0[1]); w[1] = pack2bf(q0[2], q0[3]);
      w[2] = pack2bf(q1[0], q1[1]); w[3] = pack2bf(q1[2], q1[3]);
    }
  } else {
    for (int e = 0; e < left; ++e) {
      uint32_t v;
      if constexpr (sizeof(S) == 2) v = p[e];
      else v = f2bf(p[e]);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k == e >> 1) w[k] |= v << (16 * (e & 1));
    }
  }
  return uint4{w[0], w[1], w[2], w[3]};
}
__global__ __launch_bounds__(256) void pack_kernel(DvPack m0, DvPack m1, int b0) {
  const bool second = (int)blockIdx.x >= b0;
  const DvPack& m = second ? m1 : m0;
  const int64_t block = second ? blockIdx.x - b0 : blockIdx.x, grid = second ? gridDim.x - b0 : b0, per = m.ldd / 8;
  for (int64_t u = block * 256 + threadIdx.x; u < m.rows * per; u += grid * 256) {
    const int64_t r = u / per;
    const int c = (int)(u - r * per) * 8;
    const uint4 d = m.bf16 ? pack8(reinterpret_cast<const u16*>(m.src) + r * m.lds + c, m.cols - c)
                           : pack8(reinterpret_cast<const float*>(m.src) + r * m.lds + c, m.cols - c);
    *reinterpret_cast<uint4*>(reinterpret_cast<u16*>(m.dst) + r * m.ldd + c) = d;
  }
}

// ------------------------------------------------------------------------------------------- host
// Tile and split of an M x N x (64 ktiles) product: the least time by a model of a K-tile's time on a full
// CU (throughput) and alone (latency) and of a block's ends, its constants fitted to times of these kernels at
// 1 .. 8192 rows, 64 .. 65536 classes and widths of 64 .. 2500.
struct Plan { int form, splits; double us; };
constexpr int FORMS = 4, OUT_FORMS = 3, FORM_M[FORMS] = {256, 128, 64, 32}, FORM_N[FORMS] = {256, 128, 64, 32};
enum Ends { STATS, GRAD, OUT };  // what a block does behind its sums
Plan plan_form(int f, int64_t M, int64_t N, int ktiles, bool may_split, Ends ends) {
  // us a K-tile: on a CU with as many blocks as fit (AT_ONCE), and alone; us of a block's two ends
  constexpr double FULL[FORMS] = {1.6, 0.58, 0.25, 0.2}, ALONE[FORMS] = {1.6, 0.65, 0.35, 0.2};
  constexpr double ENDS[3][FORMS] = {{4, 2.5, 2, 2.5}, {16, 9, 4, 5}, {6, 2.5, 1}};
  constexpr int AT_ONCE[FORMS] = {1, 2, 5, 2};
  Plan best{f, 1, 1e30};
  const int64_t tiles = (int64_t)cdiv(M, FORM_M[f]) * cdiv(N, FORM_N[f]);
  for (int s = 1; s <= (may_split ? std::min(ktiles, 32) : 1); ++s) {
    const double k = cdiv(ktiles, s), blocks = (double)tiles * s;
    const double per_cu = f == 0 ? std::ceil(blocks / 256) : std::max(1.0, blocks / 256);
    const double rounds = std::ceil(blocks / (256 * AT_ONCE[f]));
    const double us = ENDS[ends][f] * rounds + std::max(per_cu * k * FULL[f], k * ALONE[f]) +
                      (s > 1 ? 4.0 + s * (double)M * N * 8 / 4e6 : 0.0);
    if (us < best.us) best = {f, s, us};
  }
  return best;
}
// a launch holds less than 2^32 threads
bool fits(int f, int64_t M, int64_t N) {
  constexpr int THREADS[FORMS] = {Big::NTHREADS, Mid::NTHREADS, Small::NTHREADS, Thin::NTHREADS};
  return (int64_t)cdiv(M, FORM_M[f]) * cdiv(N, FORM_N[f]) * THREADS[f] < 1LL << 32;
}
Plan plan(int64_t M, int64_t N, int ktiles, Ends ends) {
  Plan best = plan_form(0, M, N, ktiles, false, ends);
  for (int f = 1; f < FORMS; ++f) {
    const Plan p = plan_form(f, M, N, ktiles, false, ends);
    if (p.us < best.us && fits(f, M, N)) best = p;
  }
  return best;
}

// f(tile, BM, BN, WM, WN); the products behind d take the first three
template <int V>
using Int = std::integral_constant<int, V>;
template <class F>
void with_wide_tile(int form, F&& f) {
  if (form == 0) f(Big{}, Int<256>{}, Int<256>{}, Int<2>{}, Int<4>{});
  else if (form == 1) f(Mid{}, Int<128>{}, Int<128>{}, Int<2>{}, Int<2>{});
  else f(Small{}, Int<64>{}, Int<64>{}, Int<2>{}, Int<2>{});
}
template <class F>
void with_tile(int form, F&& f) {
  if (form == 3) f(Thin{}, Int<32>{}, Int<32>{}, Int<1>{}, Int<1>{});
  else with_wide_tile(form, f);
}
constexpr int FORM_WM[FORMS] = {2, 2, 2, 1}, FORM_WN[FORMS] = {4, 2, 2, 1};

// more than 64 KB of LDS, allowed once for each kernel and device
template <class K>
void allow_lds(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  (void)hipGetDevice(&dev);
  if (done[dev & 63]) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  done[dev & 63] = true;
}

struct FwdLayout { Plan p; int parts, rows, blocks; int64_t part, psum, label, block, bytes; };
FwdLayout fwd_layout(const DvXent& a) {
  FwdLayout l;
  l.p = plan(a.V, a.N, a.D / 64, STATS);
  l.parts = cdiv(a.V, FORM_M[l.p.form]) * FORM_WM[l.p.form];
  l.rows = a.N <= 256 && l.parts <= 128 ? 256 : 16;  // small: one block joins every row
  l.blocks = cdiv(a.N, l.rows);
  int64_t at = 0;
  auto take = [&](int64_t b) { const int64_t o = at; at += up(b, 256); return o; };
  l.part = take((int64_t)l.parts * a.N * 8);
  l.psum = take(a.smooth > 0.f ? (int64_t)l.parts * a.N * 4 : 0);
  l.label = take((int64_t)a.N * 4);
  l.block = take((int64_t)l.blocks * 8);
  l.bytes = at;
  return l;
}

struct BwdLayout {
  int piece;           // columns of the vocabulary at a time
  Plan pg, px, pw;     // the logits again, dx, dw
  int ldt;             // rows rounded up to 64
  int bias_parts;
  bool dx_slab;
  int64_t P, xt, sx, sw, pb, bytes;
};
constexpr int64_t PIECE_BYTES = 1LL << 30;  // a piece's d
BwdLayout bwd_layout(const DvXent& a, bool need_x, bool need_w, bool need_b) {
  BwdLayout l;
  l.ldt = (int)up(a.N, 64);
  const int64_t most = std::max<int64_t>(PIECE_BYTES / (2 * l.ldt) / 256 * 256, 256);
  const int pieces = cdiv(a.V, most);
  l.piece = (int)std::min<int64_t>(up(cdiv(a.V, pieces), 256), a.V);
  l.pg = plan(l.piece, a.N, a.D / 64, GRAD);
  // dx and dw run in one launch and share a tile form, whichever of them is wanted: a gradient's bits do
  // not depend on which others are asked for
  double least = 1e30;
  for (int f = 0; f < OUT_FORMS; ++f) {
    const Plan x = plan_form(f, a.width, a.N, cdiv(l.piece, 64), true, OUT),
               w = plan_form(f, a.width, l.piece, cdiv(a.N, 64), true, OUT);
    if (x.us + w.us < least) { least = x.us + w.us; l.px = x; l.pw = w; }
  }
  l.bias_parts = cdiv(l.ldt, FORM_N[l.pg.form]) * FORM_WN[l.pg.form];
  l.dx_slab = l.px.splits > 1 || pieces > 1;
  int64_t at = 0;
  auto take = [&](int64_t b) { const int64_t o = at; at += up(b, 256); return o; };
  l.P = take(l.ldt * up(l.piece, 64) * 2);
  l.xt = take(need_w ? (int64_t)a.width * l.ldt * 2 : 0);
  l.sx = take(need_x && l.dx_slab ? (int64_t)l.px.splits * a.N * a.width * 4 : 0);
  l.sw = take(need_w && l.pw.splits > 1 ? (int64_t)l.pw.splits * l.piece * a.width * 4 : 0);
  l.pb = take(need_b ? (int64_t)l.bias_parts * l.piece * 4 : 0);
  l.bytes = at;
  return l;
}

bool sane(const DvXent& a) {
  return a.N > 0 && a.N <= DV_XENT_MAX_ROWS && a.V > 0 && a.V <= DV_XENT_MAX_CLASSES &&
         (int64_t)cdiv(a.V, 32) * cdiv(a.N, 32) < 0x7fffffff && a.D > 0 && a.D % 64 == 0 && a.width > 0 && a.width <= a.D &&
         a.ldx >= a.D && a.ldw >= a.D && a.ldx % 8 == 0 && a.ldw % 8 == 0 && a.ldx <= (1 << 22) && a.ldw <= (1 << 22) &&
         ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0;
}

void launch_out(const DvXent& a, int form, const OutArgs& gx, const OutArgs& gw, const BiasArgs& bias, hipStream_t st) {
  with_wide_tile(form, [&](auto tile, auto bm, auto bn, auto wm, auto wn) {
    using T = decltype(tile);
    constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    const int b0 = cdiv(gx.M, BM) * cdiv(gx.N, BN) * gx.splits, b1 = cdiv(gw.M, BM) * cdiv(gw.N, BN) * gw.splits;
    const int b2 = bias.db ? cdiv(bias.pv, 64) : 0;
    if (b0 + b1 + b2 == 0) return;
    static bool done[64];
    allow_lds(out_kernel<BM, BN, WM, WN>, T::LDS, done);
    out_kernel<BM, BN, WM, WN><<<(unsigned)(b0 + b1 + b2), T::NTHREADS, T::LDS, st>>>(a, gx, gw, bias, b0, b1);
  });
}
void launch_reduce(const DvXent& a, const OutArgs& g, hipStream_t st) {
  const int64_t units = (int64_t)g.N * ((g.M + 3) / 4);
  reduce_kernel<<<(unsigned)std::min<int64_t>((units + 255) / 256, 4096), 256, 0, st>>>(a, g);
}
}  // namespace

int64_t dv_linear_xent_fwd_bytes(const DvXent& a) {
  const FwdLayout l = fwd_layout(a);
  return fits(l.p.form, a.V, a.N) ? l.bytes : -1;
}
int64_t dv_linear_xent_bwd_bytes(const DvXent& a, int need_x, int need_w, int need_b) {
  return bwd_layout(a, need_x, need_w, need_b).bytes;
}

int dv_linear_xent_fwd(const DvXent& a, void* ws, float* lse, float* loss_rows, float* total, float* out, hipStream_t st) {
  if (!sane(a)) return -1;
  const FwdLayout l = fwd_layout(a);
  if (!fits(l.p.form, a.V, a.N)) return -1;
  char* w = reinterpret_cast<char*>(ws);
  float2* part = reinterpret_cast<float2*>(w + l.part);
  float* psum = a.smooth > 0.f ? reinterpret_cast<float*>(w + l.psum) : nullptr;
  float* at_label = reinterpret_cast<float*>(w + l.label);
  float2* blocks = out ? reinterpret_cast<float2*>(w + l.block) : nullptr;
  with_tile(l.p.form, [&](auto tile, auto bm, auto bn, auto wm, auto) {
    using T = decltype(tile);
    constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value;
    static bool done[64];
    allow_lds(stats_kernel<T, BM, BN, WM>, T::LDS, done);
    stats_kernel<T, BM, BN, WM><<<(unsigned)(cdiv(a.V, BM) * cdiv(a.N, BN)), T::NTHREADS, T::LDS, st>>>(a, part, psum, at_label);
  });
  const int cols = FORM_M[l.p.form] / FORM_WM[l.p.form];
  float2* lse2 = reinterpret_cast<float2*>(lse);
  if (l.rows == 256) join_kernel<256><<<l.blocks, 1024, 0, st>>>(a, part, psum, at_label, l.parts, cols, lse2, loss_rows, blocks, out, total);
  else join_kernel<16><<<l.blocks, 1024, 0, st>>>(a, part, psum, at_label, l.parts, cols, lse2, loss_rows, blocks, out, total);
  if (out && l.blocks > 1) total_kernel<<<1, 256, 0, st>>>(blocks, l.blocks, a.reduction == DV_XENT_MEAN, out, total);
  return 0;
}

int dv_linear_xent_bwd(const DvXent& a, void* ws, const float* lse, void* dx, void* dw, int dw_f32, int dw_add, float* db,
                       int db_add, hipStream_t st) {
  if (!sane(a)) return -1;
  const bool need_w = dw != nullptr, need_x = dx != nullptr;
  const BwdLayout l = bwd_layout(a, need_x, need_w, db != nullptr);
  char* w = reinterpret_cast<char*>(ws);
  u16 *P = reinterpret_cast<u16*>(w + l.P), *xt = reinterpret_cast<u16*>(w + l.xt);
  float* pb = db ? reinterpret_cast<float*>(w + l.pb) : nullptr;
  OutArgs gx{};
  for (int p0 = 0; p0 < a.V; p0 += l.piece) {
    const int pv = std::min(l.piece, a.V - p0), pvp = (int)up(pv, 64);
    const Transpose tx{xt, l.ldt, need_w && p0 == 0 ? l.ldt / 64 * cdiv(a.width, 64) : 0};
    // in the gradient's launch, but for the largest tiles: a block there takes a CU's LDS, whatever it does
    const bool apart = l.pg.form == 0;
    if (apart && tx.blocks) transpose_kernel<<<(unsigned)tx.blocks, 256, 0, st>>>(a, tx);
    with_tile(l.pg.form, [&](auto tile, auto bm, auto bn, auto, auto wn) {
      using T = decltype(tile);
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WN = decltype(wn)::value;
      static bool done[64];
      allow_lds(grad_kernel<T, BM, BN, WN>, T::LDS, done);
      const int tiles = cdiv(pvp, BM) * cdiv(l.ldt, BN), beside = apart ? 0 : cdiv(tx.blocks, T::NTHREADS / 256);
      grad_kernel<T, BM, BN, WN><<<(unsigned)(tiles + beside), T::NTHREADS, T::LDS, st>>>(
          a, reinterpret_cast<const float2*>(lse), p0, pv, pvp, P, l.ldt, pb, tiles, tx);
    });
    OutArgs gw{};
    if (need_x)
      gx = OutArgs{a.w + (int64_t)p0 * a.ldw, P, a.ldw, pvp, a.width, a.N, pvp / 64, std::min(l.px.splits, pvp / 64),
                   l.dx_slab ? reinterpret_cast<float*>(w + l.sx) : nullptr, p0 > 0, dx, 0, 0, 1, pv};
    if (need_w) {
      char* to = reinterpret_cast<char*>(dw) + (int64_t)p0 * a.width * (dw_f32 ? 4 : 2);
      gw = OutArgs{xt, P, l.ldt, pvp, a.width, pv, l.ldt / 64, l.pw.splits,
                   l.pw.splits > 1 ? reinterpret_cast<float*>(w + l.sw) : nullptr, 0, to, dw_f32, dw_add, 0, l.ldt};
    }
    const BiasArgs gb{pb, l.bias_parts, pv, db ? db + p0 : nullptr, db_add};
    launch_out(a, l.px.form, gx, gw, gb, st);
    if (need_w && l.pw.splits > 1) launch_reduce(a, gw, st);
  }
  if (need_x && l.dx_slab) {
    gx.splits = l.px.splits;
    launch_reduce(a, gx, st);
  }
  return 0;
}

int dv_pack_rows(const DvPack& m0, const DvPack& m1, hipStream_t st) {
  int grid[2];
  const DvPack* all[2] = {&m0, &m1};
  for (int i = 0; i < 2; ++i) {
    const DvPack& m = *all[i];
    grid[i] = 0;
    if (!m.rows) continue;
    if (m.rows < 0 || m.cols <= 0 || m.ldd % 8 || m.ldd < m.cols || m.lds < m.cols) return -1;
    grid[i] = (int)std::min<int64_t>((m.rows * (m.ldd / 8) + 255) / 256, 8192);
  }
  if (grid[0] + grid[1]) pack_kernel<<<(unsigned)(grid[0] + grid[1]), 256, 0, st>>>(m0, m1, grid[0]);
  return 0;
}
