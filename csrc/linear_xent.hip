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
//  * backward, for each piece of the vocabulary: the product again, its epilogue writes d in bf16 both
//    ways round ([n][v] and [v][n]), because each of the two products that follow wants its own sum
//    index contiguous; then dx += d w and dw = d' x. x' and the piece of w' are laid out once a call.
//  * d is rounded to bf16 before it is scaled: (p - 1) is then exact to half a step whatever the batch
//    size, and the scale is applied to the fp32 sums. Only with an upstream gradient for each row
//    does d' carry it (the sum over n cannot).
//  * a row whose label is ignored (or lies outside [0, V)) takes no part: its d is zero and so is its
//    row of x', whatever x holds there.
//  * sums that split an axis go through fp32 slabs added in a fixed order: no atomics, the same bits
//    every time.
#include "gemm_tile.h"
#include "kernels.h"

#include <algorithm>

namespace {
using Big = GemmTile<256, 256, 2, 4>;
using Mid = GemmTile<128, 128, 2, 2>;
using Small = GemmTile<64, 64, 2, 2>;

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
// the factor of every row's gradient that does not depend on the row
DV_DEVICE float common_scale(const DvXent& a) {
  return a.reduction == DV_XENT_NONE ? 1.f : a.reduction == DV_XENT_SUM ? a.go[0] : a.go[0] / fmaxf(a.total[1], 1.f);
}

// acc + bias, -inf behind the last class; `last`: the tile holds columns behind it
template <class T>
DV_DEVICE void add_bias(T& t, const DvXent& a, int v0) {
  const bool last = v0 + T::TM * 32 * 8 > a.V;  // (conservative: any tile near the end)
  if (!a.bias && !last) return;
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int v = v0 + t.row(i, r);
      const float b = a.bias && v < a.V ? a.bias[v] : 0.f;
#pragma unroll
      for (int j = 0; j < T::TN; ++j) t.acc[i][j][r] = v < a.V ? t.acc[i][j][r] + b : -INFINITY;
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
  add_bias(t, a, v0);
#pragma unroll
  for (int j = 0; j < T::TN; ++j) {
    const int n = n0 + t.col(j);
    const int64_t label = n < a.N ? a.labels[n] : -1;
    const bool use = counted(label, a);
    float top = -INFINITY, s = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float l = t.acc[i][j][r];
        top = fmaxf(top, l);
        if (use && v0 + t.row(i, r) == (int)label) at_label[n] = l;
      }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s += __expf(t.acc[i][j][r] - ref);
    s += __shfl_xor(s, 32, 64);
    if (psum) {
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += v0 + t.row(i, r) < a.V ? t.acc[i][j][r] : 0.f;
      sum += __shfl_xor(sum, 32, 64);
    }
    if (t.lane < 32 && n < a.N) {
      const int64_t o = (int64_t)(at.m * WM + t.wm) * a.N + n;
      part[o] = {top, s};
      if (psum) psum[o] = sum;
    }
  }
}

// 64 rows a block, 16 strips of the parts: lse and the row's loss; the block's (sum, count)
__global__ __launch_bounds__(1024) void join_kernel(DvXent a, const float2* __restrict__ part, const float* __restrict__ psum,
                                                    const float* __restrict__ at_label, int parts,
                                                    float* __restrict__ lse, float* __restrict__ loss,
                                                    float2* __restrict__ blocks) {
  __shared__ float sh[3][16][64];
  const int j = threadIdx.x & 63, k = threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * 64 + j;
  float m = -INFINITY, s = 0.f, sum = 0.f;
  if (n < a.N)
    for (int p = k; p < parts; p += 16) {
      const float2 q = part[(int64_t)p * a.N + n];
      const float t = fmaxf(m, q.x);
      if (t != -INFINITY) s = s * __expf(m - t) + q.y * __expf(q.x - t);
      else s += q.y;  // nothing but -inf so far (q.y is 0), or NaN
      m = t;
      if (psum) sum += psum[(int64_t)p * a.N + n];
    }
  sh[0][k][j] = m;
  sh[1][k][j] = s;
  sh[2][k][j] = sum;
  __syncthreads();
  if (k) return;
  float top = -INFINITY, tot = 0.f, all = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, sh[0][i][j]);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    tot += top == -INFINITY ? sh[1][i][j] : sh[1][i][j] * __expf(sh[0][i][j] - top);
    all += sh[2][i][j];
  }
  float l = 0.f, one = 0.f;
  if (n < a.N) {
    const float z = top + logf(tot);
    if (counted(a.labels[n], a)) {
      one = 1.f;
      l = z - (1.f - a.smooth) * at_label[n];
      if (psum) l -= a.smooth * (all / a.V);
    }
    if (lse) lse[n] = z;
    if (loss) loss[n] = l;
  }
  if (blocks) {
    l = wave_sum(l);
    one = wave_sum(one);
    if (j == 0) blocks[blockIdx.x] = {l, one};
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
// d of the piece [p0, p0 + pv) of the vocabulary: P [n][ldp], zero up to pvp columns, and
// Q = t . d [v][ldq], zero up to ldq; db partial sums [n block and wave][pv]
template <class T, int BM, int BN, int WN>
__global__ __launch_bounds__(T::NTHREADS, T::NTHREADS / 256) void grad_kernel(DvXent a, const float* __restrict__ lse, int p0,
                                                                              int pv, int pvp, u16* __restrict__ P,
                                                                              u16* __restrict__ Q, int64_t ldq,
                                                                              float* __restrict__ pbias) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int PITCH = 144;  // bytes: 64 bf16 + 16, conflict-free both ways
  constexpr int MG = T::TM < 2 ? 1 : 2, MW = 32 * MG, NW = 32 * T::TN;
  const int tm = (pv + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
  const TileAt at = tile_at(blockIdx.x, gridDim.x, tm, tn);
  const int v0 = at.m * BM, n0 = at.n * BN;  // v: within the piece
  T t;
  t.run({a.w + (int64_t)(p0 + v0) * a.ldw, a.ldw, pv - v0}, {a.x + (int64_t)n0 * a.ldx, a.ldx, a.N - n0}, a.D / 64, smem);
  add_bias(t, a, p0 + v0);
  const float off = a.smooth / a.V, hot = 1.f - a.smooth;
  float ts[T::TN];
#pragma unroll
  for (int j = 0; j < T::TN; ++j) {
    const int n = n0 + t.col(j);
    const int64_t label = n < a.N ? a.labels[n] : -1;
    const bool use = n < a.N && counted(label, a);
    const float z = use ? lse[n] : 0.f;
    ts[j] = use ? (a.reduction == DV_XENT_NONE ? a.go[n] : 1.f) : 0.f;
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int v = p0 + v0 + t.row(i, r);
        float d = __expf(t.acc[i][j][r] - z) - off;
        if (v == (int)label) d -= hot;
        t.acc[i][j][r] = use && v < p0 + pv ? d : 0.f;
      }
  }
  if (pbias) {  // over the wave's rows n: in registers, then over the 32 lanes of a column of blocks
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < T::TN; ++j) s += t.acc[i][j][r] * ts[j];
        s = row16_sum(s);
        s += __shfl_xor(s, 16, 64);
        const int v = v0 + t.row(i, r);
        if ((t.lane & 31) == 0 && v < pv) pbias[(int64_t)(at.n * WN + t.wn) * pv + v] = s;
      }
  }
  // both layouts through this wave's own part of LDS, MW columns of the vocabulary at a time
  char* mine = smem + t.wave * (NW > MW ? NW : MW) * PITCH;
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
          const uint2 d{pack2bf(c[4 * q], c[4 * q + 1]), pack2bf(c[4 * q + 2], c[4 * q + 3])};
          *reinterpret_cast<uint2*>(mine + (j * 32 + (t.lane & 31)) * PITCH + (i * 32 + 8 * q + 4 * (t.lane >> 5)) * 2) = d;
        }
    wave_sync();
#pragma unroll
    for (int e = 0; e < NW * MW / 512; ++e) {
      const int u = e * 64 + t.lane, n = u / (MW / 8), c = u % (MW / 8) * 8;
      const uint4 d = *reinterpret_cast<const uint4*>(mine + n * PITCH + c * 2);
      if (nw + n < a.N && vw + c < pvp) *reinterpret_cast<uint4*>(P + (int64_t)(nw + n) * pvp + vw + c) = d;
    }
    wave_sync();
    if (Q) {
#pragma unroll
      for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int i = 0; i < MG; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int v = i * 32 + (r & 3) + 8 * (r >> 2) + 4 * (t.lane >> 5);
            *reinterpret_cast<u16*>(mine + v * PITCH + (j * 32 + (t.lane & 31)) * 2) = f2bf(t.acc[h * MG + i][j][r] * ts[j]);
          }
      wave_sync();
#pragma unroll
      for (int e = 0; e < NW * MW / 512; ++e) {
        const int u = e * 64 + t.lane, v = u / (NW / 8), c = u % (NW / 8) * 8;
        const uint4 d = *reinterpret_cast<const uint4*>(mine + v * PITCH + c * 2);
        if (vw + v < pv && nw + c < ldq) *reinterpret_cast<uint4*>(Q + (int64_t)(vw + v) * ldq + nw + c) = d;
      }
      wave_sync();
    }
  }
}

// out[n][m] = scale * sum_k A[m][k] B[n][k] over this split's K-tiles
struct OutArgs {
  const u16 *a, *b;
  int64_t lda, ldb;
  int M, N, ktiles, splits;
  float* slab;       // [split][N][M], added to where slab_add; or null: `out` itself
  int slab_add;
  void* out;         // [N][M], bf16 or fp32
  int out_f32, out_add;
  int by_row;        // the scale is that of row n (0 where its label does not count)
};
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));

DV_DEVICE float out_scale(const DvXent& x, bool by_row, int64_t n, float common) {
  if (!by_row) return common;
  if (!counted(x.labels[n], x)) return 0.f;
  return x.reduction == DV_XENT_NONE ? x.go[n] : common;
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

template <class T, int BM, int BN>
__global__ __launch_bounds__(T::NTHREADS, T::NTHREADS / 256) void out_kernel(DvXent x, OutArgs g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int PITCH = 144, NW = 32 * T::TN;
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  // splits of one tile sit next to each other in the grid only where tiles are few; whole tiles first
  const int tiles = tm * tn, split = blockIdx.x / tiles;
  const TileAt at = tile_at(blockIdx.x - split * tiles, tiles, tm, tn);
  const int m0 = at.m * BM, n0 = at.n * BN;
  const int k0 = (int)((int64_t)g.ktiles * split / g.splits), k1 = (int)((int64_t)g.ktiles * (split + 1) / g.splits);
  T t;
  t.run({g.a + (int64_t)m0 * g.lda + k0 * 64, g.lda, g.M - m0}, {g.b + (int64_t)n0 * g.ldb + k0 * 64, g.ldb, g.N - n0},
        k1 - k0, smem);
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

// db[v] (+)= scale * sum of the partial rows
__global__ __launch_bounds__(256) void bias_kernel(DvXent x, const float* __restrict__ part, int parts, int pv,
                                                   float* __restrict__ db, int add) {
  __shared__ float sh[4][64];
  const int j = threadIdx.x & 63, k = threadIdx.x >> 6, v = blockIdx.x * 64 + j;
  float s = 0.f;
  if (v < pv)
    for (int p = k; p < parts; p += 4) s += part[(int64_t)p * pv + v];
  sh[k][j] = s;
  __syncthreads();
  if (k == 0 && v < pv) {
    s = ((sh[0][j] + sh[1][j]) + (sh[2][j] + sh[3][j])) * common_scale(x);
    db[v] = add ? db[v] + s : s;
  }
}

// dst[c][r] = src[r][c] for r < rows (labels given: only of counted rows), 0 up to ldd; 64 x 64 a block
__global__ __launch_bounds__(256) void transpose_kernel(DvXent x, const u16* __restrict__ src, int64_t lds_, int rows, int cols,
                                                        u16* __restrict__ dst, int64_t ldd, int by_label) {
  __shared__ u16 sh[64][66];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int r = e >> 6, c = e & 63;
    const bool in = r0 + r < rows && c0 + c < cols && (!by_label || counted(x.labels[r0 + r], x));
    sh[r][c] = in ? src[(int64_t)(r0 + r) * lds_ + c0 + c] : (u16)0;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int c = e >> 6, r = e & 63;
    if (c0 + c < cols && r0 + r < ldd) dst[(int64_t)(c0 + c) * ldd + r0 + r] = sh[r][c];
  }
}

// dst [rows][ldd] bf16 = src [rows][cols] (bf16 or fp32), zero behind cols
template <class S>
__global__ __launch_bounds__(256) void pack_kernel(const S* __restrict__ src, int64_t lds_, int64_t rows, int cols,
                                                   u16* __restrict__ dst, int64_t ldd) {
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < rows * (ldd / 8); u += (int64_t)gridDim.x * 256) {
    const int64_t r = u / (ldd / 8);
    const int c = (int)(u - r * (ldd / 8)) * 8;
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float f[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = c + 2 * e + k;
        if constexpr (sizeof(S) == 2) f[k] = i < cols ? bf2f(src[r * lds_ + i]) : 0.f;
        else f[k] = i < cols ? src[r * lds_ + i] : 0.f;
      }
      w[e] = pack2bf(f[0], f[1]);
    }
    *reinterpret_cast<uint4*>(dst + r * ldd + c) = uint4{w[0], w[1], w[2], w[3]};
  }
}

// ------------------------------------------------------------------------------------------- host
// Tile and split of an M x N x (64 ktiles) product: the least time by a model of one K-tile's time on
// a full CU (throughput) and alone (latency), both measured.
struct Plan { int form, splits; };
constexpr int FORM_TILE[3] = {256, 128, 64};
Plan plan(int64_t M, int64_t N, int ktiles, bool may_split) {
  constexpr double FULL[3] = {1.7, 0.58, 0.25}, ALONE[3] = {1.7, 0.8, 0.5};  // us a K-tile
  Plan best{0, 1};
  double least = 1e30;
  for (int f = 0; f < 3; ++f) {
    const int64_t tiles = (int64_t)cdiv(M, FORM_TILE[f]) * cdiv(N, FORM_TILE[f]);
    for (int s = 1; s <= (may_split ? std::min(ktiles, 32) : 1); ++s) {
      const double k = cdiv(ktiles, s), blocks = (double)tiles * s;
      const double per_cu = f == 0 ? std::ceil(blocks / 256) : std::max(1.0, blocks / 256);
      const double us = std::max(per_cu * k * FULL[f], k * ALONE[f]) + (s > 1 ? 3.0 + s * (double)M * N * 8 / 4e6 : 0.0);
      if (us < least) { least = us; best = {f, s}; }
    }
  }
  return best;
}

template <class F>
void with_tile(int form, F&& f) {
  if (form == 0) f(Big{}, std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
  else if (form == 1) f(Mid{}, std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
  else f(Small{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
}
constexpr int FORM_WM[3] = {2, 2, 2}, FORM_WN[3] = {4, 2, 2};

// more than 64 KB of LDS, allowed once for each kernel and device
template <class K>
void allow_lds(K kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  (void)hipGetDevice(&dev);
  if (done[dev & 63]) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  done[dev & 63] = true;
}

struct FwdLayout { Plan p; int parts, blocks; int64_t part, psum, label, block, bytes; };
FwdLayout fwd_layout(const DvXent& a) {
  FwdLayout l;
  l.p = plan(a.V, a.N, a.D / 64, false);
  l.parts = cdiv(a.V, FORM_TILE[l.p.form]) * FORM_WM[l.p.form];
  l.blocks = cdiv(a.N, 64);
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
  int64_t ldq;
  int bias_parts;
  bool dx_slab;
  int64_t P, Q, xt, wt, sx, sw, pb, bytes;
};
constexpr int64_t PIECE_BYTES = 1LL << 30;  // both layouts of a piece's d
BwdLayout bwd_layout(const DvXent& a, bool need_x, bool need_w, bool need_b, bool have_wt) {
  BwdLayout l;
  l.ldq = up(a.N, 64);
  const int64_t most = std::max<int64_t>(PIECE_BYTES / (4 * l.ldq) / 256 * 256, 256);
  const int pieces = cdiv(a.V, most);
  l.piece = (int)std::min<int64_t>(up(cdiv(a.V, pieces), 256), a.V);
  l.pg = plan(l.piece, a.N, a.D / 64, false);
  l.px = plan(a.width, a.N, cdiv(l.piece, 64), true);
  l.pw = plan(a.width, l.piece, cdiv(a.N, 64), true);
  l.bias_parts = cdiv(a.N, FORM_TILE[l.pg.form]) * FORM_WN[l.pg.form];
  l.dx_slab = l.px.splits > 1 || pieces > 1;
  const int64_t pvp = up(l.piece, 64);
  int64_t at = 0;
  auto take = [&](int64_t b) { const int64_t o = at; at += up(b, 256); return o; };
  l.P = take((int64_t)a.N * pvp * 2);
  l.Q = take(need_w ? (int64_t)l.piece * l.ldq * 2 : 0);
  l.xt = take(need_w ? (int64_t)a.width * l.ldq * 2 : 0);
  l.wt = take(need_x && !have_wt ? (int64_t)a.width * pvp * 2 : 0);
  l.sx = take(need_x && l.dx_slab ? (int64_t)l.px.splits * a.N * a.width * 4 : 0);
  l.sw = take(need_w && l.pw.splits > 1 ? (int64_t)l.pw.splits * l.piece * a.width * 4 : 0);
  l.pb = take(need_b ? (int64_t)l.bias_parts * l.piece * 4 : 0);
  l.bytes = at;
  return l;
}

bool sane(const DvXent& a) {
  return a.N > 0 && a.N <= DV_XENT_MAX_ROWS && a.V > 0 && a.D > 0 && a.D % 64 == 0 && a.width > 0 && a.width <= a.D &&
         a.ldx >= a.D && a.ldw >= a.D && a.ldx % 8 == 0 && a.ldw % 8 == 0 && a.ldx <= (1 << 22) && a.ldw <= (1 << 22) &&
         ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0;
}

void launch_out(const DvXent& a, OutArgs g, const Plan& p, hipStream_t st) {
  with_tile(p.form, [&](auto tile, auto b, auto, auto) {
    using T = decltype(tile);
    constexpr int B = decltype(b)::value;
    const unsigned grid = (unsigned)(cdiv(g.M, B) * cdiv(g.N, B) * g.splits);
    static bool done[64];
    allow_lds(out_kernel<T, B, B>, T::LDS, done);
    out_kernel<T, B, B><<<grid, T::NTHREADS, T::LDS, st>>>(a, g);
  });
}
void launch_reduce(const DvXent& a, const OutArgs& g, hipStream_t st) {
  const int64_t units = (int64_t)g.N * ((g.M + 3) / 4);
  reduce_kernel<<<(unsigned)std::min<int64_t>((units + 255) / 256, 4096), 256, 0, st>>>(a, g);
}
}  // namespace

int64_t dv_linear_xent_fwd_bytes(const DvXent& a) { return fwd_layout(a).bytes; }
int64_t dv_linear_xent_bwd_bytes(const DvXent& a, int need_x, int need_w, int need_b, int have_wt) {
  return bwd_layout(a, need_x, need_w, need_b, have_wt).bytes;
}

int dv_linear_xent_fwd(const DvXent& a, void* ws, float* lse, float* loss_rows, float* total, float* out, hipStream_t st) {
  if (!sane(a)) return -1;
  const FwdLayout l = fwd_layout(a);
  char* w = reinterpret_cast<char*>(ws);
  float2* part = reinterpret_cast<float2*>(w + l.part);
  float* psum = a.smooth > 0.f ? reinterpret_cast<float*>(w + l.psum) : nullptr;
  float* at_label = reinterpret_cast<float*>(w + l.label);
  float2* blocks = out ? reinterpret_cast<float2*>(w + l.block) : nullptr;
  with_tile(l.p.form, [&](auto tile, auto b, auto wm, auto) {
    using T = decltype(tile);
    constexpr int B = decltype(b)::value, WM = decltype(wm)::value;
    static bool done[64];
    allow_lds(stats_kernel<T, B, B, WM>, T::LDS, done);
    stats_kernel<T, B, B, WM><<<(unsigned)(cdiv(a.V, B) * cdiv(a.N, B)), T::NTHREADS, T::LDS, st>>>(a, part, psum, at_label);
  });
  join_kernel<<<l.blocks, 1024, 0, st>>>(a, part, psum, at_label, l.parts, lse, loss_rows, blocks);
  if (out) total_kernel<<<1, 256, 0, st>>>(blocks, l.blocks, a.reduction == DV_XENT_MEAN, out, total);
  return 0;
}

int dv_linear_xent_bwd(const DvXent& a, void* ws, const float* lse, const void* wt_all, int64_t ldwt, void* dx, void* dw,
                       int dw_f32, int dw_add, float* db, int db_add, hipStream_t st) {
  if (!sane(a)) return -1;
  const bool need_w = dw != nullptr, need_x = dx != nullptr;
  const BwdLayout l = bwd_layout(a, need_x, need_w, db != nullptr, wt_all != nullptr);
  char* w = reinterpret_cast<char*>(ws);
  u16 *P = reinterpret_cast<u16*>(w + l.P), *Q = need_w ? reinterpret_cast<u16*>(w + l.Q) : nullptr;
  u16 *xt = reinterpret_cast<u16*>(w + l.xt), *wt = reinterpret_cast<u16*>(w + l.wt);
  float* pb = db ? reinterpret_cast<float*>(w + l.pb) : nullptr;
  if (need_w) {
    const dim3 grid((unsigned)(l.ldq / 64), (unsigned)cdiv(a.width, 64));
    transpose_kernel<<<grid, 256, 0, st>>>(a, a.x, a.ldx, a.N, a.width, xt, l.ldq, 1);
  }
  OutArgs gx{};
  for (int p0 = 0; p0 < a.V; p0 += l.piece) {
    const int pv = std::min(l.piece, a.V - p0), pvp = (int)up(pv, 64);
    with_tile(l.pg.form, [&](auto tile, auto b, auto, auto wn) {
      using T = decltype(tile);
      constexpr int B = decltype(b)::value, WN = decltype(wn)::value;
      static bool done[64];
      allow_lds(grad_kernel<T, B, B, WN>, T::LDS, done);
      grad_kernel<T, B, B, WN><<<(unsigned)(cdiv(pv, B) * cdiv(a.N, B)), T::NTHREADS, T::LDS, st>>>(a, lse, p0, pv, pvp, P, Q,
                                                                                                     l.ldq, pb);
    });
    if (db) bias_kernel<<<cdiv(pv, 64), 256, 0, st>>>(a, pb, l.bias_parts, pv, db + p0, db_add);
    if (need_x) {
      const u16* wp = reinterpret_cast<const u16*>(wt_all) + p0;
      int64_t ld = ldwt;
      if (!wt_all) {
        const dim3 grid((unsigned)(pvp / 64), (unsigned)cdiv(a.width, 64));
        transpose_kernel<<<grid, 256, 0, st>>>(a, a.w + (int64_t)p0 * a.ldw, a.ldw, pv, a.width, wt, pvp, 0);
        wp = wt;
        ld = pvp;
      }
      gx = OutArgs{wp, P, ld, pvp, a.width, a.N, pvp / 64, std::min(l.px.splits, pvp / 64),
                   l.dx_slab ? reinterpret_cast<float*>(w + l.sx) : nullptr, p0 > 0, dx, 0, 0, 1};
      launch_out(a, gx, l.px, st);
    }
    if (need_w) {
      char* to = reinterpret_cast<char*>(dw) + (int64_t)p0 * a.width * (dw_f32 ? 4 : 2);
      OutArgs gw{xt, Q, l.ldq, l.ldq, a.width, pv, (int)(l.ldq / 64), l.pw.splits,
                 l.pw.splits > 1 ? reinterpret_cast<float*>(w + l.sw) : nullptr, 0, to, dw_f32, dw_add, 0};
      launch_out(a, gw, l.pw, st);
      if (l.pw.splits > 1) launch_reduce(a, gw, st);
    }
  }
  if (need_x && l.dx_slab) {
    gx.splits = l.px.splits;
    launch_reduce(a, gx, st);
  }
  return 0;
}

int dv_pack_rows(const void* src, int is_bf16, int64_t lds_, int64_t rows, int cols, void* dst, int64_t ldd, hipStream_t st) {
  if (rows <= 0 || cols <= 0 || ldd % 8 || ldd < cols) return -1;
  const unsigned grid = (unsigned)std::min<int64_t>((rows * (ldd / 8) + 255) / 256, 8192);
  if (is_bf16) pack_kernel<u16><<<grid, 256, 0, st>>>((const u16*)src, lds_, rows, cols, (u16*)dst, ldd);
  else pack_kernel<float><<<grid, 256, 0, st>>>((const float*)src, lds_, rows, cols, (u16*)dst, ldd);
  return 0;
}
