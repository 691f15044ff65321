// Layer norm over the last dimension, forward and backward.
//
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) * rstd, y = w * xh + b
//   h = dy * w,  dx = rstd * (h - mean(h) - xh * mean(h * xh)),  dw = sum_rows dy * xh,  db = sum_rows dy
//
// Bound by memory: forward reads x and writes y once, backward reads x and dy and writes dx once.
// A row stays in the registers of its LANES lanes (16 bytes a load, VECS loads a lane), so the
// variance is summed over (x - mu) itself, in fp32 and without cancellation. Each lane owns the
// same columns of every row it visits: w and b are loaded once a block, and the sums for dw / db
// stay in registers until the block's last row. Those partial sums go to a [block][2][D] slab that
// a second launch folds in a fixed order: no atomics, the same bits every time.
//
// Rows may be slices of wider ones (row stride ldx / ldg) and start at any element: 16-byte loads of
// global memory need no alignment on this hardware. D is padded to whole vectors per lane by
// masking, the last vector of a row that ends inside one is read element by element. The next row's loads
// run under this row's sums.
//
// Measured: 12544 x 2048 bf16 forward 18 us (5.7 TB/s), backward 33 us and 4 for the fold (4.2); 401408 x 256
// forward 70 us (5.9), backward 130 and 5 (4.6). Non-temporal stores of y or dx gain nothing where the
// next operator reads them.
//
// Rows wider than 16384 columns are walked in a loop of 2- or 4-byte loads, three passes forward and two
// backward, the later ones from cache, and the parameter sums in a launch of their own: 1024 x 20000 bf16 forward
// 41 us (2.0 TB/s), backward 38 + 21 and 5 for the fold. No model here has such rows; they are right, not fast.
#include "common.h"
#include "kernels.h"

namespace {
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));

template <class T>
struct Vec;  // E elements of T in 16 bytes
template <>
struct Vec<u16> {
  static constexpr int E = 8;
  static DV_DEVICE float get(u16 v) { return bf2f(v); }
  static DV_DEVICE u16 put(float v) { return f2bf(v); }
  static DV_DEVICE u32x4 load(const u16* p) { return *reinterpret_cast<const u32x4_a2*>(p); }
  static DV_DEVICE void unpack(u32x4 r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    }
  }
  static DV_DEVICE void store(u16* p, const float (&v)[8]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2bf(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<u32x4_a2*>(p) = r;
  }
};
template <>
struct Vec<float> {
  static constexpr int E = 4;
  static DV_DEVICE float get(float v) { return v; }
  static DV_DEVICE float put(float v) { return v; }
  static DV_DEVICE u32x4 load(const float* p) { return *reinterpret_cast<const u32x4_a4*>(p); }
  static DV_DEVICE void unpack(u32x4 r, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  }
  static DV_DEVICE void store(float* p, const float (&v)[4]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[i]);
    *reinterpret_cast<u32x4_a4*>(p) = r;
  }
};

// the 16 bytes at element c of a row of D, zeros behind its end. Whole vectors only (TAIL false): no
// branch, a lane behind the end reads the last one and drops it.
template <class T, bool TAIL>
DV_DEVICE u32x4 load_cols(const T* row, int c, int D) {
  constexpr int E = Vec<T>::E;
  if constexpr (!TAIL) {
    const u32x4 r = Vec<T>::load(row + min(c, D - E));
    return c < D ? r : u32x4{0, 0, 0, 0};
  }
  if (c + E <= D) return Vec<T>::load(row + c);
  u32x4 r{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (c + e < D) {
      if constexpr (sizeof(T) == 2) r[e >> 1] |= (uint32_t)row[c + e] << (16 * (e & 1));
      else r[e] = __float_as_uint(row[c + e]);
    }
  return r;
}
template <class T, bool TAIL, int E = Vec<T>::E>
DV_DEVICE void store_cols(T* row, int c, int D, const float (&v)[E]) {
  if (TAIL ? c + E <= D : c < D) {
    Vec<T>::store(row + c, v);
  } else if constexpr (TAIL) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < D) row[c + e] = Vec<T>::put(v[e]);
  }
}
template <int E>
DV_DEVICE void load_param(const float* w, int c, int D, float fill, float (&v)[E]) {
  if (w && c + E <= D) {
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const u32x4 r = *reinterpret_cast<const u32x4_a4*>(w + c + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] = __uint_as_float(r[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = w && c + e < D ? w[c + e] : fill;
  }
}

// sums of a and b over the LANES lanes of a row; LANES > 64 means the whole block
template <int LANES>
DV_DEVICE void row_sum2(float& a, float& b, float (*sh)[2]) {
  a = row16_sum(a);  // 16 lanes by DPP, the rest through LDS
  b = row16_sum(b);
#pragma unroll
  for (int o = 16; o < (LANES < 64 ? LANES : 64); o <<= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if constexpr (LANES > 64) {
    __syncthreads();  // the previous use of sh is over
    if ((threadIdx.x & 63) == 0) { sh[threadIdx.x >> 6][0] = a; sh[threadIdx.x >> 6][1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < LANES / 64; ++i) { a += sh[i][0]; b += sh[i][1]; }
  }
}

constexpr int block_of(int lanes) { return lanes > 256 ? lanes : 256; }
constexpr int bwd_block_of(int lanes) { return lanes == 64 ? 512 : block_of(lanes); }

template <class T, int LANES, int VECS, bool TAIL>
__global__ __launch_bounds__(block_of(LANES)) void ln_fwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                                 const float* __restrict__ w, const float* __restrict__ b,
                                                                 T* __restrict__ y, float* __restrict__ stats, int64_t rows,
                                                                 int D, float eps) {
  constexpr int E = Vec<T>::E, RPB = block_of(LANES) / LANES;
  __shared__ float sh[LANES > 64 ? LANES / 64 : 1][2];
  const int lane = threadIdx.x % LANES;
  float wv[VECS][E], bv[VECS][E];
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    load_param<E>(w, (lane + k * LANES) * E, D, 1.f, wv[k]);
    load_param<E>(b, (lane + k * LANES) * E, D, 0.f, bv[k]);
  }
  const float inv = 1.f / D;
  u32x4 next[VECS];
  int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / LANES;
  if (r < rows) {
#pragma unroll
    for (int k = 0; k < VECS; ++k) next[k] = load_cols<T, TAIL>(x + r * ldx, (lane + k * LANES) * E, D);
  }
  for (; r < rows; r += (int64_t)gridDim.x * RPB) {
    float v[VECS][E], s = 0.f, q = 0.f, none = 0.f;
#pragma unroll
    for (int k = 0; k < VECS; ++k) Vec<T>::unpack(next[k], v[k]);
    const int64_t r2 = r + (int64_t)gridDim.x * RPB;  // its loads run under this row's sums
    if (r2 < rows) {
#pragma unroll
      for (int k = 0; k < VECS; ++k) next[k] = load_cols<T, TAIL>(x + r2 * ldx, (lane + k * LANES) * E, D);
    }
#pragma unroll
    for (int k = 0; k < VECS; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) s += v[k][e];
    row_sum2<LANES>(s, none, sh);
    const float mu = s * inv;
#pragma unroll
    for (int k = 0; k < VECS; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[k][e] = (lane + k * LANES) * E + e < D ? v[k][e] - mu : 0.f;
        q += v[k][e] * v[k][e];
      }
    row_sum2<LANES>(q, none, sh);
    const float rstd = 1.f / sqrtf(q * inv + eps);
    if (lane == 0 && stats) { stats[2 * r] = mu; stats[2 * r + 1] = rstd; }
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = v[k][e] * rstd * wv[k][e] + bv[k][e];
      store_cols<T, TAIL>(y + r * D, (lane + k * LANES) * E, D, v[k]);
    }
  }
}

template <class T, int LANES, int VECS, bool TAIL>
__global__ __launch_bounds__(bwd_block_of(LANES)) void ln_bwd_kernel(const T* __restrict__ x, int64_t ldx,
                                                                     const T* __restrict__ dy, int64_t ldg,
                                                                     const float* __restrict__ w,
                                                                     const float* __restrict__ stats, T* __restrict__ dx,
                                                                     float* __restrict__ part, int64_t rows, int D) {
  constexpr int E = Vec<T>::E, RPB = bwd_block_of(LANES) / LANES, COLS = LANES * VECS * E;
  __shared__ float sh[LANES > 64 ? LANES / 64 : 1][2];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  float aw[VECS][E] = {}, ab[VECS][E] = {};
  // w from LDS (the widest form: from cache) for every row: in registers it would spill the sums
  constexpr bool W_LDS = COLS * 4 <= 32768;
  __shared__ __attribute__((aligned(16))) float ws[W_LDS ? COLS : 4];
  if constexpr (W_LDS) {
    for (int c = threadIdx.x; c < COLS; c += bwd_block_of(LANES)) ws[c] = w && c < D ? w[c] : 1.f;
    __syncthreads();
  }
  auto weight = [&](int k, float (&v)[E]) {
    const int c = (lane + k * LANES) * E;
    if constexpr (W_LDS) {
#pragma unroll
      for (int q = 0; q < E; q += 4) {
        const float4 f = *reinterpret_cast<const float4*>(ws + c + q);
        v[q] = f.x; v[q + 1] = f.y; v[q + 2] = f.z; v[q + 3] = f.w;
      }
    } else {
      load_param<E>(w, c, D, 1.f, v);
    }
  };
  const float inv = 1.f / D;
  u32x4 nx[VECS], ng[VECS];
  float2 nst{0.f, 0.f};
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      nx[k] = load_cols<T, TAIL>(x + r * ldx, (lane + k * LANES) * E, D);
      ng[k] = load_cols<T, TAIL>(dy + r * ldg, (lane + k * LANES) * E, D);
    }
    nst = *reinterpret_cast<const float2*>(stats + 2 * r);
  };
  int64_t r = (int64_t)blockIdx.x * RPB + group;
  if (r < rows) fetch(r);
  for (; r < rows; r += (int64_t)gridDim.x * RPB) {
    u32x4 cx[VECS], cg[VECS];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int k = 0; k < VECS; ++k) { cx[k] = nx[k]; cg[k] = ng[k]; }
    const float mu = nst.x, rstd = nst.y;
    const int64_t r2 = r + (int64_t)gridDim.x * RPB;  // its loads run under this row's sums
    if (r2 < rows) fetch(r2);
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      float v[E], g[E], wv[E];
      Vec<T>::unpack(cx[k], v);
      Vec<T>::unpack(cg[k], g);
      weight(k, wv);
#pragma unroll
      for (int e = 0; e < E; ++e) {  // behind the row's end g is 0, so every sum there adds nothing
        v[e] = (v[e] - mu) * rstd;
        aw[k][e] += g[e] * v[e];
        ab[k][e] += g[e];
        g[e] *= wv[e];
        s += g[e];
        q += g[e] * v[e];
      }
    }
    row_sum2<LANES>(s, q, sh);
    s *= inv * rstd;
    q *= inv * rstd * rstd;
    if (dx) {
#pragma unroll
      for (int k = 0; k < VECS; ++k) {
        // from the packed words again: kept unpacked since the sums they would take twice the registers
        asm volatile("" : "+v"(cx[k]), "+v"(cg[k]));
        float v[E], g[E], wv[E];
        Vec<T>::unpack(cx[k], v);
        Vec<T>::unpack(cg[k], g);
        weight(k, wv);
#pragma unroll
        for (int e = 0; e < E; ++e) g[e] = g[e] * (wv[e] * rstd) - ((v[e] - mu) * q + s);
        store_cols<T, TAIL>(dx + r * D, (lane + k * LANES) * E, D, g);
      }
    }
  }
  if (!part) return;
  part += (int64_t)blockIdx.x * 2 * D;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int k = 0; k < VECS; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (lane + k * LANES) * E + e;
        if (c < D) { part[c] = aw[k][e]; part[D + c] = ab[k][e]; }
      }
  } else {  // the block's row groups, added in order
    __shared__ float fold[2][COLS];
    for (int i = 0; i < RPB; ++i) {
      if (group == i) {
#pragma unroll
        for (int k = 0; k < VECS; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int c = (lane + k * LANES) * E + e;
            fold[0][c] = i ? fold[0][c] + aw[k][e] : aw[k][e];
            fold[1][c] = i ? fold[1][c] + ab[k][e] : ab[k][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < D; c += bwd_block_of(LANES)) {
      part[c] = fold[0][c];
      part[D + c] = fold[1][c];
    }
  }
}

// Rows of any width: one block a row, the row read three times (twice from cache).
template <class T>
__global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(const T* __restrict__ x, int64_t ldx, const float* __restrict__ w,
                                                           const float* __restrict__ b, T* __restrict__ y,
                                                           float* __restrict__ stats, int D, float eps) {
  __shared__ float sh[16][2];
  const int64_t r = blockIdx.x;
  const T* row = x + r * ldx;
  float s = 0.f, q = 0.f, none = 0.f;
  for (int c = threadIdx.x; c < D; c += 1024) s += Vec<T>::get(row[c]);
  row_sum2<1024>(s, none, sh);
  const float mu = s / D;
  for (int c = threadIdx.x; c < D; c += 1024) {
    const float d = Vec<T>::get(row[c]) - mu;
    q += d * d;
  }
  row_sum2<1024>(q, none, sh);
  const float rstd = 1.f / sqrtf(q / D + eps);
  if (threadIdx.x == 0 && stats) { stats[2 * r] = mu; stats[2 * r + 1] = rstd; }
  for (int c = threadIdx.x; c < D; c += 1024)
    y[r * D + c] = Vec<T>::put((Vec<T>::get(row[c]) - mu) * rstd * (w ? w[c] : 1.f) + (b ? b[c] : 0.f));
}

template <class T>
__global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                           int64_t ldg, const float* __restrict__ w,
                                                           const float* __restrict__ stats, T* __restrict__ dx, int D) {
  __shared__ float sh[16][2];
  const int64_t r = blockIdx.x;
  const float mu = stats[2 * r], rstd = stats[2 * r + 1];
  float s = 0.f, q = 0.f;
  for (int c = threadIdx.x; c < D; c += 1024) {
    const float h = Vec<T>::get(dy[r * ldg + c]) * (w ? w[c] : 1.f);
    s += h;
    q += h * (Vec<T>::get(x[r * ldx + c]) - mu) * rstd;
  }
  row_sum2<1024>(s, q, sh);
  s /= D;
  q /= D;
  for (int c = threadIdx.x; c < D; c += 1024) {
    const float h = Vec<T>::get(dy[r * ldg + c]) * (w ? w[c] : 1.f);
    dx[r * D + c] = Vec<T>::put((h - s - (Vec<T>::get(x[r * ldx + c]) - mu) * rstd * q) * rstd);
  }
}
// its parameter gradients: a thread a column, blockIdx.y a strip of rows
template <class T>
__global__ __launch_bounds__(256) void ln_param_wide_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                            int64_t ldg, const float* __restrict__ stats,
                                                            float* __restrict__ part, int64_t rows, int D) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= D) return;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float aw = 0.f, ab = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float g = Vec<T>::get(dy[r * ldg + c]);
    aw += g * (Vec<T>::get(x[r * ldx + c]) - stats[2 * r]) * stats[2 * r + 1];
    ab += g;
  }
  part[(int64_t)blockIdx.y * 2 * D + c] = aw;
  part[(int64_t)blockIdx.y * 2 * D + D + c] = ab;
}

// dw / db [D] (+)= sum over the slab's rows: 16 columns a block (4 lanes of 16 bytes), 64 row lanes
__global__ __launch_bounds__(256) void ln_fold_kernel(const float* __restrict__ part, int parts, int D,
                                                      float* __restrict__ dw, float* __restrict__ db, int acc_w, int acc_b) {
  __shared__ float sh[64][17];
  __shared__ float half[16][17];
  const int64_t width = 2 * (int64_t)D;
  {
    const int j = (threadIdx.x & 3) * 4, i = threadIdx.x >> 2;
    const int64_t c = (int64_t)blockIdx.x * 16 + j;
    float s[4] = {};
    if (c + 4 <= width) {
#pragma unroll 4
      for (int p = i; p < parts; p += 64) {
        const u32x4 r = *reinterpret_cast<const u32x4_a4*>(part + p * width + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += __uint_as_float(r[e]);
      }
    } else {
      for (int p = i; p < parts; p += 64)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < width) s[e] += part[p * width + c + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sh[i][j + e] = s[e];
  }
  __syncthreads();
  const int j = threadIdx.x & 15, i = threadIdx.x >> 4;
  half[i][j] = (sh[4 * i][j] + sh[4 * i + 1][j]) + (sh[4 * i + 2][j] + sh[4 * i + 3][j]);
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.x * 16 + j;
  if (i == 0 && c < width) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += half[k][j];
    float* out = c < D ? dw : db;
    const int64_t o = c < D ? c : c - D;
    if (out) out[o] = (c < D ? acc_w : acc_b) ? out[o] + t : t;
  }
}

constexpr int MAX_ELEMS = 32;  // fp32 values of a row a lane holds

// f(LANES, VECS, TAIL) of the narrowest form that holds D columns: the fewest lanes with at most
// MAX_ELEMS values each, so that narrow rows share a wave
template <class T, class F>
bool with_form(int D, F&& f) {
  constexpr int E = Vec<T>::E, V = MAX_ELEMS / E;
  const int vecs = (D + E - 1) / E;
#define LN_FORM(L, K) \
  if (vecs <= (L) * (K)) { \
    if (D % E) f(std::integral_constant<int, L>{}, std::integral_constant<int, K>{}, std::true_type{}); \
    else f(std::integral_constant<int, L>{}, std::integral_constant<int, K>{}, std::false_type{}); \
    return true; \
  }
  LN_FORM(16, 1)
  LN_FORM(32, 1)
  LN_FORM(64, 1)
  LN_FORM(64, 2)
  LN_FORM(64, 4)
  if constexpr (V > 4) { LN_FORM(64, V) }
  LN_FORM(256, 2)
  LN_FORM(256, 4)
  if constexpr (V > 4) { LN_FORM(256, V) }
  LN_FORM(512, V)
#undef LN_FORM
  return false;
}

template <class T>
void ln_fwd(const T* x, int64_t ldx, const float* w, const float* b, T* y, float* stats, int64_t rows, int D, float eps,
            hipStream_t st) {
  const bool held = with_form<T>(D, [&](auto l, auto k, auto t) {
    constexpr int L = decltype(l)::value, K = decltype(k)::value, RPB = block_of(L) / L;
    // as many blocks as run at once: each loads w and b once for all its rows
    const int64_t grid = std::min<int64_t>((rows + RPB - 1) / RPB, 256 * (K * Vec<T>::E > 16 ? 3 : K * Vec<T>::E > 8 ? 5 : 8));
    ln_fwd_kernel<T, L, K, decltype(t)::value><<<(unsigned)grid, block_of(L), 0, st>>>(x, ldx, w, b, y, stats, rows, D, eps);
  });
  if (!held) ln_fwd_wide_kernel<T><<<(unsigned)rows, 1024, 0, st>>>(x, ldx, w, b, y, stats, D, eps);
}

template <class T>
int ln_bwd(const T* x, int64_t ldx, const T* dy, int64_t ldg, const float* w, const float* stats, T* dx, float* part,
           int parts, int64_t rows, int D, hipStream_t st) {
  const bool held = with_form<T>(D, [&](auto l, auto k, auto t) {
    constexpr int L = decltype(l)::value, K = decltype(k)::value;
    ln_bwd_kernel<T, L, K, decltype(t)::value><<<(unsigned)parts, bwd_block_of(L), 0, st>>>(x, ldx, dy, ldg, w, stats, dx, part, rows, D);
  });
  if (!held) {
    if (dx) ln_bwd_wide_kernel<T><<<(unsigned)rows, 1024, 0, st>>>(x, ldx, dy, ldg, w, stats, dx, D);
    if (part) {
      const dim3 grid((unsigned)((D + 255) / 256), (unsigned)parts);
      ln_param_wide_kernel<T><<<grid, 256, 0, st>>>(x, ldx, dy, ldg, stats, part, rows, D);
    }
  }
  return 0;
}
}  // namespace

// Blocks of the backward kernel = rows of its slab. Enough waves to cover the memory's latency (the
// narrow forms hold less in flight a wave), few enough that the slab stays small beside the data.
int dv_layer_norm_parts(int is_bf16, int64_t rows, int D) {
  int per = 0, most = 0;
  auto form = [&](auto l, auto k, auto) {
    constexpr int L = decltype(l)::value;
    per = bwd_block_of(L) / L;
    most = L < 64 ? 1280 : L == 64 ? (decltype(k)::value == 1 ? 512 : 256) : L == 256 ? 512 : 256;
  };
  const bool held = is_bf16 ? with_form<u16>(D, form) : with_form<float>(D, form);
  if (!held) return (int)std::min<int64_t>(rows, 64);
  return (int)std::min<int64_t>((rows + per - 1) / per, most);
}

int dv_layer_norm_fwd(const void* x, int is_bf16, int64_t ldx, const float* w, const float* b, void* y, float* stats,
                      int64_t rows, int D, float eps, hipStream_t st) {
  if (rows <= 0 || rows > 0x7fffffff || D <= 0 || ldx < D) return -1;
  if (is_bf16) ln_fwd<u16>((const u16*)x, ldx, w, b, (u16*)y, stats, rows, D, eps, st);
  else ln_fwd<float>((const float*)x, ldx, w, b, (float*)y, stats, rows, D, eps, st);
  return 0;
}

int dv_layer_norm_bwd(const void* x, int is_bf16, int64_t ldx, const void* dy, int64_t ldg, const float* w,
                      const float* stats, void* dx, float* part, int parts, float* dw, float* db, int acc_w, int acc_b,
                      int64_t rows, int D, hipStream_t st) {
  if (rows <= 0 || rows > 0x7fffffff || D <= 0 || ldx < D || ldg < D || parts <= 0 ||
      parts != dv_layer_norm_parts(is_bf16, rows, D) || (!part && (dw || db)))
    return -1;
  if (is_bf16) ln_bwd<u16>((const u16*)x, ldx, (const u16*)dy, ldg, w, stats, (u16*)dx, part, parts, rows, D, st);
  else ln_bwd<float>((const float*)x, ldx, (const float*)dy, ldg, w, stats, (float*)dx, part, parts, rows, D, st);
  if (dw || db) {
    const unsigned grid = (unsigned)((2 * (int64_t)D + 15) / 16);
    ln_fold_kernel<<<grid, 256, 0, st>>>(part, parts, D, dw, db, acc_w, acc_b);
  }
  return 0;
}
