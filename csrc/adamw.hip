// AdamW over every tensor of a flat fp32 buffer in one launch, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 bytes a value with 32-bit moments (p, m, v read and written, g read), 16 with
// 8-bit ones. Measured, moments, gradients and parameters out of cache: 25.6M values 123 us with 32-bit
// moments (5.8 TB/s of those bytes), 84 us with 8-bit ones (4.9); 138M values in 8 bits 430 us (5.1; the
// non-temporal policy made that 445).
//
// 8-bit moments: m and r = sqrt(v) are held as e4m3 codes (the type torch calls float8_e4m3fn)
// times one fp32 scale for each BLOCK = 256 values; a block never crosses a tensor, so a tensor's
// state does not depend on its neighbours. r and not v: the square root halves the range of
// exponents a block has to span. The update uses the new m and v before they are rounded.
//  * Rounding is stochastic. v moves by a thousandth of itself a step while neighbouring codes are
//    an eighth apart: rounded to nearest it would never move. A code is rounded up with the
//    probability of the part cut off (20 bits of it), so the mean of m and of the root is kept. The
//    random bits are a hash of (seed, step, place), the same on every run. v, the square of a rounded root, gains
//    the rounding's variance: a step moves a root by some (1 - b2) / 2 of itself, which goes to the next code, a
//    sixteenth to an eighth away, with that part of the way as probability. For normal gradients v settles 1 % above
//    its mean for b2 = .9, 4 % for .99 and 5 to 6 % for .999; the roots, which updates are divided by, 1.4 %.
//  * A root above zero keeps at least the smallest code: it is divided by, and losing it while m
//    keeps a code of its own would give a step of any size.
//  * One multiplication by 2^-120 puts e4m3's exponent field and fraction where the float's are
//    (its values under the least normal one become the float's denormals), so the code is the
//    rounded bit pattern shifted down by 20, and decoding is the reverse.
//  * A value that is not finite becomes the NaN code and is read back as NaN: its parameter is NaN from the next
//    step on at the latest, as with 32-bit moments it stays NaN or stuck. The scale is that of the block's finite
//    values, which keep theirs.
#include "common.h"
#include "kernels.h"

namespace {
constexpr int NT = 256;
constexpr int BLOCK = DV_ADAMW_BLOCK;  // values a scale
constexpr int PER_WAVE = DV_ADAMW_CHUNK / BLOCK / (NT / 64);

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

struct Coef {
  float decay, b1, omb1, b2, omb2, size, root_bc2, eps, gscale;
};
// the scalars of this step; hp / skip as in the other optimizers (device-side values of a captured step)
DV_DEVICE Coef coefs(const DvAdamW& a) {
  float lr = a.lr, bc1 = a.bc1, bc2 = a.bc2;
  if (a.hp) { lr = a.hp[0]; bc1 = a.hp[1]; bc2 = a.hp[2]; }
  if (a.hp && a.skip) {
    const float t = a.skip[4] + 1.f;
    bc1 = 1.f - powf(a.b1, t);
    bc2 = 1.f - powf(a.b2, t);
  }
  return {1.f - lr * a.wd, a.b1, a.omb1, a.b2, a.omb2, lr / bc1, 1.f / sqrtf(bc2), a.eps, a.gscale};
}

// products and sums rounded one by one: the host's form of the same step gives the same codes
DV_DEVICE void moments(const Coef& c, float g, float& m, float& v) {
#pragma clang fp contract(off)
  m = m * c.b1 + g * c.omb1;
  v = v * c.b2 + (g * g) * c.omb2;
}
DV_DEVICE float update(const Coef& c, float p, float m, float root) {
  return p * c.decay - c.size * (m / (root * c.root_bc2 + c.eps));
}

// STREAM: every access with the non-temporal policy, for buffers that cannot stay in the 256 MB memory-side
// cache from one step to the next. p, g, m, v of 25.6M values (409 MB): 138.5 -> 123.4 us; 138M values
// 708 -> 642 us (6.0 TB/s); but 16M values (256 MB), updated again at once, 64 -> 73 us.
template <bool STREAM>
DV_DEVICE f32x4 load4(const float* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const f32x4_a4*>(p));
  return *reinterpret_cast<const f32x4_a4*>(p);
}
template <bool STREAM>
DV_DEVICE void store4(float* p, f32x4 v) {
  if constexpr (STREAM) __builtin_nontemporal_store((f32x4_a4)v, reinterpret_cast<f32x4_a4*>(p));
  else *reinterpret_cast<f32x4_a4*>(p) = v;
}
constexpr int64_t STREAM_VALUES = 20 << 20;

template <bool STREAM>
__global__ __launch_bounds__(NT) void adamw32_kernel(DvAdamW a, float* __restrict__ p, const float* __restrict__ g,
                                                     float* __restrict__ m, float* __restrict__ v, int64_t n) {
  if (a.skip && *a.skip != 0.f) return;
  const Coef c = coefs(a);
  const int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 4;
  if (i + 4 <= n) {
    f32x4 pv = load4<STREAM>(p + i), gv = load4<STREAM>(g + i);
    f32x4 mv = load4<STREAM>(m + i), vv = load4<STREAM>(v + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float me = mv[e], ve = vv[e];
      moments(c, gv[e] * c.gscale, me, ve);
      mv[e] = me;
      vv[e] = ve;
      pv[e] = update(c, pv[e], me, sqrtf(ve));
    }
    store4<STREAM>(m + i, mv);
    store4<STREAM>(v + i, vv);
    store4<STREAM>(p + i, pv);
  } else {
    for (int64_t j = i; j < n; ++j) {
      float me = m[j], ve = v[j];
      moments(c, g[j] * c.gscale, me, ve);
      m[j] = me;
      v[j] = ve;
      p[j] = update(c, p[j], me, sqrtf(ve));
    }
  }
}

// 32-bit mixing by multiplications and shifted exclusive ors: every bit of the result depends on
// every bit of h (half of them flip with any input bit, within 0.5 %)
DV_DEVICE uint32_t mix(uint32_t h) {
  h ^= h >> 16;
  h *= 0x6C8E9CF5u;
  h ^= h >> 15;
  h *= 0x5D2A4B35u;
  return h ^ (h >> 16);
}
// whether one of the four codes is NaN
DV_DEVICE bool any_nan(uint32_t codes) { return ((codes & 0x7f7f7f7f) + 0x01010101) & 0x80808080; }
// of any code but NaN
DV_DEVICE float from8(uint32_t code, float scale) {
  return __uint_as_float((code & 0x7f) << 20 | (code & 0x80) << 24) * 0x1p+120f * scale;
}
// code of |t|, `bits` < 2^20
DV_DEVICE uint32_t to8(float t, float up, uint32_t bits) {
  const float s = fabsf(t) * up;
  if (!(s < 1e30f)) return 0x7f;
  const uint32_t code = (__float_as_uint(s * 0x1p-120f) + bits) >> 20;
  return code < 126 ? code : 126;
}

// the wave's largest |t|, infinities apart; `top`: this lane's
DV_DEVICE float finite_max(float top, const float (&t)[4]) {
  top = wave_max(top);
  if (top < INFINITY) return top;
  top = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = fabsf(t[e]) < INFINITY ? fmaxf(top, fabsf(t[e])) : top;
  return wave_max(top);
}

__global__ __launch_bounds__(NT) void adamw8_kernel(DvAdamW a, const DvAdamWChunk* __restrict__ chunks, float* __restrict__ p,
                                                    const float* __restrict__ g, uint8_t* __restrict__ m8,
                                                    float* __restrict__ ms, uint8_t* __restrict__ r8,
                                                    float* __restrict__ rs) {
  if (a.skip && *a.skip != 0.f) return;
  const Coef c = coefs(a);
  const uint32_t step = a.hp ? (uint32_t)a.hp[3] : a.step;
  const uint32_t key = mix(a.seed + step * 0x9E3779B1u);
  const DvAdamWChunk ch = chunks[blockIdx.x];
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int q = 0; q < PER_WAVE; ++q) {
    const int at = ((threadIdx.x >> 6) * PER_WAVE + q) * BLOCK;  // the block's first value within the chunk
    if (at >= ch.n) return;
    const int64_t blk = ch.block + at / BLOCK, i = ch.first + at + lane * 4, k = blk * BLOCK + lane * 4;
    const int left = ch.n - at - lane * 4;  // values of this lane
    float pv[4] = {}, gv[4] = {}, mv[4], rv[4];
    if (left >= 4) {
      const f32x4 pq = *reinterpret_cast<const f32x4_a4*>(p + i), gq = *reinterpret_cast<const f32x4_a4*>(g + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) { pv[e] = pq[e]; gv[e] = gq[e]; }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) { pv[e] = p[i + e]; gv[e] = g[i + e]; }
    }
    const uint32_t mq = *reinterpret_cast<const uint32_t*>(m8 + k), rq = *reinterpret_cast<const uint32_t*>(r8 + k);
    const float msc = ms[blk], rsc = rs[blk];
    float mtop = 0.f, rtop = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mv[e] = from8(mq >> (8 * e), msc);
      rv[e] = from8(rq >> (8 * e), rsc);
    }
    if (__any(any_nan(mq) || any_nan(rq))) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((mq >> (8 * e) & 0x7f) == 0x7f) mv[e] = NAN;
        if ((rq >> (8 * e) & 0x7f) == 0x7f) rv[e] = NAN;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma clang fp contract(off)
      float v = rv[e] * rv[e];
      moments(c, gv[e] * c.gscale, mv[e], v);
      rv[e] = sqrtf(v);
      if (e >= left) mv[e] = rv[e] = 0.f;  // behind the tensor's end the state stays zero
      mtop = fmaxf(mtop, fabsf(mv[e]));
      rtop = fmaxf(rtop, rv[e]);
      pv[e] = update(c, pv[e], mv[e], rv[e]);
    }
    mtop = finite_max(mtop, mv);  // (fmaxf has left NaN out)
    rtop = finite_max(rtop, rv);
    const float mup = mtop >= 0x1p-100f ? 448.f / mtop : 0.f, rup = rtop >= 0x1p-100f ? 448.f / rtop : 0.f;
    uint32_t mc = 0, rc = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t place = (uint64_t)k + e;
      const uint32_t h = mix((uint32_t)place * 0x2545F491u + (uint32_t)(place >> 32) * 0x7A6B3C5Du + key);
      mc |= (to8(mv[e], mup, h & 0xFFFFF) | (mv[e] < 0.f ? 0x80u : 0u)) << (8 * e);
      const uint32_t r = to8(rv[e], rup, h >> 12);
      rc |= (r == 0 && rv[e] > 0.f ? 1u : r) << (8 * e);
    }
    if (left >= 4) {
      *reinterpret_cast<f32x4_a4*>(p + i) = f32x4{pv[0], pv[1], pv[2], pv[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) p[i + e] = pv[e];
    }
    *reinterpret_cast<uint32_t*>(m8 + k) = mc;
    *reinterpret_cast<uint32_t*>(r8 + k) = rc;
    if (lane == 0) { ms[blk] = mtop * (1.f / 448.f); rs[blk] = rtop * (1.f / 448.f); }
  }
}
}  // namespace

int dv_adamw32(const DvAdamW& a, float* p, const float* g, float* m, float* v, int64_t n, hipStream_t st) {
  const int64_t grid = (n + NT * 4 - 1) / (NT * 4);
  if (n <= 0 || grid > 0x7fffffff) return -1;
  if (n >= STREAM_VALUES) adamw32_kernel<true><<<(unsigned)grid, NT, 0, st>>>(a, p, g, m, v, n);
  else adamw32_kernel<false><<<(unsigned)grid, NT, 0, st>>>(a, p, g, m, v, n);
  return 0;
}

int dv_adamw8(const DvAdamW& a, const void* chunks, int nchunks, float* p, const float* g, uint8_t* m8, float* ms,
              uint8_t* r8, float* rs, hipStream_t st) {
  if (nchunks <= 0) return -1;
  adamw8_kernel<<<nchunks, NT, 0, st>>>(a, reinterpret_cast<const DvAdamWChunk*>(chunks), p, g, m8, ms, r8, rs);
  return 0;
}
