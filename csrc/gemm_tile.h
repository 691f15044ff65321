// One output tile of C[m][n] = sum_k A[m][k] * B[n][k], both operands bf16 with contiguous rows of k
// (k a multiple of 64, rows 16-byte aligned), fp32 sums in registers.
//
// A workgroup of WM x WN waves computes BM x BN; a wave TM x TN blocks of 32 x 32 with
// v_mfma_f32_32x32x16_bf16. K-tiles of 64 go from global memory to two LDS images by
// LDS-DMA. Fragments are read from LDS one step of 16 ahead of their products, across tiles too: the
// barrier of a tile stands before its last step, whose fragments are in registers by then, so
// the matrix cores have work while the first fragments of the next tile come. Half of a tile's loads are
// issued behind that barrier and half in the next tile's first step: issued together they held
// the products behind them up. 8192^3 with 256 x 256 tiles: 1360 TFLOP/s (the first form, every load
// at the tile's start and the barrier at its end, 1218; the library's product 1473). An LDS row
// is 128 bytes; its 16-byte chunks are exclusive-or swizzled by (row >> 1) & 7, so that the 16 lanes of
// a ds_read_b128 cycle, 16 different rows, touch all 64 banks once.
//
// Rows behind the operand's last are read from its last one: the caller drops their results.
//
// An operand may also lie the other way round, [k][row] (KA, KB): its image is then [k][row] too, and
// ds_read_b64_tr_b16 gives each lane four k of its row. 16 lanes read 4 rows of k by 32 bytes; the 64-byte
// units of an LDS row are exclusive-or swizzled by k, so that the lanes of a half wave touch all 64 banks
// once. 8192^3: 1345 TFLOP/s with KA, 1370 with KB.
#pragma once
#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct GemmOperand {
  const u16* p;  // first row of the tile
  int64_t ld;    // elements between rows
  int rows;      // valid rows from p on, at least 1
  int deep = 0;  // where it lies [k][row]: valid k from p on, at least 1; those behind are read from the last one
};

template <int BM, int BN, int WM, int WN, bool KA = false, bool KB = false>
struct GemmTile {
  static constexpr int NW = WM * WN, NTHREADS = 64 * NW;
  static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int BK = 64, STAGE = (BM + BN) * BK * 2, LDS = 2 * STAGE;
  static constexpr int IA = BM / 8 / NW, IB = BN / 8 / NW;  // 1-KB pieces (8 rows) a wave loads
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM % (32 * WM) == 0 && BN % (32 * WN) == 0, "tile");

  f32x16 acc[TM][TN];
  int lane, wave, wm, wn;

  // row m / column n, within the tile, of acc[i][j][r]
  DV_DEVICE int row(int i, int r) const { return (wm * TM + i) * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }
  DV_DEVICE int col(int j) const { return (wn * TN + j) * 32 + (lane & 31); }
  DV_DEVICE bool active() const { return true; }  // whether this wave holds a part of the tile

  static DV_DEVICE void dma(const u16* base, uint32_t off, uint32_t dst) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(dst)
                 : "memory");
  }
  // this wave's LDS-DMA has landed and its LDS reads are done; then every wave's
  static DV_DEVICE void landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x7 << 4);  // vmcnt(0) lgkmcnt(0); the builtin, which hipcc counts with
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  // what the 64-byte units of row k are swizzled by: rows of 256 bytes or more, of 128 bytes
  template <int B>
  static DV_DEVICE int unit_swizzle(int k) { return B >= 128 ? k & 3 : (k >> 1) & 1; }
  // byte offsets, from a K-tile's start, of the 16 bytes this lane loads for each of its pieces
  template <bool K, int B, int I>
  DV_DEVICE void offsets(const GemmOperand& o, int deep, uint32_t (&off)[I]) const {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if constexpr (K) {
        const int at = (wave * I + i) * 64 + lane, k = at / (B / 8), c = at % (B / 8);
        const int row = (c ^ (unit_swizzle<B>(k) << 2)) * 8;
        off[i] = (uint32_t)(min(k, deep - 1) * o.ld * 2) + (uint32_t)min(row, (o.rows - 1) & ~7) * 2;
      } else {
        const int r = (wave * I + i) * 8 + (lane >> 3);
        off[i] = (uint32_t)(min(r, o.rows - 1) * o.ld * 2) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
      }
    }
  }
  // byte offsets, in an operand's image, of this lane's fragments of step 0: one for each block of 32 rows where
  // it lies [k][row], else the row's (its chunk depends on the step)
  template <bool K, int B, int T, int I>
  DV_DEVICE void places(int w, int (&at)[I]) const {
    const int k = (lane & 15) >> 2;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if constexpr (K)
        at[i] = ((lane >> 5) * 8 + k) * B * 2 + (((w * T + i) ^ unit_swizzle<B>(k)) << 6) + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
      else at[i] = (w * T * 32 + (lane & 31)) * 128;
    }
  }
  // eight k of this lane's row
  template <int B>
  static DV_DEVICE bf16x8 turned(char* at) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    using Lds = __attribute__((address_space(3))) s16x4*;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(at + 4 * B * 2));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  DV_DEVICE void run(const GemmOperand& a, const GemmOperand& b, int ktiles, char* smem) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave / WN;
    wn = wave % WN;
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(smem));
    uint32_t oa[IA], ob[IB];
    offsets<KA, BM>(a, a.deep, oa);
    offsets<KB, BN>(b, b.deep, ob);
    const u16 *pa = a.p, *pb = b.p;
    int da = a.deep, db = b.deep;
    auto stage_a = [&](int slot) {
      if constexpr (KA)
        if (da < BK) offsets<KA, BM>(a, da, oa);
#pragma unroll
      for (int i = 0; i < IA; ++i) dma(pa, oa[i], lds + slot * STAGE + (wave * IA + i) * 1024);
      pa += KA ? BK * a.ld : BK;
      da -= BK;
    };
    auto stage_b = [&](int slot) {
      if constexpr (KB)
        if (db < BK) offsets<KB, BN>(b, db, ob);
#pragma unroll
      for (int i = 0; i < IB; ++i) dma(pb, ob[i], lds + slot * STAGE + BM * 128 + (wave * IB + i) * 1024);
      pb += KB ? BK * b.ld : BK;
      db -= BK;
    };
    int ra[KA ? TM : 1], rb[KB ? TN : 1];
    places<KA, BM, TM>(wm, ra);
    places<KB, BN, TN>(wn, rb);
    const int swz = ((lane & 31) >> 1) & 7, half = lane >> 5;
    bf16x8 fa[2][TM], fb[2][TN];
    auto read = [&](int f, int slot, int k) {
      char *ia = smem + slot * STAGE, *ib = ia + BM * 128;
      const int chunk = ((k * 2 + half) ^ swz) << 4;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        if constexpr (KB) fb[f][j] = turned<BN>(ib + rb[j] + k * 16 * BN * 2);
        else fb[f][j] = *reinterpret_cast<const bf16x8*>(ib + rb[0] + chunk + j * 32 * 128);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (KA) fa[f][i] = turned<BM>(ia + ra[i] + k * 16 * BM * 2);
        else fa[f][i] = *reinterpret_cast<const bf16x8*>(ia + ra[0] + chunk + i * 32 * 128);
      }
    };
    auto multiply = [&](int f) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[f][i], fb[f][j], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    stage_a(0);
    stage_b(0);
    if (ktiles > 1) stage_a(1);
    landed();
    read(0, 0, 0);
    // the scheduling barriers keep a step's reads before its products: hipcc sinks them to save registers
    auto tile = [&](int t, int cur, int nxt) {
      read(1, cur, 1);
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < ktiles) stage_b(nxt);  // of tile t + 1
      multiply(0);
      __builtin_amdgcn_sched_barrier(0);
      read(0, cur, 2);
      __builtin_amdgcn_sched_barrier(0);
      multiply(1);
      __builtin_amdgcn_sched_barrier(0);
      read(1, cur, 3);
      __builtin_amdgcn_sched_barrier(0);
      multiply(0);
      __builtin_amdgcn_sched_barrier(0);
      landed();  // tile t's fragments are in registers, its slot is free; tile t + 1 is in LDS
      if (t + 1 < ktiles) read(0, nxt, 0);
      __builtin_amdgcn_sched_barrier(0);
      if (t + 2 < ktiles) stage_a(cur);
      multiply(1);
      __builtin_amdgcn_sched_barrier(0);
    };
    int t = 0;
    for (; t + 1 < ktiles; t += 2) {
      tile(t, 0, 1);
      tile(t + 1, 1, 0);
    }
    if (t < ktiles) tile(t, 0, 1);
    landed();  // LDS is free for the caller
  }
};

// A 32 x 32 tile for products with few rows and columns, where latency counts: 8 waves split the sum by
// K-tiles instead of the tile. A wave has every load of up to 4 K-tiles in flight at once (8 lanes a row
// of 128 bytes; fragments straight from memory, a row a lane, touched four times the cache lines and took
// half as long again), turns them into fragments through its own part of LDS without a barrier, and
// the waves meet once at the end. The first wave holds the result. Logits and their statistics of 8 rows by
// 1000 columns, sum of 2048: 7.6 us, of 256 rows 9.8 us; in 64 x 64 tiles, a chain of 32 K-tiles, 11.7 and 18.6.
struct ThinTile {
  static constexpr int NW = 8, NTHREADS = 512, TM = 1, TN = 1, BK = 64, IMAGE = 64 * 128, LDS = NW * IMAGE;

  f32x16 acc[1][1];
  int lane, wave, wm, wn;

  DV_DEVICE int row(int, int r) const { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }
  DV_DEVICE int col(int) const { return lane & 31; }
  DV_DEVICE bool active() const { return wave == 0; }

  DV_DEVICE void run(const GemmOperand& a, const GemmOperand& b, int ktiles, char* smem) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    constexpr int CHUNK = 4;
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wn = 0;
    const int per = (ktiles + NW - 1) / NW, t0 = min(wave * per, ktiles), t1 = min(t0 + per, ktiles);
    const u16 *pa[4], *pb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 3), c = (lane & 7) * 8;
      pa[i] = a.p + (int64_t)min(r, a.rows - 1) * a.ld + c;
      pb[i] = b.p + (int64_t)min(r, b.rows - 1) * b.ld + c;
    }
    char* mine = smem + wave * IMAGE;
    const int w0 = (lane >> 3) * 128;  // rows 8 apart: (row >> 1) & 7 is that of lane >> 3 and of i
    f32x16 c0, c1;
#pragma unroll
    for (int r = 0; r < 16; ++r) c0[r] = c1[r] = 0.f;
    for (int t = t0; t < t1; t += CHUNK) {
      u32x4 ra[CHUNK][4], rb[CHUNK][4];
#pragma unroll
      for (int k = 0; k < CHUNK; ++k)
        if (t + k < t1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ra[k][i] = *reinterpret_cast<const u32x4*>(pa[i] + (t + k) * BK);
            rb[k][i] = *reinterpret_cast<const u32x4*>(pb[i] + (t + k) * BK);
          }
        }
#pragma unroll
      for (int k = 0; k < CHUNK; ++k)
        if (t + k < t1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int swz = ((i * 8 + (lane >> 3)) >> 1) & 7, at = w0 + i * 1024 + (((lane & 7) ^ swz) << 4);
            *reinterpret_cast<u32x4*>(mine + at) = ra[k][i];
            *reinterpret_cast<u32x4*>(mine + 4096 + at) = rb[k][i];
          }
          asm volatile("" ::: "memory");
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = lane & 31, at = r * 128 + (((q * 2 + (lane >> 5)) ^ ((r >> 1) & 7)) << 4);
            const bf16x8 fa = *reinterpret_cast<const bf16x8*>(mine + at), fb = *reinterpret_cast<const bf16x8*>(mine + 4096 + at);
            if (q & 1) c1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb, c1, 0, 0, 0);
            else c0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa, fb, c0, 0, 0, 0);
          }
          asm volatile("" ::: "memory");  // the LDS works in order: the next tile's writes come behind these reads
        }
    }
    __syncthreads();
    f32x4* meet = reinterpret_cast<f32x4*>(smem);  // [wave][quad][lane]
#pragma unroll
    for (int q = 0; q < 4; ++q)
      meet[(wave * 4 + q) * 64 + lane] = f32x4{c0[4 * q] + c1[4 * q], c0[4 * q + 1] + c1[4 * q + 1], c0[4 * q + 2] + c1[4 * q + 2],
                                               c0[4 * q + 3] + c1[4 * q + 3]};
    __syncthreads();
    if (active()) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) t += meet[(w * 4 + q) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][0][4 * q + e] = t[e];
      }
    }
    __syncthreads();  // LDS is free for the caller
  }
};
