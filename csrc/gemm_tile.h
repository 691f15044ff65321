// One output tile of C[m][n] = sum_k A[m][k] * B[n][k], both operands bf16 with contiguous rows of k
// (k a multiple of 64, rows 16-byte aligned), fp32 sums in registers.
//
// A workgroup of WM x WN waves computes BM x BN; a wave TM x TN blocks of 32 x 32 with
// v_mfma_f32_32x32x16_bf16. K-tiles of 64 go from global memory to a double-buffered LDS image by
// LDS-DMA: the loads of tile t + 1 run under the products of tile t, one barrier a tile. An LDS row
// is 128 bytes; its 16-byte chunks are exclusive-or swizzled by (row >> 1) & 7, so that the 16 lanes of
// a ds_read_b128 cycle, 16 different rows, touch all 64 banks once.
//
// Rows behind the operand's last are read from its last one: the caller drops their results.
#pragma once
#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct GemmOperand {
  const u16* p;  // first row of the tile
  int64_t ld;    // elements between rows
  int rows;      // valid rows from p on, at least 1
};

template <int BM, int BN, int WM, int WN>
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

  static DV_DEVICE void dma(const u16* base, uint32_t off, uint32_t dst) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(dst)
                 : "memory");
  }
  static DV_DEVICE bf16x8 frag(const char* img, int r, int chunk) {
    return *reinterpret_cast<const bf16x8*>(img + r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4));
  }

  DV_DEVICE void run(const GemmOperand& a, const GemmOperand& b, int ktiles, char* smem) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave / WN;
    wn = wave % WN;
    const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)LDS_PTR(smem));
    uint32_t oa[IA], ob[IB];
#pragma unroll
    for (int i = 0; i < IA; ++i) {
      const int r = (wave * IA + i) * 8 + (lane >> 3);
      oa[i] = (uint32_t)(min(r, a.rows - 1) * a.ld * 2) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
#pragma unroll
    for (int i = 0; i < IB; ++i) {
      const int r = (wave * IB + i) * 8 + (lane >> 3);
      ob[i] = (uint32_t)(min(r, b.rows - 1) * b.ld * 2) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
    const u16 *pa = a.p, *pb = b.p;
    auto stage = [&](int buf) {
      const uint32_t at = lds + buf * STAGE;
#pragma unroll
      for (int i = 0; i < IA; ++i) dma(pa, oa[i], at + (wave * IA + i) * 1024);
#pragma unroll
      for (int i = 0; i < IB; ++i) dma(pb, ob[i], at + BM * 128 + (wave * IB + i) * 1024);
      pa += BK;
      pb += BK;
    };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    stage(0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int t = 0; t < ktiles; ++t) {
      const int cur = t & 1;
      if (t + 1 < ktiles) stage(cur ^ 1);
      const char* ia = smem + cur * STAGE;
      const char* ib = ia + BM * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bf16x8 fa[TM], fb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[i] = frag(ia, (wm * TM + i) * 32 + (lane & 31), k * 2 + (lane >> 5));
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j] = frag(ib, (wn * TN + j) * 32 + (lane & 31), k * 2 + (lane >> 5));
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
  }
};
