// Product of 8-bit integers for gfx950 with a scale for each row of A (token) and each column of B (channel):
//   C[M,N] = cast( (sum_k A[m,k] B[k,n]) * scale_a[m] * scale_b[n] + bias[n] )
// The sum is exact (32-bit integers, K <= 131071: 128 * 128 * K stays below 2^31); scales and bias are applied in fp32.
//
// The kernels read K-contiguous rows of A and of B^T in pieces of 16 bytes.  Operands that are not like that (another
// stride order, K % 16 != 0, unaligned rows) are copied into the workspace with rows padded to a multiple of 128.  A K that
// is a multiple of 16 but not of 128 needs no copy: rows are read on behind K (clamped to the end of the matrix) and A's
// part of that is set to zero where it has landed; what stands in the other factor of a zero does not matter for integers.
// (777 x 4100 x 4112 with a copy of A 29.2 us, without 27.1.)
#include "hx_common.h"

#include <type_traits>

#define I8_BK 128  // bytes of k per tile row

struct I8Args {
  const uint8_t *a, *b;  // rows of A and of B^T, K contiguous
  void* c;
  const float *sa, *sb;
  const void* bias;
  int M, N, nk;  // nk: k-tiles of 128
  int tail;      // bytes of the last k-tile in front of K
  long lda, ldb, ldc;
  int bias_dt;
  int tiles_m, bn, kt_per_split;
  uint32_t a_max, b_max;  // last byte offsets of A and B^T a 16-byte read may start at
};

__device__ __forceinline__ float i8_bias(const void* bias, int dt, long n) {
  return dt == HX_F32 ? ((const float*)bias)[n] : dt == HX_BF16 ? (float)((const __bf16*)bias)[n] : (float)((const _Float16*)bias)[n];
}

// ------------------------------------------------------------------------------------------
// tile: BM x 128 outputs per workgroup, 4 waves (2 x 2) of BM/2 x 64.  Ring of NS k-tiles in the LDS, filled by DMA
// (eight rows x 128 bytes per instruction, 16-byte chunk c of row r at position c ^ ((r >> 1) & 7)); a 16x16x64 MFMA takes
// 16 bytes per lane, so a k-tile is two of them per pair of blocks: lane group g multiplies chunks 2kq and 2kq+1 with
// kq = 0, 3, 1, 2 (the order in which the 16-byte reads of a wave meet no bank twice).
// split-K (kt_per_split): workgroup row blockIdx.y adds up its k-tiles into its own slab of 32-bit integers.
// KT: K is not a multiple of 128 and A or B is read on behind it.
// For batches between a decode step and a prompt: 777 x 4096 x 4096 (one round of 224 tiles of 128) 20.6 us, 512 x 4096 x
// 4096 (256 of 64) 15.5.  A k-tile takes 0.47 and 0.33 us, of which its MFMAs are 0.21 and 0.11: with one workgroup per
// compute unit the rest is the barrier, the LDS and the landing of the next k-tile.
// ------------------------------------------------------------------------------------------
template <int OUT, int BM, bool KT, bool SPLIT>
__global__ __launch_bounds__(256) void hx_int8_gemm_tile(I8Args p) {
  constexpr int NS = BM == 64 ? 6 : 4;
  constexpr int STAGE = (BM + 128) * 128;
  constexpr int WMB = BM / 32;
  constexpr int AJ = BM / 32, IPW = AJ + 4;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NS][STAGE];

  const int kt0 = SPLIT ? p.kt_per_split * (int)blockIdx.y : 0;
  const int nk = SPLIT ? min(p.kt_per_split, p.nk - kt0) : p.nk;
  // 256 consecutive tiles of a raster of eight tile rows at a time, in eight contiguous pieces, one per XCD (workgroup i
  // runs on XCD i % 8), so that the tiles resident on one share panels of A and B in its L2
  int tm, tn;
  {
    const int nwg = gridDim.x, wg = blockIdx.x, run = wg & ~255, n = min(nwg - run, 256), l = wg & 255, tiles_n = nwg / p.tiles_m;
    const int per = n >> 3, rem = n & 7, xcd = l & 7;
    const int tile = run + xcd * per + min(xcd, rem) + (l >> 3);
    const int group = 8 * tiles_n, first = (tile / group) * 8, gm = min(p.tiles_m - first, 8);
    tm = first + (tile % group) % gm;
    tn = (tile % group) / gm;
  }
  const long m0 = (long)tm * BM, n0 = (long)tn * p.bn;
  const int nlast = (int)min(n0 + p.bn, (long)p.N) - 1;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w >> 1, wn = w & 1;

  // ---- DMA: instruction j of an operand covers rows 8j .. 8j+7; wave w issues j = w, w+4, ...
  const int lrow = lane >> 3, lpos = lane & 7;
  const uint32_t chunk = (uint32_t)((lpos ^ ((4 * (w & 1) + (lrow >> 1)) & 7)) * 16);
  uint32_t a_vo[AJ], b_vo[4];
#pragma unroll
  for (int jj = 0; jj < AJ; ++jj) a_vo[jj] = (uint32_t)min((int)m0 + 8 * (w + 4 * jj) + lrow, p.M - 1) * (uint32_t)p.lda + chunk;
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) b_vo[jj] = (uint32_t)min((int)n0 + 8 * (w + 4 * jj) + lrow, nlast) * (uint32_t)p.ldb + chunk;
  const uint32_t lds0 = hx_lds_addr(&smem[0][0]);
  // past the last k-tile: that one again, so that every step issues IPW instructions and the counted waits stay exact
  auto issue_one = [&](int kt, int i) {
    const long t = (long)(kt0 + min(kt, nk - 1)) * I8_BK;
    const uint32_t base = lds0 + (uint32_t)(kt % NS) * STAGE;
    if (i < AJ && KT) hx_g2l16_s(hx_uniform_ptr(p.a), min(a_vo[i] + (uint32_t)t, p.a_max), base + (w + 4 * i) * 1024);
    else if (i < AJ) hx_g2l16_s(hx_uniform_ptr(p.a + t), a_vo[i], base + (w + 4 * i) * 1024);
    else if (KT) hx_g2l16_s(hx_uniform_ptr(p.b), min(b_vo[i - AJ] + (uint32_t)t, p.b_max), base + BM * 128 + (w + 4 * (i - AJ)) * 1024);
    else hx_g2l16_s(hx_uniform_ptr(p.b + t), b_vo[i - AJ], base + BM * 128 + (w + 4 * (i - AJ)) * 1024);
  };

  // what this wave has fetched of A behind K becomes zero, between its landing and the barrier that hands the tile over
  auto zero_tail = [&](int kt) {
    if (!KT || kt0 + kt != p.nk - 1 || (int)chunk < p.tail) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int jj = 0; jj < AJ; ++jj) *(v4i*)&smem[kt % NS][(w + 4 * jj) * 1024 + lane * 16] = (v4i){0, 0, 0, 0};
  };

  const int r16 = lane & 15, gq = lane >> 4;
  const int kq = (gq >> 1) ^ ((gq & 1) * 3);
  const int x16 = ((2 * kq) ^ ((r16 >> 1) & 7)) * 16;
  const int a_base = (wm * (BM / 2) + r16) * 128, b_base = BM * 128 + (wn * 64 + r16) * 128;
  v4i fa[WMB][2], fb[4][2];
  auto load_a = [&](int f, int kt) {
    const uint8_t* st = &smem[kt % NS][0] + a_base + f * 2048;
    fa[f][0] = *(const v4i*)(st + x16), fa[f][1] = *(const v4i*)(st + (x16 ^ 16));
  };
  auto load_b = [&](int f, int kt) {
    const uint8_t* st = &smem[kt % NS][0] + b_base + f * 2048;
    fb[f][0] = *(const v4i*)(st + x16), fb[f][1] = *(const v4i*)(st + (x16 ^ 16));
  };
  // acc[bj][bi][r] is C[m0 + wm*BM/2 + 16 bi + lane%16][n0 + wn*64 + 16 bj + 4*(lane/16) + r]
  v4i acc[4][WMB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < WMB; ++j) {
      acc[i][j] = (v4i){0, 0, 0, 0};
      hx_acc_pin(acc[i][j]);
    }

  constexpr int EVERY = 8 * WMB >= 4 * IPW ? 4 : 2;
  // One k-tile: its MFMAs row block by row block; a fragment takes the next tile's rows as soon as its last MFMA is out,
  // one DMA instruction follows every EVERY MFMAs.
  auto step = [&](int kt) {
    __builtin_amdgcn_s_waitcnt(hx_vmcnt_imm((NS - 2) * IPW));  // this wave's part of tile kt+1 has landed
    zero_tail(kt + 1);
    __syncthreads();  // ... everybody's has, and every wave has read tile kt out of its stage
#pragma unroll
    for (int i = 0; i < 8 * WMB; ++i) {  // row block, half of the k-tile, column block: an accumulator rests for three others
      const int bj = i & 3, hi = (i >> 2) & 1, bi = i >> 3;
      hx_mfma_16x16x64_i8_acc(acc[bj][bi], fb[bj][hi], fa[bi][hi]);
      if (i % EVERY == EVERY - 1 && i / EVERY < IPW) issue_one(kt + NS, i / EVERY);
      if (hi && bj == 3) load_a(bi, kt + 1);
      if (hi && bi == WMB - 1) load_b(bj, kt + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  static_assert(8 * WMB >= EVERY * IPW, "every DMA instruction of a k-tile has an MFMA to follow");
  for (int t = 0; t < NS; ++t)
#pragma unroll
    for (int i = 0; i < IPW; ++i) issue_one(t, i);
  __builtin_amdgcn_s_waitcnt(hx_vmcnt_imm((NS - 1) * IPW));
  zero_tail(0);
  __syncthreads();
#pragma unroll
  for (int f = 0; f < WMB; ++f) load_a(f, 0);
#pragma unroll
  for (int f = 0; f < 4; ++f) load_b(f, 0);
  hx_mfma_settle();
  for (int kt = 0; kt < nk; ++kt) step(kt);
  HX_WAIT_VM0();  // no DMA may still be writing this workgroup's LDS when it ends
  hx_mfma_settle();
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < WMB; ++j) hx_acc_pin(acc[i][j]);  // no copy of an accumulator before the wait

  if (SPLIT) {
    int* C = (int*)p.c + (long)blockIdx.y * p.M * p.N;
#pragma unroll
    for (int bi = 0; bi < WMB; ++bi) {
      const long m = m0 + wm * (BM / 2) + 16 * bi + r16;
      if (m >= p.M) continue;
#pragma unroll
      for (int bj = 0; bj < 4; ++bj) {
        const long n = n0 + wn * 64 + 16 * bj + 4 * gq;
        int* dst = C + m * p.N + n;
        if (n + 3 <= nlast && (p.N & 3) == 0) {
          *(v4i*)dst = acc[bj][bi];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r <= nlast) dst[r] = acc[bj][bi][r];
        }
      }
    }
    return;
  }
  typedef typename OutT<OUT>::T out_t;
  typedef out_t ov4 __attribute__((ext_vector_type(4)));
  out_t* C = (out_t*)p.c;
  const bool vec_ok = p.ldc % 4 == 0 && ((uintptr_t)C & (4 * sizeof(out_t) - 1)) == 0;
  v4f sb[4], add[4];
#pragma unroll
  for (int bj = 0; bj < 4; ++bj)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long n = min(n0 + wn * 64 + 16 * bj + 4 * gq + r, (long)nlast);
      sb[bj][r] = p.sb[n];
      add[bj][r] = p.bias ? i8_bias(p.bias, p.bias_dt, n) : 0.f;
    }
#pragma unroll
  for (int bi = 0; bi < WMB; ++bi) {
    const long m = m0 + wm * (BM / 2) + 16 * bi + r16;
    if (m >= p.M) continue;
    const float sa = p.sa[m];
#pragma unroll
    for (int bj = 0; bj < 4; ++bj) {
      const long n = n0 + wn * 64 + 16 * bj + 4 * gq;
      out_t* dst = C + m * p.ldc + n;
      ov4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (out_t)((float)acc[bj][bi][r] * sa * sb[bj][r] + add[bj][r]);
      if (n + 3 <= nlast && vec_ok) {
        *(ov4*)dst = o;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r <= nlast) dst[r] = o[r];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// tile256: 256 x 256 outputs per workgroup, 4 waves (2 x 2) of 128 x 128: 256 accumulators and one set of 8 + 8 fragments
// per lane, two stages of 64 KB.  The k-tile's 128 MFMAs run in two halves (columns 0..3, then 4..7 of the wave's eight
// blocks): under the first one the DMA of tile kt+2 goes out into this tile's own stage, whose fragments are all in
// registers; between the halves "tile kt+1 has landed" is awaited; under the second the fragments of tile kt+1 replace
// those that have had their last MFMA.  Rows past M or N re-read the last one and are not stored.
// Bound by the matrix pipes and power: 8192 x 8192 x 8192 391 to 420 us, 2.6 to 2.8 POP/s, in runs of seconds; the first twenty
// launches after idle take 407 to 519 while the clock finds its place.  An MFMA runs in 68 % of the busy
// cycles (tiles of 128 x 128: 721 us, twice the LDS traffic per MFMA).
// ------------------------------------------------------------------------------------------
template <int OUT, bool KT>
__global__ __launch_bounds__(256) void hx_int8_gemm_tile256(I8Args p) {
  typedef typename OutT<OUT>::T out_t;
  constexpr int TILE = 256 * I8_BK;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2][2][TILE];  // [stage][A|B]

  int tm, tn;
  {  // every XCD (workgroup i runs on XCD i % 8) walks a contiguous range of a raster eight tile rows tall
    const int nwg = gridDim.x, wg = blockIdx.x, per = nwg >> 3, rem = nwg & 7, xcd = wg & 7, loc = wg >> 3;
    const int tile = xcd < rem ? xcd * (per + 1) + loc : rem * (per + 1) + (xcd - rem) * per + loc;
    const int group = 8 * (nwg / p.tiles_m), first = (tile / group) * 8, gm = min(p.tiles_m - first, 8);
    tm = first + (tile % group) % gm;
    tn = (tile % group) / gm;
  }
  const long m0 = (long)tm * 256, n0 = (long)tn * 256;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = w >> 1, wn = w & 1;

  // ---- DMA: wave w fetches rows 64w .. 64w+63 of both tiles, eight rows per instruction
  const int lrow = lane >> 3, lpos = lane & 7;
  uint32_t a_vo[8], b_vo[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t chunk = (uint32_t)((lpos ^ ((4 * (i & 1) + (lrow >> 1)) & 7)) * 16);
    a_vo[i] = (uint32_t)min((int)m0 + 64 * w + 8 * i + lrow, p.M - 1) * (uint32_t)p.lda + chunk;
    b_vo[i] = (uint32_t)min((int)n0 + 64 * w + 8 * i + lrow, p.N - 1) * (uint32_t)p.ldb + chunk;
  }
  const uint8_t *A = p.a, *B = p.b;
  const uint32_t a_max = p.a_max, b_max = p.b_max, lds0 = hx_lds_addr(&smem[0][0][0]) + (uint32_t)w * 64 * 128;
  const int nk = p.nk;
  auto issue_one = [&](int kt, int stage, int i) {
    const uint32_t la = lds0 + (uint32_t)stage * 2 * TILE;
    const long t = (long)kt * I8_BK;
    if (i < 8 && KT) hx_g2l16_s(hx_uniform_ptr(A), min(a_vo[i] + (uint32_t)t, a_max), la + i * 1024);
    else if (i < 8) hx_g2l16_s(hx_uniform_ptr(A + t), a_vo[i], la + i * 1024);
    else if (KT) hx_g2l16_s(hx_uniform_ptr(B), min(b_vo[i - 8] + (uint32_t)t, b_max), la + TILE + (i - 8) * 1024);
    else hx_g2l16_s(hx_uniform_ptr(B + t), b_vo[i - 8], la + TILE + (i - 8) * 1024);
  };

  auto zero_tail = [&](int kt) {  // as in the kernel above; rows 8i .. of the wave hold chunk c at c ^ (4 (i & 1) + row / 2)
    if (!KT || kt != nk - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((lpos ^ ((4 * (i & 1) + (lrow >> 1)) & 7)) * 16 >= p.tail)
        *(v4i*)&smem[kt & 1][0][w * 64 * 128 + i * 1024 + lane * 16] = (v4i){0, 0, 0, 0};
  };

  const int r16 = lane & 15, gq = lane >> 4;
  const int kq = (gq >> 1) ^ ((gq & 1) * 3);
  const int x16 = ((2 * kq) ^ ((r16 >> 1) & 7)) * 16;
  const int a_base = (wm * 128 + r16) * 128, b_base = (wn * 128 + r16) * 128;
  v4i fa[8][2], fb[8][2];
  auto load_a = [&](int stage, int f) {
    const uint8_t* st = &smem[stage][0][0] + a_base + f * 2048;
    fa[f][0] = *(const v4i*)(st + x16), fa[f][1] = *(const v4i*)(st + (x16 ^ 16));
  };
  auto load_b = [&](int stage, int f) {
    const uint8_t* st = &smem[stage][1][0] + b_base + f * 2048;
    fb[f][0] = *(const v4i*)(st + x16), fb[f][1] = *(const v4i*)(st + (x16 ^ 16));
  };
  // acc[bj][bi][r] is C[m0 + wm*128 + 16 bi + lane%16][n0 + wn*128 + 16 bj + 4*(lane/16) + r]
  v4i acc[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      acc[i][j] = (v4i){0, 0, 0, 0};
      hx_acc_pin(acc[i][j]);
    }

  auto ktile = [&](int kt, auto with_dma) {
    constexpr bool dma = decltype(with_dma)::value;
    const int stage = kt & 1;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      const int bj = i & 3, hi = (i >> 2) & 1, bi = i >> 3;
      hx_mfma_16x16x64_i8_acc(acc[bj][bi], fb[bj][hi], fa[bi][hi]);
      if (dma && (i & 3) == 3) issue_one(kt + 2, stage, i >> 2);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (dma) __builtin_amdgcn_s_waitcnt(hx_vmcnt_imm(16));  // tile kt+1 has landed, tile kt+2 stays in flight
    else HX_WAIT_VM0();
    zero_tail(kt + 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      const int bj = 4 + (i & 3), hi = (i >> 2) & 1, bi = i >> 3;
      hx_mfma_16x16x64_i8_acc(acc[bj][bi], fb[bj][hi], fa[bi][hi]);
      if ((i & 7) == 7) load_a(stage ^ 1, bi);
      if ((i & 15) == 2) load_b(stage ^ 1, i >> 4);
      if (i >= 60) load_b(stage ^ 1, 4 + (i - 60));  // its last MFMA of this tile is out
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();  // every wave has read tile kt+1's fragments: its stage is free
  };
#pragma unroll
  for (int i = 0; i < 16; ++i) issue_one(0, 0, i);
  if (nk > 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i) issue_one(1, 1, i);
    __builtin_amdgcn_s_waitcnt(hx_vmcnt_imm(16));
  } else {
    HX_WAIT_VM0();
  }
  zero_tail(0);
  __syncthreads();
#pragma unroll
  for (int f = 0; f < 8; ++f) load_a(0, f), load_b(0, f);
  __syncthreads();
  hx_mfma_settle();
  int kt = 0;
  for (; kt + 2 < nk; ++kt) ktile(kt, std::true_type{});
  for (; kt < nk; ++kt) ktile(kt, std::false_type{});  // the last two have nothing left to fetch
  // (past the last tile the fragments are refilled from a stage that holds an older tile, or nothing; nobody uses them)
  hx_mfma_settle();
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) hx_acc_pin(acc[i][j]);  // no copy of an accumulator before the wait

  // ---- epilogue: 32 rows x 128 columns at a time through the wave's own quarter of the LDS, so that every store
  // instruction writes whole row pieces
  constexpr int ESZ = (int)sizeof(out_t), ROWB = 128 * ESZ, RSTR = ROWB + 16, LPR = ROWB / 16, RPI = 64 / LPR;
  typedef out_t ov4 __attribute__((ext_vector_type(4)));
  uint8_t* st = &smem[0][0][0] + w * TILE;
  out_t* C = (out_t*)p.c;
  const long col0 = n0 + wn * 128;
  v4f sb[8], add[8];
#pragma unroll
  for (int bj = 0; bj < 8; ++bj)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long n = min(col0 + 16 * bj + 4 * gq + r, (long)p.N - 1);
      sb[bj][r] = p.sb[n];
      add[bj][r] = p.bias ? i8_bias(p.bias, p.bias_dt, n) : 0.f;
    }
  const bool vec = p.ldc % (16 / ESZ) == 0 && ((uintptr_t)C & 15) == 0;
#pragma unroll
  for (int b32 = 0; b32 < 4; ++b32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float sa = p.sa[min(m0 + wm * 128 + b32 * 32 + h * 16 + r16, (long)p.M - 1)];
#pragma unroll
      for (int bj = 0; bj < 8; ++bj) {
        ov4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (out_t)((float)acc[bj][2 * b32 + h][r] * sa * sb[bj][r] + add[bj][r]);
        *(ov4*)(st + (h * 16 + r16) * RSTR + (bj * 16 + 4 * gq) * ESZ) = o;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (the LDS runs one wave's operations in order)
#pragma unroll
    for (int q = 0; q < 32 / RPI; ++q) {
      const int row = q * RPI + lane / LPR;
      const v4i v = *(const v4i*)(st + row * RSTR + lane % LPR * 16);
      const long m = m0 + wm * 128 + b32 * 32 + row, n = col0 + lane % LPR * (16 / ESZ);
      if (m < p.M) {
        out_t* dst = C + m * p.ldc + n;
        if (vec && n + 16 / ESZ <= p.N) {
          *(v4i*)dst = v;
        } else {
          const out_t* e = (const out_t*)&v;
          for (int b = 0; b < 16 / ESZ; ++b)
            if (n + b < p.N) dst[b] = e[b];
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// ------------------------------------------------------------------------------------------
// skinny: M <= 32 (MB blocks of 16 rows).  The weights are read once, straight into registers; one workgroup of 8 waves per
// compute unit walks groups of 16 columns, wave w multiplies the 128-byte k-steps w, w+8, ... of each and keeps the rows of
// A for them in registers all along.  One load instruction covers eight rows of 128 bytes (whole lines): lane (j = lane%16,
// g = lane/16) takes chunk 2g + (j&1) of row j>>1, a second instruction rows 8..15 with the other chunk; one exchange with
// the neighbouring lane leaves chunks 2g and 2g+1 of row (j>>1) + 8 (j&1), two MFMA operands.  The registers of a step are
// refilled with the same step of the next group as soon as the operands are built, so that about one group per wave (128 KB
// per compute unit) is in flight, also across the barrier that adds up the eight waves' sums.
// NS > 0: every wave has NS steps and the loads in flight can be counted; NS = 0: any number up to eight, and a K that is
// not a multiple of 128 (rows are read on, clamped to the end of the matrix, and A becomes zero there).
// split (gridDim.y > 1): workgroup row y adds up its steps into its own slab of 32-bit integers.
// Bound by memory: 16 x 28672 x 8192 37.0 us, 6.3 TB/s (through the LDS tiles above 50.6), 32 rows 43.0 (48.4), 1 x 4096 x
// 4096 4.8 (10.7).
// ------------------------------------------------------------------------------------------
#define I8S_WAVES 8
#define I8S_STEPS 8
template <int OUT, int NS, int MB, bool SPLIT>
__global__ __launch_bounds__(512) void hx_int8_gemm_skinny(I8Args p) {
  typedef typename OutT<OUT>::T out_t;
  constexpr bool FULL = NS > 0;
  __shared__ __attribute__((aligned(16))) int red[2][I8S_WAVES][MB * 4][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, g = lane >> 4, odd = j & 1;
  const int first = SPLIT ? p.kt_per_split * (int)blockIdx.y : 0;                  // k-steps of this workgroup
  const int steps = SPLIT ? min(p.kt_per_split, p.nk - first) : p.nk;
  const int nmine = FULL ? NS : (steps - w + I8S_WAVES - 1) / I8S_WAVES;
  const int ncg = (p.N + 15) >> 4, grid = (int)gridDim.x;

  const int c_lo = (2 * g + odd) * 16, c_hi = (2 * g + (odd ^ 1)) * 16;
  const long k0 = (long)(first + w) * I8_BK;
  const uint8_t *p0, *p1;
  const uint8_t *a_end = p.a + p.a_max, *end = p.b + p.b_max;
  auto point_at = [&](int cg) {
    p0 = p.b + (long)min(cg * 16 + (j >> 1), p.N - 1) * p.ldb + c_lo + k0;
    p1 = p.b + (long)min(cg * 16 + 8 + (j >> 1), p.N - 1) * p.ldb + c_hi + k0;
  };
  v4i x0[I8S_STEPS], x1[I8S_STEPS];
  auto load_step = [&](int s) {
    const uint8_t *q0 = p0 + (long)s * I8S_WAVES * I8_BK, *q1 = p1 + (long)s * I8S_WAVES * I8_BK;
    if (!FULL) q0 = q0 < end ? q0 : end, q1 = q1 < end ? q1 : end;
    x0[s] = __builtin_nontemporal_load((const v4i*)q0);
    x1[s] = __builtin_nontemporal_load((const v4i*)q1);
  };
  int cg = (int)blockIdx.x;  // grid <= ncg: every workgroup has a group
  point_at(cg);
#pragma unroll
  for (int s = 0; s < I8S_STEPS; ++s)
    if (FULL ? s < NS : s < nmine) load_step(s);

  // rows of A like those of B: lane (j, g) ends up with chunks 2g, 2g+1 of row 16 mb + (j>>1) + 8 (j&1)
  v4i alo[MB][I8S_STEPS], ahi[MB][I8S_STEPS];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const uint8_t* ap0 = p.a + (long)min(mb * 16 + (j >> 1), p.M - 1) * p.lda + c_lo + k0;
    const uint8_t* ap1 = p.a + (long)min(mb * 16 + 8 + (j >> 1), p.M - 1) * p.lda + c_hi + k0;
#pragma unroll
    for (int s = 0; s < I8S_STEPS; ++s)
      if (FULL ? s < NS : s < nmine) {
        const uint8_t *q0 = ap0 + (long)s * I8S_WAVES * I8_BK, *q1 = ap1 + (long)s * I8S_WAVES * I8_BK;
        if (!FULL) q0 = q0 < a_end ? q0 : a_end, q1 = q1 < a_end ? q1 : a_end;
        v4i a0 = *(const v4i*)q0, a1 = *(const v4i*)q1;
        if (!FULL && first + w + s * I8S_WAVES == p.nk - 1) {  // nothing behind K
          if (c_lo >= p.tail) a0 = (v4i){0, 0, 0, 0};
          if (c_hi >= p.tail) a1 = (v4i){0, 0, 0, 0};
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          alo[mb][s][d] = odd ? a1[d] : a0[d];
          ahi[mb][s][d] = __builtin_amdgcn_mov_dpp(odd ? a0[d] : a1[d], 0xB1, 0xF, 0xF, true);  // from lane ^ 1
        }
        if (MB > 1) __builtin_amdgcn_sched_barrier(0);  // bounds the raw lines in flight
      }
  }

  int parity = 0;
  // whether there is a next group is a property of the body, so that its loads stay countable
  auto one_group = [&](auto more_c) {
    constexpr bool more = decltype(more_c)::value;
    if (more) point_at(cg + grid);
    v4i acc[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[mb] = (v4i){0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < I8S_STEPS; ++s)
      if (FULL ? s < NS : s < nmine) {
        v4i lo, hi;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          lo[d] = odd ? x1[s][d] : x0[s][d];
          hi[d] = __builtin_amdgcn_mov_dpp(odd ? x0[s][d] : x1[s][d], 0xB1, 0xF, 0xF, true);
        }
        if (more) load_step(s);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          acc[mb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(alo[mb][s], lo, acc[mb], 0, 0, 0);
          acc[mb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ahi[mb][s], hi, acc[mb], 0, 0, 0);
        }
      }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[parity][w][4 * mb + r][lane] = acc[mb][r];
    __syncthreads();
    if (tid < 256 * MB) {
      const int l2 = tid & 63, rr = tid >> 6;
      int sum = 0;
#pragma unroll
      for (int ww = 0; ww < I8S_WAVES; ++ww) sum += red[parity][ww][rr][l2];
      const int j2 = l2 & 15, i2 = 4 * (l2 >> 4) + (rr & 3);  // column and row of the MFMA
      const int m = 16 * (rr >> 2) + (i2 >> 1) + 8 * (i2 & 1), n = cg * 16 + (j2 >> 1) + 8 * (j2 & 1);
      if (m < p.M && n < p.N) {
        if (SPLIT) ((int*)p.c)[((long)blockIdx.y * p.M + m) * p.N + n] = sum;
        else ((out_t*)p.c)[(long)m * p.ldc + n] = (out_t)((float)sum * p.sa[m] * p.sb[n] + (p.bias ? i8_bias(p.bias, p.bias_dt, n) : 0.f));
      }
    }
    parity ^= 1;  // the next group writes the other buffer: one barrier per group is enough
    cg += grid;
  };
  while (cg + grid < ncg) one_group(std::true_type{});
  one_group(std::false_type{});
}

// split-K: C = cast(sum over the slabs [split][M][N] * scales + bias); one thread per four columns
template <int OUT>
__global__ __launch_bounds__(256) void hx_int8_gemm_split_reduce(I8Args p, const int* __restrict__ part, int splits) {
  typedef typename OutT<OUT>::T out_t;
  const int n4 = (p.N + 3) >> 2;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)p.M * n4) return;
  const long m = id / n4, n = (id % n4) * 4;
  int acc[4] = {0, 0, 0, 0};
  for (int s = 0; s < splits; ++s)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < p.N) acc[r] += part[((long)s * p.M + m) * p.N + n + r];
  const float sa = p.sa[m];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < p.N)
      ((out_t*)p.c)[m * p.ldc + n + r] = (out_t)((float)acc[r] * sa * p.sb[n + r] + (p.bias ? i8_bias(p.bias, p.bias_dt, n + r) : 0.f));
}

// src[r * sr + k * sk] -> dst[r][ld], zeros behind K.  Rows of contiguous bytes: 16 at a time whatever their alignment.
__global__ __launch_bounds__(256) void hx_int8_pack_rows(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, long rows, int K, long sr,
                                                        int ld) {
  const int per = ld >> 4;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= rows * per) return;
  const long r = id / per;
  const int k = (int)(id % per) * 16;
  const uint8_t* s = src + r * sr + k;
  typedef int v4iu __attribute__((ext_vector_type(4), aligned(1)));
  v4i v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    v = *(const v4iu*)s;
  } else {
    for (int e = 0; e < 16; ++e)
      if (k + e < K) ((uint8_t*)&v)[e] = s[e];
  }
  *(v4i*)(dst + r * ld + k) = v;
}
// any strides, through a 64 x 64 tile
__global__ __launch_bounds__(256) void hx_int8_pack_any(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, int rows, int K, long sr,
                                                       long sk, int ld) {
  __shared__ uint8_t t[64][64 + 4];
  const int r0 = blockIdx.x * 64, k0 = blockIdx.y * 64, x = threadIdx.x & 63;
  for (int y = threadIdx.x >> 6; y < 64; y += 4) {
    const int r = r0 + x, k = k0 + y;
    t[y][x] = r < rows && k < K ? src[r * sr + k * sk] : (uint8_t)0;
  }
  __syncthreads();
  for (int y = threadIdx.x >> 6; y < 64; y += 4) {
    const int r = r0 + y, k = k0 + x;
    if (r < rows && k < ld) dst[(long)r * ld + k] = t[x][y];
  }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
struct I8Plan {
  bool copy_a, copy_b, tail;  // tail: K % 128 != 0 with A or B read in place
  int64_t ka;                 // padded row length of the copies
  int bm, bn, splits, kt_per_split;
  int ns;                     // skinny kernel: steps per wave as a constant, 0 not constant; -1 another kernel
  size_t a_off, b_off, part_off, bytes;
};

static void i8_offsets(I8Plan& p, int64_t M, int64_t N) {
  size_t at = 0;
  auto take = [&](bool want, int64_t bytes) {
    const size_t here = at;
    if (want) at += ((size_t)bytes + 255) & ~(size_t)255;
    return here;
  };
  p.a_off = take(p.copy_a, M * p.ka);
  p.b_off = take(p.copy_b, N * p.ka);
  p.part_off = take(p.splits > 1, (int64_t)p.splits * M * N * 4);
  p.bytes = at;
}

// Up to 32 rows: k in pieces of at most 64 steps per workgroup (eight waves of up to eight), as few as that takes.  More of them,
// for the compute units that the groups of 16 columns leave idle, cost more in partial sums and a second launch than they
// give: 16 x 2048 x 2048 6.5 us, whole 3.6; 16 x 64 x 8192 8.8 and 5.9; 32 x 256 x 8192 9.9 and 8.2; 1 x 64 x 65536 in 64 pieces
// 31.4, in eight 11.3; 16 x 1024 x 16384 in four 8.8, in two 9.2.
static I8Plan i8_plan_skinny(I8Plan p, int64_t M, int64_t N, int64_t K) {
  const int64_t nk = p.ka / I8_BK;
  const int64_t s = (nk + 63) / 64;
  const int64_t per = ((nk + s - 1) / s + 7) / 8 * 8;
  p.bm = 16, p.bn = 16;
  p.splits = (int)((nk + per - 1) / per);
  p.kt_per_split = p.splits > 1 ? (int)per : 0;
  p.ns = nk % per == 0 && !p.tail ? (int)(per / 8) : 0;
  i8_offsets(p, M, N);
  return p;
}

static I8Plan i8_plan(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb_k, int64_t ldb_n, bool a_aligned, bool b_aligned) {
  I8Plan p;
  p.ka = (K + I8_BK - 1) / I8_BK * I8_BK;
  p.copy_a = !(K % 16 == 0 && lda % 16 == 0 && a_aligned && M * lda <= (1LL << 32) - 512);
  p.copy_b = !(K % 16 == 0 && ldb_k == 1 && ldb_n >= K && ldb_n % 16 == 0 && b_aligned && N * ldb_n <= (1LL << 32) - 512);
  p.tail = K % I8_BK != 0 && !(p.copy_a && p.copy_b);
  p.ns = -1;
  if (M <= 32) return i8_plan_skinny(p, M, N, K);
  // Rows of the tile, 64 or 128 (of 128 columns) or 256 (of 256), and workgroups that share the k-tiles of one: what a
  // launch takes in units of 10 ns, from rounds of one workgroup per compute unit, a k-tile's time and what surrounds the
  // loop, and for a split the partial sums' way through memory and the second launch.  At least eight k-tiles each, partial
  // sums below 32 MB.  Measured with 64, 128, 256 rows: 512 x 4096 x 4096 15.4, 20 (23.5 split in two), 44 us; 128 x 8192 x
  // 8192 21.2 (in two), 25.0 (in four), 76; 777 x 4096 x 4096 28.3, 20.4, 45; 1024 x 8192 x 8192 98.6, 70.8, 87.5;
  // 8192 x 8192 x 8192 128 and 256 rows: 721 and 411.
  const int64_t nk = p.ka / I8_BK, cus = hx_cu_count();
  static const struct { int bm, bn, step, around; } tile[3] = {{64, 128, 33, 360}, {128, 128, 47, 530}, {256, 256, 150, 600}};
  int64_t least = INT64_MAX;
  for (const auto& t : tile) {
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
    if (t.bm == 256 && M <= 128) continue;
    for (int64_t s = 1; s == 1 || (t.bm != 256 && s * tiles <= cus && 8 * s <= nk && s * M * N * 4 <= (32LL << 20)); ++s) {
      const int64_t per = (nk + s - 1) / s, n = (nk + per - 1) / per;
      const int64_t cost = (tiles * n + cus - 1) / cus * (t.step * per + t.around) + (n > 1 ? 300 + n * M * N * 4 / 20000 : 0);
      if (cost >= least) continue;
      least = cost;
      p.bm = t.bm, p.bn = t.bn, p.splits = (int)n, p.kt_per_split = n > 1 ? (int)per : 0;
    }
  }
  i8_offsets(p, M, N);
  return p;
}

static int i8_check(const char* who, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) {
    hx_set_error("%s: negative size M=%lld N=%lld K=%lld", who, (long long)M, (long long)N, (long long)K);
    return HX_ERR_BAD_ARG;
  }
  if (K > 131071) {
    hx_set_error("%s: K=%lld: a sum of more than 131071 products does not fit in 32 bits", who, (long long)K);
    return HX_ERR_UNSUPPORTED;
  }
  const int64_t ka = (K + I8_BK - 1) / I8_BK * I8_BK;
  if (M >= (1LL << 31) - 256 || N >= (1LL << 31) - 256 || (M + 63) / 64 * ((N + 127) / 128) >= (1LL << 31) || M * ka >= (1LL << 32) ||
      N * ka >= (1LL << 32)) {
    hx_set_error("%s: operands of 4 GB or more", who);
    return HX_ERR_UNSUPPORTED;
  }
  return 0;
}

extern "C" size_t hx_int8_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb_k, int64_t ldb_n, const void* a,
                                               const void* b) {
  if (M <= 0 || N <= 0 || K <= 0 || i8_check("hx_int8_gemm", M, N, K) != 0) return 0;
  return i8_plan(M, N, K, lda, ldb_k, ldb_n, ((uintptr_t)a & 15) == 0, ((uintptr_t)b & 15) == 0).bytes;
}

extern "C" int hx_int8_gemm_path(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb_k, int64_t ldb_n, const void* a, const void* b) {
  if (M <= 0 || N <= 0 || K <= 0 || i8_check("hx_int8_gemm", M, N, K) != 0) return 0;
  const I8Plan p = i8_plan(M, N, K, lda, ldb_k, ldb_n, ((uintptr_t)a & 15) == 0, ((uintptr_t)b & 15) == 0);
  return (p.ns >= 0 ? 1 : p.bm == 64 ? 2 : p.bm == 128 ? 3 : 4) + (p.splits > 1 ? 8 : 0) + (p.tail ? 16 : 0);
}

static void i8_pack(const void* src, uint8_t* dst, int64_t rows, int64_t K, int64_t sr, int64_t sk, int64_t ld, hipStream_t s) {
  if (sk == 1)
    hx_launch(hx_int8_pack_rows, dim3((unsigned)((rows * (ld / 16) + 255) / 256)), dim3(256), 0, s, (const uint8_t*)src, dst, (long)rows, (int)K,
              (long)sr, (int)ld);
  else
    hx_launch(hx_int8_pack_any, dim3((unsigned)((rows + 63) / 64), (unsigned)((ld + 63) / 64)), dim3(256), 0, s, (const uint8_t*)src, dst,
              (int)rows, (int)K, (long)sr, (long)sk, (int)ld);
}

template <int OUT, int BM>
static void i8_launch_tile(const I8Args& a, const I8Plan& p, dim3 grid, hipStream_t s) {
  if (p.splits > 1) {
    if (p.tail) hx_launch(hx_int8_gemm_tile<HX_F32, BM, true, true>, grid, dim3(256), 0, s, a);
    else hx_launch(hx_int8_gemm_tile<HX_F32, BM, false, true>, grid, dim3(256), 0, s, a);
  } else {
    if (p.tail) hx_launch(hx_int8_gemm_tile<OUT, BM, true, false>, grid, dim3(256), 0, s, a);
    else hx_launch(hx_int8_gemm_tile<OUT, BM, false, false>, grid, dim3(256), 0, s, a);
  }
}

template <int OUT, int MB, bool SPLIT>
static void i8_launch_skinny(const I8Args& a, int ns, dim3 grid, hipStream_t s) {
  switch (ns) {
#define I8S_CASE(NS) \
  case NS: hx_launch(hx_int8_gemm_skinny<OUT, NS, MB, SPLIT>, grid, dim3(512), 0, s, a); break;
    I8S_CASE(1) I8S_CASE(2) I8S_CASE(3) I8S_CASE(4) I8S_CASE(5) I8S_CASE(6) I8S_CASE(7) I8S_CASE(8)
#undef I8S_CASE
    default: hx_launch(hx_int8_gemm_skinny<OUT, 0, MB, SPLIT>, grid, dim3(512), 0, s, a);
  }
}

template <int OUT>
static void i8_launch(I8Args a, const I8Plan& p, void* ws, hipStream_t s) {
  a.tiles_m = (a.M + p.bm - 1) / p.bm, a.bn = p.bn, a.kt_per_split = p.kt_per_split;
  const dim3 grid((unsigned)(a.tiles_m * ((a.N + p.bn - 1) / p.bn)), (unsigned)p.splits);
  void* c = a.c;
  if (p.splits > 1) a.c = (uint8_t*)ws + p.part_off;
  if (p.ns >= 0) {
    const int ncg = (a.N + 15) / 16, cus = hx_cu_count();
    const dim3 sg((unsigned)(ncg < cus ? ncg : cus), (unsigned)p.splits);
    if (p.splits > 1) {
      if (a.M <= 16) i8_launch_skinny<HX_F32, 1, true>(a, p.ns, sg, s);
      else i8_launch_skinny<HX_F32, 2, true>(a, p.ns, sg, s);
    } else {
      if (a.M <= 16) i8_launch_skinny<OUT, 1, false>(a, p.ns, sg, s);
      else i8_launch_skinny<OUT, 2, false>(a, p.ns, sg, s);
    }
  } else if (p.bm == 256) {
    if (p.tail) hx_launch(hx_int8_gemm_tile256<OUT, true>, grid, dim3(256), 0, s, a);
    else hx_launch(hx_int8_gemm_tile256<OUT, false>, grid, dim3(256), 0, s, a);
  } else if (p.bm == 64) i8_launch_tile<OUT, 64>(a, p, grid, s);
  else i8_launch_tile<OUT, 128>(a, p, grid, s);
  if (p.splits > 1) {
    const int* part = (const int*)a.c;
    a.c = c;
    const long quads = (long)a.M * ((a.N + 3) / 4);
    hx_launch(hx_int8_gemm_split_reduce<OUT>, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, a, part, p.splits);
  }
}

extern "C" int hx_int8_gemm(const void* a, const void* b, void* c, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb_k, int64_t ldb_n,
                            int64_t ldc, const float* scale_a, const float* scale_b, const void* bias, int bias_dtype, int out_dtype,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "hx_int8_gemm";
  int rc = i8_check(who, M, N, K);
  if (rc != 0) return rc;
  if (out_dtype != HX_F16 && out_dtype != HX_BF16 && out_dtype != HX_F32) {
    hx_set_error("%s: out_dtype must be HX_F16, HX_BF16 or HX_F32, got %d", who, out_dtype);
    return HX_ERR_BAD_ARG;
  }
  if (bias && bias_dtype != HX_F16 && bias_dtype != HX_BF16 && bias_dtype != HX_F32) {
    hx_set_error("%s: bias dtype must be HX_F16, HX_BF16 or HX_F32, got %d", who, bias_dtype);
    return HX_ERR_BAD_ARG;
  }
  if (M == 0 || N == 0) return 0;
  if (K == 0) {
    hx_set_error("%s: K = 0", who);
    return HX_ERR_UNSUPPORTED;
  }
  if (!a || !b || !c || !scale_a || !scale_b) {
    hx_set_error("%s: null pointer", who);
    return HX_ERR_BAD_ARG;
  }
  if (lda < K || ldc < N || ldb_k < 1 || ldb_n < 1) {
    hx_set_error("%s: leading dimension smaller than row length (lda=%lld K=%lld ldc=%lld N=%lld ldb=%lld,%lld)", who, (long long)lda,
                 (long long)K, (long long)ldc, (long long)N, (long long)ldb_k, (long long)ldb_n);
    return HX_ERR_BAD_ARG;
  }
  const uintptr_t oes = out_dtype == HX_F32 ? 4 : 2, bes = bias_dtype == HX_F32 ? 4 : 2;
  if (((uintptr_t)c & (oes - 1)) || (bias && ((uintptr_t)bias & (bes - 1))) || (((uintptr_t)scale_a | (uintptr_t)scale_b) & 3)) {
    hx_set_error("%s: pointers must be aligned to their elements", who);
    return HX_ERR_UNSUPPORTED;
  }
  const I8Plan p = i8_plan(M, N, K, lda, ldb_k, ldb_n, ((uintptr_t)a & 15) == 0, ((uintptr_t)b & 15) == 0);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || ((uintptr_t)workspace & 255))) {
    hx_set_error("%s: workspace must be 256-byte aligned and at least %zu bytes (got %zu)", who, p.bytes, workspace_bytes);
    return HX_ERR_WORKSPACE;
  }
  hipStream_t s = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  I8Args g;
  g.a = (const uint8_t*)a, g.b = (const uint8_t*)b, g.c = c, g.sa = scale_a, g.sb = scale_b, g.bias = bias, g.bias_dt = bias_dtype;
  g.M = (int)M, g.N = (int)N, g.nk = (int)(p.ka / I8_BK), g.lda = lda, g.ldb = ldb_n, g.ldc = ldc;
  if (p.copy_a) {
    i8_pack(a, ws + p.a_off, M, K, lda, 1, p.ka, s);
    g.a = ws + p.a_off, g.lda = p.ka;
  }
  if (p.copy_b) {
    i8_pack(b, ws + p.b_off, N, K, ldb_n, ldb_k, p.ka, s);
    g.b = ws + p.b_off, g.ldb = p.ka;
  }
  g.tail = (int)(K - (p.ka - I8_BK));
  g.a_max = (uint32_t)((M - 1) * g.lda + (p.copy_a ? p.ka : K) - 16);
  g.b_max = (uint32_t)((N - 1) * g.ldb + (p.copy_b ? p.ka : K) - 16);
  if (out_dtype == HX_F16) i8_launch<HX_F16>(g, p, ws, s);
  else if (out_dtype == HX_BF16) i8_launch<HX_BF16>(g, p, ws, s);
  else i8_launch<HX_F32>(g, p, ws, s);
  const hipError_t e = hx_launch_status();
  if (e != hipSuccess) {
    hx_set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return (int)e;
  }
  return 0;
}
