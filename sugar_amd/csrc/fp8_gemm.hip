// Matrix product of two 8-bit operands with block scales (format and instructions: blockfp8.h), gfx950.
//
//   y[r][o] = relu(sum_k a[r][k] w[o][k]) * scale[o] + shift[o]
//
//   direct     few rows: operands from memory into registers, K dealt out over the waves of a workgroup
//   tile       TM channels x TN rows a workgroup, k-tiles of one 128-column block through two LDS stages filled by DMA
//   short      K <= 512, many rows: weights in registers, only rows move
//   persist    256 x 256 tiles walked by one workgroup per CU (bf16 outputs of large products)
//
// A k-tile row is 128 bytes in LDS as it is in the 16-bit GEMMs of conv1x1.hip (there 64 columns): the same bytes per
// step, the same chunk swizzle, the same matrix-pipe time per step, and twice the operations.
#include "blockfp8.h"

namespace sugar {

namespace {

struct LinearArgs {
  const uint8_t *a, *ae, *w, *we;
  unsigned lda, ldae, ldw, ldwe;      // rows x stride fits 32 bits (launch_fp8_linear cuts longer operands)
  int64_t ldy;
  void* y;
  const float *scale, *shift;         // under EPI_AFFINE; either may be missing (1 / 0), not both
  int rows, n, kb, flags, out_f32;
  int n_co_tiles;
  bf16* y2;                           // second store of columns >= y2_from (whole chunks of 8), or nullptr
  int64_t ldy2;
  int y2_from;
};

// ReLU in one instruction that hands NaN on (a maximum, not a maxNum)
__device__ __forceinline__ float relu_nan(float v) { return __builtin_elementwise_maximum(v, 0.f); }

// Memory -> LDS, BYTES a lane to consecutive LDS addresses: uniform base (in scalar registers, kept apart from the lane's
// 32-bit offset: hipcc would otherwise carry a 64-bit address per instruction through the k-loop and spill) + offset.
template <int BYTES>
__device__ __forceinline__ void dma(const uint8_t* base, unsigned off, unsigned char* lds) {
  asm("" : "+s"(base));
  const auto src = (const __attribute__((address_space(1))) void*)(base + off);
  const auto dst = (__attribute__((address_space(3))) void*)lds;
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds(src, dst, 4, 0, 0);
}

// lane (fr, fq)'s 32 bytes of a k-tile row: chunks fq and 4 + fq (any 32, the same for both operands)
__device__ __forceinline__ i32x8 frag(const unsigned char* base, int row, int fq) {
  i32x8 f;
  *(i32x4*)&f = *(const i32x4*)(base + swz(row, fq));
  *((i32x4*)&f + 1) = *(const i32x4*)(base + swz(row, 4 + fq));
  return f;
}

__device__ __forceinline__ f32x4 epilogue4(f32x4 v, bool relu, bool affine, f32x4 sc, f32x4 sh) {
  if (relu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = relu_nan(v[i]);
  }
  if (affine) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(v[i], sc[i], sh[i]);
  }
  return v;
}

// Four consecutive results of one row, from channel co on.
__device__ __forceinline__ void store_out4(const LinearArgs& p, int64_t r, int co, f32x4 v) {
  if (p.out_f32) {
    float* y = (float*)p.y + r * p.ldy + co;
    if (co + 4 <= p.n) {
      *(f32x4_u*)y = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (co + i < p.n) y[i] = v[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (co + i >= p.n) break;
    ((bf16*)p.y)[r * p.ldy + co + i] = (bf16)v[i];
    if (p.y2 && co + i >= p.y2_from) p.y2[r * p.ldy2 + co + i] = (bf16)v[i];
  }
}

// ------------------------------------------------------------------------------------------ few rows
// Operands straight from memory into the matrix instruction's registers, 16 channels x 16 rows a workgroup, K dealt out over
// its waves (a wave's loads are all independent: the latency of one trip to memory bounds the call, not its bytes) and their
// sums joined in LDS in wave order.  WIDE: 16-bit products (float32 outputs).
// 1 x 1536 -> 1536 (2.4 MB of weights): 3.5 us on the device.
template <int NW, bool WIDE>
__global__ __launch_bounds__(64 * NW) void fp8_linear_direct_kernel(LinearArgs p) {
  __shared__ f32x4 part[NW][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
  const int co = blockIdx.x * 16, r0 = blockIdx.y * 16;
  const int wrow = min(co + fr, p.n - 1), ar = min(r0 + fr, p.rows - 1);
  const uint8_t *wp = p.w + (unsigned)wrow * p.ldw + fq * 32, *wep = p.we + (unsigned)wrow * p.ldwe;
  const uint8_t *ap = p.a + (unsigned)ar * p.lda + fq * 32, *aep = p.ae + (unsigned)ar * p.ldae;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int kb = wv; kb < p.kb; kb += NW) {
    i32x8 wf, af;
    *(i32x4*)&wf = *(const i32x4*)(wp + kb * 128);
    *((i32x4*)&wf + 1) = *(const i32x4*)(wp + kb * 128 + 16);
    *(i32x4*)&af = *(const i32x4*)(ap + kb * 128);
    *((i32x4*)&af + 1) = *(const i32x4*)(ap + kb * 128 + 16);
    const int ew = wep[kb], ea = aep[kb];
    if constexpr (WIDE) {
      bf16x8 wh[4], ah[4];
      fp8_to_bf16(wf, ew, wh);
      fp8_to_bf16(af, ea, ah);
      acc = mfma_wide(wh, ah, acc);
    } else {
      acc = mfma_fp8<0, 0>(wf, af, acc, ew, ea);
    }
  }
  part[wv][lane] = acc;
  __syncthreads();
  if (wv) return;
  f32x4 v = part[0][lane], sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 1; k < NW; ++k) v += part[k][lane];
  if (p.flags & EPI_AFFINE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p.scale) sc[i] = p.scale[min(co + 4 * fq + i, p.n - 1)];
      if (p.shift) sh[i] = p.shift[min(co + 4 * fq + i, p.n - 1)];
    }
  }
  v = epilogue4(v, p.flags & EPI_RELU, p.flags & EPI_AFFINE, sc, sh);
  if (r0 + fr < p.rows) store_out4(p, r0 + fr, co + 4 * fq, v);
}

// ------------------------------------------------------------------------------------------ one tile
// One TM x TN output tile by a workgroup of NW waves = 2 (channels) x NW / 2 (rows).  Steps of KS k-tiles through two stages: wait
// for this wave's share of a step, barrier, issue the DMA of the next into the buffer the last was read from, compute; what a
// workgroup waits for the DMA, the two to four others of its CU fill.  A CU with one workgroup has nothing to fill a step's
// barrier and latencies with: steps of 4 (301 x 1536 -> 1536 5.5 us, by single k-tiles 5.9; deeper rings of single k-tiles do not
// help).  Exponents travel as one dword per row and four k-tiles, staged with the first of the four (double buffer) and shifted
// down a byte per k-tile.
// Bound by the DMA into LDS (128 x 128 tiles: 128 operations a byte) and, at few k-tiles, by the first tile's way in and the
// stores: 301 x 1536 -> 1536 5.5 us (64 x 64), float32 output 8.0; 19264 x 528 -> 536 14.8 us, float32 21.8.
// 128 x 128 with float32 outputs: 4 waves of 64 x 64 convert 8 fragments for 16 products where 8 waves of 64 x 32 convert 6 for
// 8; 77056 x 1536 -> 1536 352 us (1.03 PF) against 377, x 100 -> 1400 121 / 153, 25000 x 300 -> 700 23.9 / 23.0.  Left out one at
// a time (8 waves): conversions 70 us, products 67, stores 79.  A persistent form that fetches the next tile under the epilogue
// and spreads the stores over its k-loop was built and dropped: 362.
constexpr int linear_tile_lds(int TM, int TN, int KS) { return (TM + TN) * (2 * KS * 128 + 8) + 8 * TM; }

template <int TM, int TN, int NW, bool WIDE, int KS = 1>
__device__ __forceinline__ void fp8_tile(const LinearArgs& p, const int co_base, const int r_base) {
  constexpr int STAGE_BYTES = (TM + TN) * 128;
  constexpr int WN = NW / 2, CW = TM / 2, FW = TN / WN, MI = CW / 16, NJ = FW / 16, WI = TM / (8 * NW), XI = TN / (8 * NW), SI = (TM + TN) / 64;
  // Written into the loop the products of a k-tile keep their reads between them, which 128 x 128 tiles with float32 outputs gain 8 %
  // by (19264 x 528 -> 536); inlined from `multiply` hipcc moves all reads in front, which narrow tiles gain 3 .. 6 % by.
  constexpr bool SPREAD = WIDE && TM > 64 && KS == 1;
  static_assert(SI <= NW && TM / 32 <= NW, "one exponent, one affine instruction per wave");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv / WN, wn = wv % WN, fr = lane & 15, fq = lane >> 4;
  unsigned* exps = (unsigned*)(smem + 2 * KS * STAGE_BYTES);     // [2][TM + TN]
  float* aff = (float*)(exps + 2 * (TM + TN));                   // [scale | shift][TM], fetched with the first k-tile
  const int nk = p.kb;
  const bool relu = p.flags & EPI_RELU, affine = p.flags & EPI_AFFINE;
  if (affine && wv < TM / 32) {
    const int c = (wv % (TM / 64)) * 64;
    const float* src = wv < TM / 64 ? p.scale : p.shift;
    float* dst = aff + (wv < TM / 64 ? 0 : TM) + c;
    if (src) dma<4>((const uint8_t*)src, 4 * min(co_base + c + lane, p.n - 1), (unsigned char*)dst);
    else dst[lane] = wv < TM / 64 ? 1.f : 0.f;
  }

  unsigned woff[WI], xoff[XI];
#pragma unroll
  for (int i = 0; i < WI; ++i) {
    const int row = wv * (WI * 8) + i * 8 + (lane >> 3);         // rows past n: any valid one, masked at the store
    woff[i] = (unsigned)min(co_base + row, p.n - 1) * p.ldw + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
#pragma unroll
  for (int i = 0; i < XI; ++i) {
    const int row = wv * (XI * 8) + i * 8 + (lane >> 3);
    xoff[i] = (unsigned)min(r_base + row, p.rows - 1) * p.lda + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  const int erow = wv * 64 + lane;
  const uint8_t* ebase = wv * 64 < TM ? p.we : p.ae;
  const unsigned eoff = wv * 64 < TM ? (unsigned)min(co_base + erow, p.n - 1) * p.ldwe
                                     : (unsigned)min(r_base + erow - TM, p.rows - 1) * p.ldae;
  auto stage = [&](int slot, int kt) {
    if ((kt & 3) == 0 && wv < SI) dma<4>(ebase + kt, eoff, (unsigned char*)(exps + ((kt >> 2) & 1) * (TM + TN) + wv * 64));
    unsigned char* wbase = smem + slot * STAGE_BYTES + wv * (WI * 8) * 128;
    unsigned char* xbase = smem + slot * STAGE_BYTES + TM * 128 + wv * (XI * 8) * 128;
#pragma unroll
    for (int i = 0; i < WI; ++i) dma<16>(p.w + kt * 128, woff[i], wbase + i * 1024);
#pragma unroll
    for (int i = 0; i < XI; ++i) dma<16>(p.a + kt * 128, xoff[i], xbase + i * 1024);
  };

  f32x4 acc[MI][NJ];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  int ew[MI], ex[NJ];

  auto multiply = [&](int slot) {
    const unsigned char* wb = smem + slot * STAGE_BYTES;
    const unsigned char* xb = wb + TM * 128;
    if constexpr (WIDE) {
      bf16x8 xh[NJ][4];
#pragma unroll
      for (int n = 0; n < NJ; ++n) fp8_to_bf16(frag(xb, wn * FW + n * 16 + fr, fq), ex[n], xh[n]);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        bf16x8 wh[4];
        fp8_to_bf16(frag(wb, wm * CW + m * 16 + fr, fq), ew[m], wh);
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = mfma_wide(wh, xh[n], acc[m][n]);
      }
    } else {
      i32x8 xf[NJ];
#pragma unroll
      for (int n = 0; n < NJ; ++n) xf[n] = frag(xb, wn * FW + n * 16 + fr, fq);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const i32x8 wf = frag(wb, wm * CW + m * 16 + fr, fq);
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = mfma_fp8<0, 0>(wf, xf[n], acc[m][n], ew[m], ex[n]);
      }
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) ew[m] = (int)((unsigned)ew[m] >> 8);
#pragma unroll
    for (int n = 0; n < NJ; ++n) ex[n] = (int)((unsigned)ex[n] >> 8);
  };
  stage(0, 0);
#pragma unroll
  for (int q = 1; q < KS; ++q)
    if (q < nk) stage(q, q);
  for (int kt = 0; kt < nk; kt += KS) {
    const int cur = (kt / KS) & 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // this wave's share of these k-tiles has landed, then everyone's
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int q = 0; q < KS; ++q)
      if (kt + KS + q < nk) stage((cur ^ 1) * KS + q, kt + KS + q);
    if ((kt & 3) == 0) {
      const unsigned* e = exps + ((kt >> 2) & 1) * (TM + TN);
#pragma unroll
      for (int m = 0; m < MI; ++m) ew[m] = e[wm * CW + m * 16 + fr];
#pragma unroll
      for (int n = 0; n < NJ; ++n) ex[n] = e[TM + wn * FW + n * 16 + fr];
    }
    if constexpr (SPREAD) {
      const unsigned char* wb = smem + cur * STAGE_BYTES;
      const unsigned char* xb = wb + TM * 128;
      bf16x8 xh[NJ][4];
#pragma unroll
      for (int n = 0; n < NJ; ++n) fp8_to_bf16(frag(xb, wn * FW + n * 16 + fr, fq), ex[n], xh[n]);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        bf16x8 wh[4];
        fp8_to_bf16(frag(wb, wm * CW + m * 16 + fr, fq), ew[m], wh);
#pragma unroll
        for (int n = 0; n < NJ; ++n) acc[m][n] = mfma_wide(wh, xh[n], acc[m][n]);
      }
#pragma unroll
      for (int m = 0; m < MI; ++m) ew[m] = (int)((unsigned)ew[m] >> 8);
#pragma unroll
      for (int n = 0; n < NJ; ++n) ex[n] = (int)((unsigned)ex[n] >> 8);
    } else if (kt + KS <= nk) {
#pragma unroll
      for (int q = 0; q < KS; ++q) multiply(cur * KS + q);
    } else {
      for (int q = 0; kt + q < nk; ++q) multiply(cur * KS + q);
    }
  }

  // ---- epilogue: accumulator tile (m, n): lane (fr, fq) holds row wn FW + n 16 + fr, channels wm CW + m 16 + 4 fq + 0..3
  f32x4 sc[MI], sh[MI];
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    sc[m] = (f32x4){1.f, 1.f, 1.f, 1.f};
    sh[m] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  if (affine) {
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      sc[m] = *(const f32x4*)(aff + wm * CW + m * 16 + 4 * fq);
      sh[m] = *(const f32x4*)(aff + TM + wm * CW + m * 16 + 4 * fq);
    }
  }
  if constexpr (WIDE) {                                          // float32 outputs: 16 bytes a lane, 64 in a row
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int r = r_base + wn * FW + n * 16 + fr;
      if (r >= p.rows) continue;
#pragma unroll
      for (int m = 0; m < MI; ++m)
        store_out4(p, r, co_base + wm * CW + m * 16 + 4 * fq, epilogue4(acc[m][n], relu, affine, sc[m], sh[m]));
    }
    return;
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // stage memory becomes the epilogue staging
  constexpr int EPI_STRIDE = CW * 2 + 16, CPR = CW / 8, RPP = 64 / CPR;
  static_assert(NW * 16 * EPI_STRIDE <= 2 * KS * STAGE_BYTES, "epilogue staging fits the stages");
  unsigned char* ep = smem + wv * (16 * EPI_STRIDE);             // this wave's [16 rows][CW channels]
#pragma unroll
  for (int n = 0; n < NJ; ++n) {
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const f32x4 v = epilogue4(acc[m][n], relu, affine, sc[m], sh[m]);
      *(bf16x4*)(ep + fr * EPI_STRIDE + (m * 16 + 4 * fq) * 2) = (bf16x4){(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the staging is the wave's own: no workgroup barrier
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 16 / RPP; ++i) {
      const int f = i * RPP + lane / CPR, ch = lane % CPR;
      const int r = r_base + wn * FW + n * 16 + f, co = co_base + wm * CW + ch * 8;
      const bf16x8 v = *(const bf16x8*)(ep + f * EPI_STRIDE + ch * 16);
      if (r < p.rows && co < p.n) {
        store_bf16x8((bf16*)p.y + (int64_t)r * p.ldy, co, p.n, v);
        if (p.y2 && co >= p.y2_from) store_bf16x8(p.y2 + (int64_t)r * p.ldy2, co, p.n, v);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int TM, int TN, int NW, bool WIDE, int KS = 1>
__global__ __launch_bounds__(64 * NW, NW / 2) void fp8_linear_tile_kernel(LinearArgs p) {
  const int vid = xcd_remap(blockIdx.x, gridDim.x);
  const int co = (vid % p.n_co_tiles) * TM, r = (vid / p.n_co_tiles) * TN;
  // a last tile that is less than half full as half a tile: float32 outputs 3 .. 6 % faster (19264 x 528 -> 536 24.9 -> 23.6 us,
  // 40000 x 700 -> 300 30.2 -> 28.6), bf16 ones between 3 % faster and 8 % slower (the same: 14.0 -> 15.1, 12.5 -> 12.2)
  if (WIDE && TM > 64 && p.n - co <= 64) fp8_tile<64, TN, NW, WIDE, KS>(p, co, r);
  else fp8_tile<TM, TN, NW, WIDE, KS>(p, co, r);
}

template <int TM, int TN, int NW, bool WIDE, int KS = 1>
int launch_tile(LinearArgs p, hipStream_t s) {
  constexpr int smem = linear_tile_lds(TM, TN, KS);
  static OptInMask opted{0};
  if (int rc = lds_opt_in((const void*)fp8_linear_tile_kernel<TM, TN, NW, WIDE, KS>, smem, &opted)) return rc;
  p.n_co_tiles = (int)ceil_div(p.n, TM);
  const int64_t grid = p.n_co_tiles * ceil_div(p.rows, TN);
  hipLaunchKernelGGL((fp8_linear_tile_kernel<TM, TN, NW, WIDE, KS>), dim3((unsigned)grid), dim3(64 * NW), smem, s, p);
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

// ------------------------------------------------------------------------------------------ weights in registers, many rows
// A tile kernel stages both operands of every tile (77 056 x 512 x 512 in 128 x 128 tiles: 315 MB through LDS for 118 MB of
// tensors), and at K <= 512 that DMA bounds it.  Here the WEIGHTS stay: a workgroup owns a slab of 256 channels, each of its
// 8 waves the fragments of 32 of them for the whole of K in registers (16 KB a wave, 256 bytes a lane, at K = 512), and walks a
// run of rows in tiles of 64.  Only rows move, once per slab, through a ring of LDS stages ([64 rows][128 bytes] per block) that runs on across
// tiles; one barrier a tile.  Row i of a wave's 16-channel tile m is channel 8 (i / 4) + 4 m + i % 4 of its 32 (wreg_row), so
// that a lane's 8 results of a row are neighbours: one 16-byte store straight from the accumulators.
// 77 056 x 512 -> 512: 30 us (3.9 TB/s; 128 x 128 tiles 33), of which the rows beyond the first take 0.27 ns each (5.7 TB/s)
// and the launch, the weights' way into registers and the first tile 9 us.  Longer K the same way (4 waves of up to 64
// channels with 512 registers each) was built and dropped: 77 056 x 1536 -> 1536 271 us against 178 of the persistent kernel;
// a lone wave per SIMD does not hide the moves between its two register halves.
struct RowRun { int begin, end, slab; };                          // rows of a workgroup

// Workgroups b and b + 8 (one XCD) take the slabs of one run of rows: all but the first read of a row hit L2.  Runs in units
// of 16 rows, as even as they go; a run's last tile may be partly the next run's (or nobody's) rows.
__device__ __forceinline__ RowRun row_run(int rows, int n_slabs, int runs) {
  const int b = blockIdx.x, xcd = b & 7, jj = b >> 3, run = xcd + 8 * (jj / n_slabs);
  const int units = (rows + 15) >> 4, q = units / runs, rem = units % runs;
  RowRun r;
  r.slab = jj % n_slabs;
  r.begin = 16 * (run * q + min(run, rem));
  r.end = min(rows, r.begin + 16 * (q + (run < rem)));
  return r;
}

template <int KB>
struct Short {
  static constexpr int SLAB = 256, NS = KB == 4 ? 4 : KB == 3 ? 5 : KB == 2 ? 6 : 8, STAGE = KB * 8192;
  static constexpr int LDS = NS * (STAGE + 256);
};

// RAGGED: n is no multiple of 8 (the store of a row's last channels one by one, in the loop of every product, cost 8 %)
template <int KB, bool RAGGED>
__global__ __launch_bounds__(512, 2) void fp8_linear_short_kernel(LinearArgs p, int n_slabs, int runs) {
  typedef Short<KB> C;
  constexpr int NS = C::NS, D = NS - 1, NST = 4;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned* exps = (unsigned*)(smem + NS * C::STAGE);             // [NS][64]
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 15, fq = lane >> 4;
  const RowRun run = row_run(p.rows, n_slabs, runs);
  const int nt = (run.end - run.begin + 63) >> 6;
  if (nt <= 0) return;                                            // (whole workgroups: no barrier is missed)
  const int co = run.slab * C::SLAB + wv * 32;

  const int row = wv * 8 + (lane >> 3);                           // DMA: wave wv fills rows 8 wv .. 8 wv + 7 of each block
  const unsigned coff = ((lane & 7) ^ ((row >> 1) & 7)) << 4;
  auto stage = [&](int t) {
    const int slot = t % NS, base = run.begin + t * 64;
    if (wv == 0) dma<4>(p.ae, (unsigned)min(base + lane, p.rows - 1) * p.ldae, (unsigned char*)(exps + slot * 64));
    const unsigned off = (unsigned)min(base + row, p.rows - 1) * p.lda + coff;
#pragma unroll
    for (int k = 0; k < KB; ++k) dma<16>(p.a + k * 128, off, smem + slot * C::STAGE + k * 8192 + wv * 1024);
  };
#pragma unroll
  for (int t = 0; t < D; ++t)
    if (t < nt) stage(t);

  i32x8 wf[KB][2];
  int ew[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const unsigned wr = (unsigned)min(co + wreg_row(m, fr), p.n - 1);
    ew[m] = *(const int*)(p.we + wr * p.ldwe);
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const uint8_t* src = p.w + wr * p.ldw + k * 128 + fq * 16;
      *(i32x4*)&wf[k][m] = *(const i32x4*)src;
      *((i32x4*)&wf[k][m] + 1) = *(const i32x4*)(src + 64);
    }
  }
  const bool relu = p.flags & EPI_RELU, affine = p.flags & EPI_AFFINE;
  const int cl = co + 8 * fq;
  float sc[8], sh[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) { sc[i] = 1.f; sh[i] = 0.f; }
  if (affine) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (p.scale) sc[i] = p.scale[min(cl + i, p.n - 1)];
      if (p.shift) sh[i] = p.shift[min(cl + i, p.n - 1)];
    }
  }
  // Every tile but a run's last stores all its rows; where this wave's channels are all inside too, D tiles' stores (and KB
  // x (D - 1) rows' DMA, and what goes to a second output) are younger than the DMA that is waited for.
  const bool counted = co + 32 <= p.n;
  for (int t = 0; t < nt; ++t) {
    if (t + D - 1 < nt) {
      if (counted && t >= D) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * KB + D * NST) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * KB) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // tile t is there, tile t - 1 has been read
    if (t + D < nt) stage(t + D);
    const unsigned char* xb = smem + (t % NS) * C::STAGE;
    int ex[4];
    f32x4 acc[2][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      ex[n] = exps[(t % NS) * 64 + n * 16 + fr];
      acc[0][n] = acc[1][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int k = 0; k < KB; ++k) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const i32x8 xf = frag(xb + k * 8192, n * 16 + fr, fq);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if (k == 0) acc[m][n] = mfma_fp8<0, 0>(wf[k][m], xf, acc[m][n], ew[m], ex[n]);
          if (k == 1) acc[m][n] = mfma_fp8<1, 1>(wf[k][m], xf, acc[m][n], ew[m], ex[n]);
          if (k == 2) acc[m][n] = mfma_fp8<2, 2>(wf[k][m], xf, acc[m][n], ew[m], ex[n]);
          if (k == 3) acc[m][n] = mfma_fp8<3, 3>(wf[k][m], xf, acc[m][n], ew[m], ex[n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = acc[i >> 2][n][i & 3];
        if (relu) v[i] = relu_nan(v[i]);
        if (affine) v[i] = fmaf(v[i], sc[i], sh[i]);
      }
      const int r = run.begin + t * 64 + n * 16 + fr;
      if (r < run.end && cl < p.n) {
        bf16x8 o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (bf16)v[i];
        if constexpr (RAGGED) store_bf16x8((bf16*)p.y + (int64_t)r * p.ldy, cl, p.n, o);
        else *(bf16x8_u*)((bf16*)p.y + (int64_t)r * p.ldy + cl) = o;
        if (p.y2 && cl >= p.y2_from) *(bf16x8_u*)(p.y2 + (int64_t)r * p.ldy2 + cl) = o;
      }
    }
  }
}

template <int KB, bool RAGGED>
int launch_short(const LinearArgs& p, int n_cu, hipStream_t s) {
  typedef Short<KB> C;
  static OptInMask opted{0};
  if (int rc = lds_opt_in((const void*)fp8_linear_short_kernel<KB, RAGGED>, C::LDS, &opted)) return rc;
  const int n_slabs = (int)ceil_div(p.n, C::SLAB);
  int runs = n_cu / n_slabs / 8 * 8;
  if (runs < 8) runs = 8;
  hipLaunchKernelGGL((fp8_linear_short_kernel<KB, RAGGED>), dim3((unsigned)(n_slabs * runs)), dim3(512), C::LDS, s, p, n_slabs, runs);
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

int launch_short(const LinearArgs& p, int n_cu, hipStream_t s) {
  const bool ragged = p.n % 8 != 0;
  switch (p.kb) {
    case 1: return ragged ? launch_short<1, true>(p, n_cu, s) : launch_short<1, false>(p, n_cu, s);
    case 2: return ragged ? launch_short<2, true>(p, n_cu, s) : launch_short<2, false>(p, n_cu, s);
    case 3: return ragged ? launch_short<3, true>(p, n_cu, s) : launch_short<3, false>(p, n_cu, s);
    default: return ragged ? launch_short<4, true>(p, n_cu, s) : launch_short<4, false>(p, n_cu, s);
  }
}

// ------------------------------------------------------------------------------------------ persistent 256 x 256 tiles
// One workgroup per CU walks its tiles; the schedule is that of gemm_tiles_persist (conv1x1.hip, two phases a k-tile):
//   phase 1   reads b0, a0, b1 | barrier | a0 x b0, a0 x b1      DMA: weights of the next k-tile
//   phase 2   reads a1         | barrier | a1 x b1, a1 x b0      DMA: activations of the k-tile after next
// on a 128 x 64 wave tile of 16 x 16 x 128 products, operand fragments in registers; the two waves of a SIMD run one
// barrier apart, so one's reads lie under the other's products.  The DMA stream runs on into the next tile under the
// epilogue.  Beside it: exponents, one dword a row and four k-tiles, issued with the weights of the first of the four; the
// affine vectors of the tile's 256 channels, issued with its first k-tile.
// k-tiles alternate between the two stages across tiles too (any number of them), the epilogue is staged through the one
// the last k-tile was in; it needs 4 KiB more than a stage, which lie between the two.
// 77 056 x 1536 -> 1536 178 us (2.04 PF, matrix pipes 43 % busy), 154 112 x 2048 -> 1536 435 (2.23 PF): 1.55 us a k-tile and 6.6 a
// tile.  Left out one at a time (of 178): stores 155, DMA 137, products 141, LDS reads 150; with rows that stay in L2 1.44 us a
// k-tile: what it waits for is rows on their way from memory, one k-tile ahead, and LDS has no room for a third stage.
constexpr int PT = 256, PSTAGE = 2 * PT * 128, PGAP = 4096;
constexpr int PEXPS = 2 * PSTAGE + PGAP, PAFF = PEXPS + 2 * 512 * 4, PERSIST_LDS = PAFF + 2 * PT * 4;

__device__ __forceinline__ void fp8_tiles_persist(const LinearArgs& p, const int first, const int stride, const int rounds) {
  constexpr int MI = 8, NJ = 4, CW = 128, FW = 64, XI = 4;
  constexpr int EPI_STRIDE = CW * 2 + 16, HN = 2, CPR = CW / 8, RPP = 64 / CPR, NSTORE = (NJ / HN) * (16 * HN / RPP);
  static_assert(8 * 16 * HN * EPI_STRIDE <= PSTAGE + PGAP, "epilogue staging");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wv >> 2, wn = wv & 3, srow = lane >> 3, fr = lane & 15, fq = lane >> 4;
  const int nk = p.kb;
  const bool relu = p.flags & EPI_RELU, affine = p.flags & EPI_AFFINE;
  unsigned* exps = (unsigned*)(smem + PEXPS);                    // [2][256 channels | 256 rows]
  float* aff = (float*)(smem + PAFF);                            // [scale 256 | shift 256]
  const float* vec = wv < 4 ? p.scale : p.shift;
  if (affine && !vec) aff[wv * 64 + lane] = wv < 4 ? 1.f : 0.f;  // the missing one, for all tiles

  unsigned woff[4], xoff[4], eoff;
  const uint8_t* ebase = wv < 4 ? p.we : p.ae;                   // exponents: waves 0..3 the channels', 4..7 the rows'
  auto point_w = [&](int co_base, int r_base) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = wv * 32 + i * 8 + srow;                    // rows past the end: any valid one, masked at the store
      woff[i] = (unsigned)min(co_base + row, p.n - 1) * p.ldw + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
    eoff = wv < 4 ? (unsigned)min(co_base + wv * 64 + lane, p.n - 1) * p.ldwe
                  : (unsigned)min(r_base + (wv - 4) * 64 + lane, p.rows - 1) * p.ldae;
  };
  auto point_x = [&](int r_base) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = wv * 32 + i * 8 + srow;
      xoff[i] = (unsigned)min(r_base + row, p.rows - 1) * p.lda + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
    }
  };
  auto stage_at = [&](int buf) { return smem + buf * (PSTAGE + PGAP); };
  auto dma_w = [&](int buf, int kt, int i0) {
    unsigned char* base = stage_at(buf) + wv * 4096;
#pragma unroll
    for (int i = i0; i < i0 + 2; ++i) dma<16>(p.w + kt * 128, woff[i], base + i * 1024);
  };
  auto dma_x = [&](int buf, int kt, int i0) {
    unsigned char* base = stage_at(buf) + PT * 128 + wv * 4096;
#pragma unroll
    for (int i = i0; i < i0 + 2; ++i) dma<16>(p.a + kt * 128, xoff[i], base + i * 1024);
  };
  int gbuf = 0;                                                  // exponent buffer the next group goes to, then is read from
  auto dma_e = [&](int kt) { dma<4>(ebase + kt, eoff, (unsigned char*)(exps + gbuf * 512 + wv * 64)); };
  auto tile_at = [&](int r, int& co_base, int& r_base) {
    const int vid = first + r * stride;
    co_base = (vid % p.n_co_tiles) * PT;
    r_base = (vid / p.n_co_tiles) * PT;
  };
  // fragment addresses within a stage: chunks fq and 4 + fq of row fr, 16 rows further are 2 KiB further
  const int a0 = swz(wm * CW + fr, fq), a1 = swz(wm * CW + fr, 4 + fq);
  const int b0 = PT * 128 + swz(wn * FW + fr, fq), b1 = PT * 128 + swz(wn * FW + fr, 4 + fq);

  f32x4 acc[MI][NJ];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = (f32x4){0.f, 0.f, 0.f, 0.f};
  int ew[MI], ex[NJ];

  int co_base, r_base, par = 0;                                  // par: stage of the tile's first k-tile
  tile_at(0, co_base, r_base);
  point_w(co_base, r_base);
  point_x(r_base);
  dma_e(0);
  dma_w(0, 0, 0);
  dma_w(0, 0, 2);
  dma_x(0, 0, 0);
  dma_x(0, 0, 2);
  bool counted = false;                                          // the wait below may leave NSTORE younger stores in flight
  for (int r = 0; r < rounds; ++r) {
    if (counted) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NSTORE) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the tile's first k-tile is there, every wave out of its epilogue
    if (affine && vec) {                                         // the tile's 256 scales | 256 shifts, 64 a wave
      const int c = min(co_base + (wv & 3) * 64 + lane, p.n - 1);
      dma<4>((const uint8_t*)vec, 4 * c, (unsigned char*)(aff + wv * 64));
    }
    dma_x(par ^ 1, 1, 0);                                        // (not staged earlier: the epilogue went through that stage)
    dma_x(par ^ 1, 1, 2);
    if (wm) asm volatile("s_barrier" ::: "memory");              // group 1 runs one barrier behind
    // the last tile prefetches itself again: the loop stays without conditions, nobody reads what arrives
    int co_next, r_next;
    tile_at(r + 1 < rounds ? r + 1 : r, co_next, r_next);
    for (int kt = 0; kt < nk; ++kt) {
      const int cur = (par + kt) & 1;
      const unsigned char* st = stage_at(cur);
      i32x8 af[4], bl[2], bh[2];
      auto read = [&](int lo, int hi, int t) {
        i32x8 f;
        *(i32x4*)&f = *(const i32x4*)(st + lo + t * 2048);
        *((i32x4*)&f + 1) = *(const i32x4*)(st + hi + t * 2048);
        return f;
      };
      // products of one 64 x 32 quadrant; the empty asm holds them on this side of the barriers (they have no side effects
      // and hipcc sinks them to the next use otherwise)
      auto quad = [&](int m0, i32x8 (&b)[2], int n0) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
            acc[m0 + m][n0 + n] = mfma_fp8<0, 0>(af[m], b[n], acc[m0 + m][n0 + n], ew[m0 + m], ex[n0 + n]);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(acc[m0 + m][n0 + n]));
        __builtin_amdgcn_s_setprio(0);
      };
      auto close_read = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      };
      auto close_mfma = [&](bool last) {
        __builtin_amdgcn_sched_barrier(0);
        if (!last) asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      };
      // ---- phase 1
      const unsigned* e = exps + gbuf * 512;
#pragma unroll
      for (int m = 0; m < MI; ++m) ew[m] = (int)(e[wm * CW + m * 16 + fr] >> (8 * (kt & 3)));
#pragma unroll
      for (int n = 0; n < NJ; ++n) ex[n] = (int)(e[256 + wn * FW + n * 16 + fr] >> (8 * (kt & 3)));
      // (opaque: hipcc would peel the last two k-tiles off into copies of the loop body that spill)
      int left = nk - 1 - kt;
      asm volatile("" : "+s"(left));
      const bool end = left == 0;
      const int kw = end ? 0 : kt + 1;                           // k-tile whose weights are staged now
      if (end) point_w(co_next, r_next);
      if ((kw & 3) == 0) {                                       // its group of exponents
        gbuf ^= 1;
        dma_e(kw);
      }
      dma_w(cur ^ 1, kw, 0);
#pragma unroll
      for (int n = 0; n < 2; ++n) bl[n] = read(b0, b1, n);
#pragma unroll
      for (int m = 0; m < 4; ++m) af[m] = read(a0, a1, m);
      dma_w(cur ^ 1, kw, 2);
#pragma unroll
      for (int n = 0; n < 2; ++n) bh[n] = read(b0, b1, 2 + n);
      close_read();
      quad(0, bl, 0);
      quad(0, bh, 2);
      close_mfma(false);
      // ---- phase 2: activations two k-tiles ahead, into the half of THIS stage that nobody reads any more
      const int kx = left > 1 ? kt + 2 : 0;
      if (left == 1) point_x(r_next);
      if (!end) dma_x(cur, kx, 0);
#pragma unroll
      for (int m = 0; m < 4; ++m) af[m] = read(a0, a1, 4 + m);
      if (!end) {
        dma_x(cur, kx, 2);
        // k-tile kt + 1 has landed (this wave's share) once only the activations issued in this phase are outstanding
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(XI) : "memory");
      }
      close_read();
      quad(4, bh, 2);
      quad(4, bl, 0);
      close_mfma(wm && end);
    }
    // ---- epilogue, staged where the last k-tile was (nobody reads it any more)
    const int co_cur = co_base, r_cur = r_base;
    counted = r_cur + PT <= p.rows && co_cur + PT <= p.n;        // exactly NSTORE stores follow, none masked off
    unsigned char* ep = smem + (((par + nk - 1) & 1) ? PSTAGE : 0) + wv * (16 * HN * EPI_STRIDE);
#pragma unroll
    for (int pass = 0; pass < NJ / HN; ++pass) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int col = m * 16 + 4 * fq;
        f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
        if (affine) {
          sc = *(const f32x4*)(aff + wm * CW + col);
          sh = *(const f32x4*)(aff + PT + wm * CW + col);
        }
#pragma unroll
        for (int nn = 0; nn < HN; ++nn) {
          f32x4 v = acc[m][pass * HN + nn];
          acc[m][pass * HN + nn] = (f32x4){0.f, 0.f, 0.f, 0.f};
          if (relu) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = relu_nan(v[e]);
          }
          if (affine) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(v[e], sc[e], sh[e]);
          }
          const bf16x4 o = {(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
          *(bf16x4*)(ep + (nn * 16 + fr) * EPI_STRIDE + col * 2) = o;
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < 16 * HN / RPP; ++i) {
        const int f = i * RPP + lane / CPR, ch = lane % CPR;
        const int rr = r_cur + wn * FW + pass * (16 * HN) + f, co = co_cur + wm * CW + ch * 8;
        const bf16x8 v = *(const bf16x8*)(ep + f * EPI_STRIDE + ch * 16);
        if (rr < p.rows && co < p.n) store_bf16x8((bf16*)p.y + (int64_t)rr * p.ldy, co, p.n, v);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
    }
    par = (par + nk) & 1;
    co_base = co_next;
    r_base = r_next;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");     // nothing on its way to LDS, staging free: a tail piece may use it
}

// grid = the CU count (a multiple of 8); rounds * grid tiles of 256 x 256, then `tail` tiles cut into 2 (256 x 128), 4 (256 x 64) or
// 16 (64 x 64) pieces, so that a last round that is not full is also shorter (14 tiles behind 7 rounds, 77 056 x 1536 -> 1536: 184.5 us
// in quarters, 182.8 in sixteenths)
__global__ __launch_bounds__(512, 2) void fp8_linear_persist_kernel(LinearArgs p, int rounds, int tail, int split) {
  const int bid = blockIdx.x, nwg = gridDim.x, xcd = bid & 7, seq = bid >> 3, wpx = nwg >> 3;
  // XCD x owns the contiguous tile range [x rounds wpx, (x + 1) rounds wpx); its workgroups take consecutive tiles of it,
  // so tiles that share activation rows run at the same time on one XCD (shared L2)
  if (rounds) fp8_tiles_persist(p, xcd * rounds * wpx + seq, wpx, rounds);
  for (int i = bid; i < tail * split; i += nwg) {
    const int tile = rounds * nwg + i / split, sub = i % split;
    const int co_base = (tile % p.n_co_tiles) * PT, r_tile = (tile / p.n_co_tiles) * PT;
    if (split == 16) {
      const int r = r_tile + (sub >> 2) * 64, co = co_base + (sub & 3) * 64;
      if (r < p.rows && co < p.n) fp8_tile<64, 64, 8, false>(p, co, r);
    } else if (split == 4) {
      if (r_tile + sub * 64 < p.rows) fp8_tile<256, 64, 8, false>(p, co_base, r_tile + sub * 64);
    } else {
      if (r_tile + sub * 128 < p.rows) fp8_tile<256, 128, 8, false>(p, co_base, r_tile + sub * 128);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the piece's epilogue staging has been read
  }
}

int launch_persist(LinearArgs p, int n_cu, hipStream_t s) {
  static OptInMask opted{0};
  if (int rc = lds_opt_in((const void*)fp8_linear_persist_kernel, PERSIST_LDS, &opted)) return rc;
  p.n_co_tiles = (int)ceil_div(p.n, PT);
  const int total = (int)(p.n_co_tiles * ceil_div(p.rows, PT)), rounds = total / n_cu, tail = total - rounds * n_cu;
  hipLaunchKernelGGL(fp8_linear_persist_kernel, dim3(n_cu), dim3(512), PERSIST_LDS, s, p, rounds, tail, tail * 16 <= n_cu ? 16 : tail * 4 <= n_cu ? 4 : 2);
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

int launch_rows(const LinearArgs& p, hipStream_t s) {
  int n_cu = 0;
  if (int rc = device_cu_count(&n_cu)) return rc;
  // Measured, us.  bf16 outputs (direct | 64 x 64 by 8 waves | by 4 | 64 x 128 | 128 x 128 | persist):
  //   1 x 1536 -> 1536       3.5 | 5.7                              600 x 1024 -> 600       8.9 | 5.2 | 5.3 | 5.8 | 7.7
  //   256 x 1536 -> 192      4.1 | 5.8                              1204 x 1536 -> 1536      -  | 8.3 | 7.9 | 8.3 | 10.5
  //   301 x 1536 -> 1536      -  | 5.5 | 6.6 | 7.4 | 10.1           12000 x 2048 -> 300      -  | 16.3 | 14.5 | 13.4 | 16.8
  //   4816 x 1536 -> 1536     -  | 22.7 | 20.7 | 20.5 | 16.1        23001 x 1149 -> 264      -  | 18.0 | 16.0 | 17.0 | 18.9
  //   77056 x 768 -> 768      -  |  -   |  -   |  -   | 61.3 | 65.8   154112 x 128 -> 192    -  | 20.0 | 18.5 | 17.6 | 19.8
  //   77056 x 1152 -> 1152    -  |  -   |  -   |  -   | 125.9 | 118.6   77056 x 1536 -> 1536  -  |  -  |  -   |  -   | 231.9 | 180.8
  //   77056 x 1536 (128 x 128 | persist)  -> 264 59.5 | 67.5, -> 384 59.0 | 64.4, -> 520 85.1 | 97.7, -> 640 87.0 | 100.5,
  //     -> 776 115.6 | 118.9;   77056 x 1152 -> 264 42.3 | 50.4, -> 520 68.5 | 79.0;   77056 x 2048 -> 264 65.8 | 76.0, -> 520 108 | 120
  // float32 outputs (64 x 64 by 8 waves | by 4 | 64 x 128 | 128 x 128 by 4):
  //   301 x 1536 -> 1536     8.0 | 9.3 | 11.3                       13446 x 704 -> 373      16.0 | 14.1 | 15.7 | 17.4
  //   4816 x 1536 -> 1536    38.6 | 33.2 | 32.6 | 27.8              154112 x 128 -> 192     26.8 | 24.1 | 26.6 | 29.4
  // weights in registers | 128 x 128:  77056 x 512 -> 512 29.9 | 33.9, -> 1024 49.4 | 59.1, -> 256 21.3 | 20.2;
  //   77056 x 384 -> 384 24.9 | 22.8;  77056 x 128 -> 512 18.3 | 19.6;  38528 x 512 -> 512 19.8 | 19.3
  // so: direct while its workgroups (each streams its 16 channels' weights once per 16 rows) are at most two a CU; weights in
  // registers for K <= 512 where two slabs or more are three quarters full and walk rows enough to pay for their fetch; the
  // persistent kernel where k-loops are long enough to hide its epilogue and two rounds of tiles or more are there (its rule does
  // not look at how full the last of its 256 channels are: at the widths of the last two lines it costs 3 .. 19 %).  Of the tiles
  // 128 x 128 once they give every CU one, unless the CU with the most of them has more to do than it has with 64 x 128, half the
  // work and a fifth more time for it (channels that end early in a tile, a second round for a few tiles); 64 x 64 below, by 8
  // waves (and in steps of four k-tiles, 128 KiB of LDS, where there are four) while there is no more than one a CU.
  const bool f32 = p.out_f32;
  if (ceil_div(p.n, 16) * ceil_div(p.rows, 16) <= 2ll * n_cu) {
    constexpr int NW = 8;
    const dim3 grid((unsigned)ceil_div(p.n, 16), (unsigned)ceil_div(p.rows, 16));
    if (f32) hipLaunchKernelGGL((fp8_linear_direct_kernel<NW, true>), grid, dim3(64 * NW), 0, s, p);
    else hipLaunchKernelGGL((fp8_linear_direct_kernel<NW, false>), grid, dim3(64 * NW), 0, s, p);
    SUGAR_LAUNCH_CHECK();
    return SUGAR_OK;
  }
  const int64_t slabs = ceil_div(p.n, 256);
  if (!f32 && p.kb <= 4 && n_cu % 8 == 0 && slabs >= 2 && 4ll * p.n >= 3 * 256 * slabs && p.rows * slabs >= 400ll * n_cu)
    return launch_short(p, n_cu, s);
  if (!f32 && !p.y2 && p.kb >= 8 && n_cu % 8 == 0 && ceil_div(p.n, 256) * ceil_div(p.rows, 256) >= 2 * n_cu)
    return launch_persist(p, n_cu, s);
  const int64_t rt = ceil_div(p.rows, 128), half = ceil_div(p.n, 64) * rt, full = ceil_div(p.n, 128) * rt, small = ceil_div(p.n, 64) * ceil_div(p.rows, 64);
  if (full >= n_cu && 5 * ceil_div(full, n_cu) < 3 * ceil_div(half, n_cu))
    return f32 ? launch_tile<128, 128, 4, true>(p, s) : launch_tile<128, 128, 8, false>(p, s);
  if (small <= n_cu && p.kb >= 4) return f32 ? launch_tile<64, 64, 8, true, 4>(p, s) : launch_tile<64, 64, 8, false, 4>(p, s);
  if (small <= n_cu) return f32 ? launch_tile<64, 64, 8, true>(p, s) : launch_tile<64, 64, 8, false>(p, s);
  if (f32) return launch_tile<64, 64, 4, true>(p, s);
  return small <= 2 * n_cu ? launch_tile<64, 64, 4, false>(p, s) : launch_tile<64, 128, 8, false>(p, s);
}

}  // namespace

int launch_fp8_linear(const Fp8Operand& a, int64_t rows, const Fp8Operand& w, int n, int k, const float* scale,
                      const float* shift, int flags, const Fp8Out& out, hipStream_t s) {
  // the kernels' row offsets are 32-bit: weights that do not fit are refused, rows beyond go to a launch of their own
  constexpr int64_t SPAN = (1ll << 32) - 4096;
  const int64_t w_ld = w.ldq > w.lde ? w.ldq : w.lde, a_ld = a.ldq > a.lde ? a.ldq : a.lde;
  SUGAR_CHECK_ARG(w_ld <= SPAN / n, "fp8_linear: weights of %d rows with stride %lld are too large", n, (long long)w_ld);
  SUGAR_CHECK_ARG(a_ld <= SPAN, "fp8_linear: row stride %lld too large", (long long)a_ld);
  SUGAR_CHECK_ARG(!out.y2 || (n % 8 == 0 && out.y2_from % 8 == 0 && out.dtype == SUGAR_BF16), "fp8_linear: second output of ragged chunks");
  const int64_t fit = SPAN / a_ld, per = fit >= 256 ? fit / 256 * 256 : fit;
  const int esz = out.dtype == SUGAR_F32 ? 4 : 2;
  LinearArgs p;
  p.lda = (unsigned)a.ldq; p.ldae = (unsigned)a.lde;
  p.w = w.q; p.we = w.e; p.ldw = (unsigned)w.ldq; p.ldwe = (unsigned)w.lde;
  p.ldy = out.ldy; p.scale = scale; p.shift = shift;
  p.n = n; p.kb = (int)fp8_blocks(k); p.flags = flags; p.out_f32 = out.dtype == SUGAR_F32; p.n_co_tiles = 0;
  p.ldy2 = out.ldy2; p.y2_from = out.y2_from;
  for (int64_t r0 = 0; r0 < rows; r0 += per) {
    p.a = a.q + r0 * a.ldq; p.ae = a.e + r0 * a.lde;
    p.y = (char*)out.y + r0 * out.ldy * esz;
    p.y2 = out.y2 ? (bf16*)out.y2 + r0 * out.ldy2 : nullptr;
    p.rows = (int)(rows - r0 < per ? rows - r0 : per);
    if (int rc = launch_rows(p, s)) return rc;
  }
  return SUGAR_OK;
}

}  // namespace sugar
