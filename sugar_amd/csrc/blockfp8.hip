// Quantisation to 8-bit operands with block scales, their reading back, and the matrix product of two of them (gfx950).
// The format is described in blockfp8.h.
#include "blockfp8.h"

namespace sugar {

namespace {

// ------------------------------------------------------------------------------------------ quantise / read back
// 16 lanes own one block of 128 columns, 8 values each: the block's largest magnitude is four DPP steps, no LDS.
template <typename T>
__global__ __launch_bounds__(256) void fp8_quant_kernel(const T* __restrict__ x, int64_t ldx, int64_t items, int cols,
                                                        int blocks, int vec, uint8_t* __restrict__ q, int64_t ldq,
                                                        uint8_t* __restrict__ e, int64_t lde) {
  const int l16 = threadIdx.x & 15;
  const int64_t stride = (int64_t)gridDim.x * 16;
  for (int64_t it = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); it < items; it += stride) {
    const int64_t row = it / blocks;
    const int kb = (int)(it - row * blocks), c = kb * FP8_BLOCK + l16 * 8;
    float v[8];
    load8(x + row * ldx, c, cols, vec, v);
    unsigned big = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { const unsigned u = fp8_finite_bits(v[i]); big = u > big ? u : big; }
    const int byte = fp8_exponent(row16_max(big));
    *(u32x2*)(q + row * ldq + c) = fp8_pack8(v, fp8_inverse(byte));
    if (l16 == 0) e[row * lde + kb] = (uint8_t)byte;
    else if (kb == blocks - 1 && kb + l16 < ((blocks + 3) & ~3)) e[row * lde + kb + l16] = 127;   // padding bytes
  }
}

template <typename T>
__global__ __launch_bounds__(256) void fp8_dequant_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                          const uint8_t* __restrict__ e, int64_t lde, int64_t items, int cols,
                                                          int blocks, int vec, T* __restrict__ y, int64_t ldy) {
  const int l16 = threadIdx.x & 15;
  const int64_t stride = (int64_t)gridDim.x * 16;
  for (int64_t it = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); it < items; it += stride) {
    const int64_t row = it / blocks;
    const int kb = (int)(it - row * blocks), c = kb * FP8_BLOCK + l16 * 8;
    const u32x2 t = *(const u32x2*)(q + row * ldq + c);
    const int byte = e[row * lde + kb];
    float v[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)t[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)t[h], true);
      v[4 * h] = a[0]; v[4 * h + 1] = a[1]; v[4 * h + 2] = b[0]; v[4 * h + 3] = b[1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = byte == 255 ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(v[i], byte - 127);
    store8(y + row * ldy, c, cols, vec, v);
  }
}

// ------------------------------------------------------------------------------------------ matrix product
struct LinearArgs {
  const uint8_t *a, *ae, *w, *we;
  int64_t lda, ldae, ldw, ldwe, ldy;
  void* y;
  const float *scale, *shift;
  int rows, n, kb, flags, out_f32, vec;
};

// Epilogue of four consecutive channels of one row.
__device__ __forceinline__ void store_out4(const LinearArgs& p, int64_t r, int co, f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (co + i >= p.n) break;
    float t = v[i];
    if (p.flags & EPI_RELU) t = t < 0.f ? 0.f : t;            // (NaN stays NaN)
    if (p.flags & EPI_AFFINE) t = fmaf(t, p.scale[co + i], p.shift[co + i]);
    if (p.out_f32) ((float*)p.y)[r * p.ldy + co + i] = t;
    else ((bf16*)p.y)[r * p.ldy + co + i] = (bf16)t;
  }
}

// Operands straight from memory into the matrix instruction's registers, K dealt out over the workgroup's waves and their
// sums joined in LDS in wave order: 16 channels x 16 NT rows a workgroup.  WIDE: 16-bit products (float32 outputs).
template <int NT, int NW, bool WIDE>
__global__ __launch_bounds__(64 * NW) void fp8_linear_direct_kernel(LinearArgs p) {
  __shared__ f32x4 part[NW][NT][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, fr = lane & 15, fq = lane >> 4;
  const int co = blockIdx.x * 16, r0 = blockIdx.y * (16 * NT);
  const int wrow = min(co + fr, p.n - 1);
  const uint8_t* wp = p.w + (int64_t)wrow * p.ldw + fq * 32;
  const uint8_t* wep = p.we + (int64_t)wrow * p.ldwe;
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int kb = wv; kb < p.kb; kb += NW) {
    i32x8 wf;
    *(i32x4*)&wf = *(const i32x4*)(wp + kb * 128);
    *((i32x4*)&wf + 1) = *(const i32x4*)(wp + kb * 128 + 16);
    bf16x8 wh[4];
    int ew[4];
    if constexpr (WIDE) {
      fp8_to_bf16(wf, wh);
#pragma unroll
      for (int i = 0; i < 4; ++i) ew[i] = p.we[(int64_t)min(co + 4 * fq + i, p.n - 1) * p.ldwe + kb];
    } else {
      ew[0] = wep[kb];
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int ar = min(r0 + t * 16 + fr, p.rows - 1);
      const uint8_t* ap = p.a + (int64_t)ar * p.lda + kb * 128 + fq * 32;
      i32x8 af;
      *(i32x4*)&af = *(const i32x4*)ap;
      *((i32x4*)&af + 1) = *(const i32x4*)(ap + 16);
      const int ea = p.ae[(int64_t)ar * p.ldae + kb];
      if constexpr (WIDE) {
        bf16x8 ah[4];
        fp8_to_bf16(af, ah);
        const f32x4 z = mfma_wide(wh, ah);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = add_scaled(acc[t][i], z[i], ea, ew[i]);
      } else {
        acc[t] = mfma_fp8<0, 0>(wf, af, acc[t], ew[0], ea);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) part[wv][t][lane] = acc[t];
  __syncthreads();
  for (int t = wv; t < NT; t += NW) {
    f32x4 v = part[0][t][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) v += part[k][t][lane];
    const int r = r0 + t * 16 + fr;
    if (r < p.rows) store_out4(p, r, co + 4 * fq, v);
  }
}

}  // namespace

static int check_operand(const char* what, const uint8_t* q, int64_t ldq, const uint8_t* e, int64_t lde, int64_t cols) {
  SUGAR_CHECK_ARG(q && e, "%s: null pointer", what);
  SUGAR_CHECK_ARG(((uintptr_t)q & 15) == 0 && ldq % 16 == 0 && ldq >= fp8_ldq(cols),
                  "%s: rows of 8-bit values must be 16-byte aligned and hold %lld columns (stride %lld)", what,
                  (long long)fp8_ldq(cols), (long long)ldq);
  SUGAR_CHECK_ARG(((uintptr_t)e & 3) == 0 && lde % 4 == 0 && lde >= fp8_lds(cols),
                  "%s: rows of exponent bytes must be 4-byte aligned and hold %lld bytes (stride %lld)", what,
                  (long long)fp8_lds(cols), (long long)lde);
  return SUGAR_OK;
}

int launch_fp8_linear(const Fp8Operand& a, int64_t rows, const Fp8Operand& w, int n, int k, const float* scale,
                      const float* shift, int flags, void* d_y, int64_t ldy, int dtype, hipStream_t s) {
  LinearArgs p;
  p.a = a.q; p.ae = a.e; p.lda = a.ldq; p.ldae = a.lde;
  p.w = w.q; p.we = w.e; p.ldw = w.ldq; p.ldwe = w.lde;
  p.y = d_y; p.ldy = ldy; p.scale = scale; p.shift = shift;
  p.rows = (int)rows; p.n = n; p.kb = (int)fp8_blocks(k); p.flags = flags; p.out_f32 = dtype == SUGAR_F32;
  p.vec = 0;
  constexpr int NT = 2, NW = 4;
  const dim3 grid((unsigned)ceil_div(n, 16), (unsigned)ceil_div(rows, 16 * NT));
  if (p.out_f32) hipLaunchKernelGGL((fp8_linear_direct_kernel<NT, NW, true>), grid, dim3(64 * NW), 0, s, p);
  else hipLaunchKernelGGL((fp8_linear_direct_kernel<NT, NW, false>), grid, dim3(64 * NW), 0, s, p);
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

}  // namespace sugar

using namespace sugar;

extern "C" {

int sugar_fp8_quant(const void* d_x, int64_t ldx, int dtype, int64_t rows, int cols, uint8_t* d_q, int64_t ldq,
                    uint8_t* d_e, int64_t lde, void* stream) {
  SUGAR_CHECK_ARG(dtype == SUGAR_F32 || dtype == SUGAR_BF16, "fp8_quant: bad dtype %d", dtype);
  SUGAR_CHECK_ARG(rows >= 0 && cols > 0 && d_x && ldx >= cols, "fp8_quant: bad arguments");
  if (int rc = check_operand("fp8_quant", d_q, ldq, d_e, lde, cols)) return rc;
  if (rows == 0) return SUGAR_OK;
  const int esz = dtype == SUGAR_F32 ? 4 : 2;
  SUGAR_CHECK_ARG((uintptr_t)d_x % esz == 0, "fp8_quant: unaligned input");
  const int64_t items = rows * fp8_blocks(cols);
  const int vec = rows_vec(d_x, ldx, cols, esz);
  const unsigned grid = (unsigned)(ceil_div(items, 16) < 65536 ? ceil_div(items, 16) : 65536);
  if (dtype == SUGAR_F32)
    hipLaunchKernelGGL(fp8_quant_kernel<float>, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const float*)d_x, ldx, items,
                       cols, (int)fp8_blocks(cols), vec, d_q, ldq, d_e, lde);
  else
    hipLaunchKernelGGL(fp8_quant_kernel<bf16>, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const bf16*)d_x, ldx, items,
                       cols, (int)fp8_blocks(cols), vec, d_q, ldq, d_e, lde);
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

int sugar_fp8_dequant(const uint8_t* d_q, int64_t ldq, const uint8_t* d_e, int64_t lde, int64_t rows, int cols, void* d_y,
                      int64_t ldy, int dtype, void* stream) {
  SUGAR_CHECK_ARG(dtype == SUGAR_F32 || dtype == SUGAR_BF16, "fp8_dequant: bad dtype %d", dtype);
  SUGAR_CHECK_ARG(rows >= 0 && cols > 0 && d_y && ldy >= cols, "fp8_dequant: bad arguments");
  if (int rc = check_operand("fp8_dequant", d_q, ldq, d_e, lde, cols)) return rc;
  if (rows == 0) return SUGAR_OK;
  const int esz = dtype == SUGAR_F32 ? 4 : 2;
  SUGAR_CHECK_ARG((uintptr_t)d_y % esz == 0, "fp8_dequant: unaligned output");
  const int64_t items = rows * fp8_blocks(cols);
  const int vec = rows_vec(d_y, ldy, cols, esz);
  const unsigned grid = (unsigned)(ceil_div(items, 16) < 65536 ? ceil_div(items, 16) : 65536);
  if (dtype == SUGAR_F32)
    hipLaunchKernelGGL(fp8_dequant_kernel<float>, dim3(grid), dim3(256), 0, (hipStream_t)stream, d_q, ldq, d_e, lde, items,
                       cols, (int)fp8_blocks(cols), vec, (float*)d_y, ldy);
  else
    hipLaunchKernelGGL(fp8_dequant_kernel<bf16>, dim3(grid), dim3(256), 0, (hipStream_t)stream, d_q, ldq, d_e, lde, items,
                       cols, (int)fp8_blocks(cols), vec, (bf16*)d_y, ldy);
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

int sugar_fp8_linear(const uint8_t* d_a, int64_t lda, const uint8_t* d_ae, int64_t ldae, int64_t rows, const uint8_t* d_w,
                     int64_t ldw, const uint8_t* d_we, int64_t ldwe, int n, int k, const float* d_scale,
                     const float* d_shift, int flags, void* d_y, int64_t ldy, int dtype, void* stream) {
  SUGAR_CHECK_ARG(dtype == SUGAR_F32 || dtype == SUGAR_BF16, "fp8_linear: bad dtype %d", dtype);
  SUGAR_CHECK_ARG(rows >= 0 && rows < (1ll << 27) && n > 0 && n < (1 << 24) && k > 0 && k < (1 << 24),
                  "fp8_linear: sizes out of range (rows %lld, n %d, k %d)", (long long)rows, n, k);
  SUGAR_CHECK_ARG((flags & ~(EPI_RELU | EPI_AFFINE)) == 0, "fp8_linear: unknown flags %d", flags);
  SUGAR_CHECK_ARG(!(flags & EPI_AFFINE) || (d_scale && d_shift), "fp8_linear: affine epilogue without scale / shift");
  SUGAR_CHECK_ARG(d_y && ldy >= n && (uintptr_t)d_y % (dtype == SUGAR_F32 ? 4 : 2) == 0, "fp8_linear: bad output");
  SUGAR_CHECK_ARG((uintptr_t)d_scale % 4 == 0 && (uintptr_t)d_shift % 4 == 0, "fp8_linear: unaligned scale / shift");
  int rc;
  if ((rc = check_operand("fp8_linear: left operand", d_a, lda, d_ae, ldae, k)) ||
      (rc = check_operand("fp8_linear: weights", d_w, ldw, d_we, ldwe, k)))
    return rc;
  if (rows == 0) return SUGAR_OK;
  Fp8Operand a, w;
  a.q = d_a; a.ldq = lda; a.e = d_ae; a.lde = ldae;
  w.q = d_w; w.ldq = ldw; w.e = d_we; w.lde = ldwe;
  return launch_fp8_linear(a, rows, w, n, k, d_scale, d_shift, flags, d_y, ldy, dtype, (hipStream_t)stream);
}

}  // extern "C"
