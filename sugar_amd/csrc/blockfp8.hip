// Quantisation to 8-bit operands with block scales, their reading back, and the C entries (gfx950; product: fp8_gemm.hip).
// The format is described in blockfp8.h.
#include <math.h>

#include <new>
#include <vector>

#include "blockfp8.h"

namespace sugar {

namespace {

// ------------------------------------------------------------------------------------------ quantise / read back
// 16 lanes own one block of 128 columns, 8 values each: the block's largest magnitude is four DPP steps, no LDS; a workgroup
// takes 16 neighbouring blocks (a row's, then the next row's).  Bound by memory, by the latency of one load and one store
// where the call is small.  Measured, bf16 / float32: 77 056 x 1536 66 us (5.4 TB/s) / 101 (5.8), back 63 (5.7) / 102 (5.8);
// 24 373 x 536 10.6 / 12.0, back 8.2 / 12.8; 301 x 512 3.0 / 2.6, back 2.6 / 2.5.  (Two blocks a group: 66.5 / 104, back
// 63 / 120; four: 72 / 110, back 62 / 127.)
template <typename T>
__global__ __launch_bounds__(256) void fp8_quant_kernel(const T* __restrict__ x, int64_t ldx, unsigned items, int cols,
                                                        unsigned blocks, uint8_t* __restrict__ q, int64_t ldq,
                                                        uint8_t* __restrict__ e, int64_t lde) {
  const int l16 = threadIdx.x & 15;
  const unsigned it = blockIdx.x * 16 + (threadIdx.x >> 4), row = it / blocks;
  if (it >= items) return;
  const int kb = (int)(it - row * blocks), c = kb * FP8_BLOCK + l16 * 8;
  float v[8];
  load8(x + row * ldx, c, cols, v);
  unsigned big = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) { const unsigned u = fp8_finite_bits(v[i]); big = u > big ? u : big; }
  const int byte = fp8_exponent(row16_max(big));
  *(u32x2*)(q + row * ldq + c) = fp8_pack8(v, fp8_inverse(byte));
  if (l16 == 0) e[row * lde + kb] = (uint8_t)byte;
  else if (kb == (int)blocks - 1 && kb + l16 < (((int)blocks + 3) & ~3)) e[row * lde + kb + l16] = 127;   // padding bytes
}

template <typename T>
__global__ __launch_bounds__(256) void fp8_dequant_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                          const uint8_t* __restrict__ e, int64_t lde, unsigned items, int cols,
                                                          unsigned blocks, T* __restrict__ y, int64_t ldy) {
  const int l16 = threadIdx.x & 15;
  const unsigned it = blockIdx.x * 16 + (threadIdx.x >> 4), row = it / blocks;
  if (it >= items) return;
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
  store8(y + row * ldy, c, cols, v);
}

// Calls f(first row, blocks) for runs of rows whose blocks times 16 threads fit a launch and count in 32 bits (dividing 64-bit
// numbers took 4 of 70 us at 77 056 x 1536, 1.5 of 12 at 24 373 x 536).
template <typename F>
int by_rows(int64_t rows, int cols, F f) {
  const int64_t per = (1ll << 27) / fp8_blocks(cols);
  for (int64_t r0 = 0; r0 < rows; r0 += per) {
    f(r0, (unsigned)((rows - r0 < per ? rows - r0 : per) * fp8_blocks(cols)));
    SUGAR_LAUNCH_CHECK();
  }
  return SUGAR_OK;
}

template <typename T>
int launch_quant(const T* x, int64_t ldx, int64_t rows, int cols, uint8_t* q, int64_t ldq, uint8_t* e, int64_t lde, hipStream_t s) {
  return by_rows(rows, cols, [&](int64_t r0, unsigned items) {
    hipLaunchKernelGGL(fp8_quant_kernel<T>, dim3((unsigned)ceil_div(items, 16)), dim3(256), 0, s, x + r0 * ldx, ldx, items, cols,
                       (unsigned)fp8_blocks(cols), q + r0 * ldq, ldq, e + r0 * lde, lde);
  });
}

template <typename T>
int launch_dequant(const Fp8Operand& a, int64_t rows, int cols, T* y, int64_t ldy, hipStream_t s) {
  return by_rows(rows, cols, [&](int64_t r0, unsigned items) {
    hipLaunchKernelGGL(fp8_dequant_kernel<T>, dim3((unsigned)ceil_div(items, 16)), dim3(256), 0, s, a.q + r0 * a.ldq, a.ldq,
                       a.e + r0 * a.lde, a.lde, items, cols, (unsigned)fp8_blocks(cols), y + r0 * ldy, ldy);
  });
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

int launch_fp8_dequant(const Fp8Operand& a, int64_t rows, int cols, void* d_y, int64_t ldy, int dtype, hipStream_t s) {
  return dtype == SUGAR_F32 ? launch_dequant(a, rows, cols, (float*)d_y, ldy, s) : launch_dequant(a, rows, cols, (bf16*)d_y, ldy, s);
}

// host side of the quantiser: e4m3 bits of |v| <= 448, to nearest with ties to even (rint in the default mode)
static uint8_t host_e4m3(float v) {
  const uint8_t sign = signbit(v) ? 0x80 : 0;
  const float a = fabsf(v);
  if (!(a <= 448.f)) return sign | 0x7f;
  if (a < 0.015625f) return sign | (uint8_t)rintf(a * 512.f);         // subnormals; 8 is the smallest normal's bits
  int e;
  (void)frexpf(a, &e);                                                // a = m 2^e, m in [0.5, 1)
  int m = (int)rintf(ldexpf(a, 4 - e));                               // [8, 16]
  if (m == 16) { m = 8; ++e; }
  return sign | (uint8_t)((e + 6) << 3 | (m - 8));
}

static int pack_fp8_rows(Fp8Weight* w, const float* h_w, int cout, int cin, int n, const int* out_map, int k, const int* in_map) {
  const int64_t ldq = fp8_ldq(k), lde = fp8_lds(k);
  std::vector<uint8_t> q((size_t)(n * ldq), 0), e((size_t)(n * lde), 127);
  std::vector<float> row((size_t)ldq);
  for (int64_t r = 0; r < n; ++r)                                     // rows no channel maps to: zeros, exponent as of zeros
    for (int64_t b = 0; b < fp8_blocks(k); ++b) e[(size_t)(r * lde + b)] = 0;
  for (int o = 0; o < cout; ++o) {
    const int64_t r = out_map ? out_map[o] : o;
    row.assign(row.size(), 0.f);
    for (int i = 0; i < cin; ++i) row[(size_t)(in_map ? in_map[i] : i)] = h_w[(size_t)o * cin + i];
    for (int64_t b = 0; b < fp8_blocks(k); ++b) {
      uint32_t big = 0;
      for (int c = 0; c < FP8_BLOCK; ++c) {
        uint32_t u;
        memcpy(&u, &row[(size_t)(b * FP8_BLOCK + c)], 4);
        u &= 0x7fffffffu;
        if (u < 0x7f800000u && u > big) big = u;
      }
      int byte = (int)((big + 0x1fffffu) >> 23) - 8;                  // fp8_exponent
      if (byte < 0) byte = 0;
      e[(size_t)(r * lde + b)] = (uint8_t)byte;
      for (int c = 0; c < FP8_BLOCK; ++c)
        q[(size_t)(r * ldq + b * FP8_BLOCK + c)] = host_e4m3(ldexpf(row[(size_t)(b * FP8_BLOCK + c)], 127 - byte));
    }
  }
  int rc;
  if ((rc = dev_alloc(&w->q, q.size())) || (rc = dev_upload(w->q, q.data(), q.size())) || (rc = dev_alloc(&w->e, e.size())) ||
      (rc = dev_upload(w->e, e.data(), e.size())))
    return rc;
  w->n = n;
  w->k = k;
  return SUGAR_OK;
}

int pack_fp8(Fp8Weight* w, const float* h_w, int cout, int cin, int n, const int* out_map, int k, const int* in_map) {
  try {                                                               // (called below a C entry)
    return pack_fp8_rows(w, h_w, cout, cin, n, out_map, k, in_map);
  } catch (const std::bad_alloc&) {
    set_error("pack_fp8: host alloc");
    return SUGAR_ENOMEM;
  }
}

void free_fp8(Fp8Weight* w) {
  dev_free(w->q);
  dev_free(w->e);
  *w = Fp8Weight();
}

}  // namespace sugar

using namespace sugar;

extern "C" {

int sugar_fp8_quant(const void* d_x, int64_t ldx, int dtype, int64_t rows, int cols, uint8_t* d_q, int64_t ldq,
                    uint8_t* d_e, int64_t lde, void* stream) {
  SUGAR_CHECK_ARG(dtype == SUGAR_F32 || dtype == SUGAR_BF16, "fp8_quant: bad dtype %d", dtype);
  SUGAR_CHECK_ARG(rows >= 0 && cols > 0 && cols < (1 << 24) && d_x && ldx >= cols, "fp8_quant: bad arguments");
  if (int rc = check_operand("fp8_quant", d_q, ldq, d_e, lde, cols)) return rc;
  if (rows == 0) return SUGAR_OK;
  const int esz = dtype == SUGAR_F32 ? 4 : 2;
  SUGAR_CHECK_ARG((uintptr_t)d_x % esz == 0, "fp8_quant: unaligned input");
  return dtype == SUGAR_F32 ? launch_quant((const float*)d_x, ldx, rows, cols, d_q, ldq, d_e, lde, (hipStream_t)stream)
                            : launch_quant((const bf16*)d_x, ldx, rows, cols, d_q, ldq, d_e, lde, (hipStream_t)stream);
}

int sugar_fp8_dequant(const uint8_t* d_q, int64_t ldq, const uint8_t* d_e, int64_t lde, int64_t rows, int cols, void* d_y,
                      int64_t ldy, int dtype, void* stream) {
  SUGAR_CHECK_ARG(dtype == SUGAR_F32 || dtype == SUGAR_BF16, "fp8_dequant: bad dtype %d", dtype);
  SUGAR_CHECK_ARG(rows >= 0 && cols > 0 && cols < (1 << 24) && d_y && ldy >= cols, "fp8_dequant: bad arguments");
  if (int rc = check_operand("fp8_dequant", d_q, ldq, d_e, lde, cols)) return rc;
  if (rows == 0) return SUGAR_OK;
  const int esz = dtype == SUGAR_F32 ? 4 : 2;
  SUGAR_CHECK_ARG((uintptr_t)d_y % esz == 0, "fp8_dequant: unaligned output");
  Fp8Operand a;
  a.q = d_q; a.ldq = ldq; a.e = d_e; a.lde = lde;
  return launch_fp8_dequant(a, rows, cols, d_y, ldy, dtype, (hipStream_t)stream);
}

int sugar_fp8_linear(const uint8_t* d_a, int64_t lda, const uint8_t* d_ae, int64_t ldae, int64_t rows, const uint8_t* d_w,
                     int64_t ldw, const uint8_t* d_we, int64_t ldwe, int n, int k, const float* d_scale,
                     const float* d_shift, int flags, void* d_y, int64_t ldy, int dtype, void* stream) {
  SUGAR_CHECK_ARG(dtype == SUGAR_F32 || dtype == SUGAR_BF16, "fp8_linear: bad dtype %d", dtype);
  SUGAR_CHECK_ARG(rows >= 0 && rows < (1ll << 27) && n > 0 && n < (1 << 24) && k > 0 && k < (1 << 24),
                  "fp8_linear: sizes out of range (rows %lld, n %d, k %d)", (long long)rows, n, k);
  SUGAR_CHECK_ARG((flags & ~(EPI_RELU | EPI_AFFINE)) == 0, "fp8_linear: unknown flags %d", flags);
  SUGAR_CHECK_ARG(!(flags & EPI_AFFINE) || d_scale || d_shift, "fp8_linear: affine epilogue without scale and shift");
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
  Fp8Out out;
  out.y = d_y; out.ldy = ldy; out.dtype = dtype;
  return launch_fp8_linear(a, rows, w, n, k, d_scale, d_shift, flags, out, (hipStream_t)stream);
}

}  // extern "C"
