// 8-bit operands with one power of two per row and block of 128 columns (gfx950).
//
//   value[r][c] = e4m3(q[r][c]) * 2^(byte[r][c / 128] - 127)
//
// e4m3 is the OCP type (largest 448, NaN 0x7f / 0xff, no infinities), the byte an E8M0 exponent (255 = NaN).  Rows of q
// are padded with zeros to a multiple of 128 columns (a block that ends inside a tile multiplies zeros), rows of exponent
// bytes to a multiple of 4 (the matrix kernels fetch four blocks' bytes as one dword).
// A power of two rather than amax / 448 itself: the matrix instructions of gfx950 apply it inside the product
// (v_mfma_scale_*_f8f6f4), accumulators stay in registers over the whole of K, and scaling is exact, so the only rounding
// of the format is the one to e4m3.  The price is at most one binade of e4m3's range at the bottom, none of its precision.
#pragma once
#include "common.h"

namespace sugar {

constexpr int FP8_BLOCK = 128;

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;

static inline int64_t fp8_blocks(int64_t cols) { return ceil_div(cols, FP8_BLOCK); }
static inline int64_t fp8_ldq(int64_t cols) { return fp8_blocks(cols) * FP8_BLOCK; }
static inline int64_t fp8_lds(int64_t cols) { return round_up(fp8_blocks(cols), 4); }

// Exponent byte of a block from the bits of its largest finite magnitude: the smallest e >= -127 with amax <= 448 2^e,
// 448 = 1.75 2^8.  amax = m 2^E (1 <= m < 2) needs e = E - 8, one more when m > 1.75, i.e. when the mantissa field is
// over 0x600000: adding 0x1fffff to the bits carries into the exponent exactly then.  (f32 subnormals and zero: 0.)
__device__ __forceinline__ int fp8_exponent(unsigned amax_bits) {
  const int e = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
  return e < 0 ? 0 : e;
}

// 2^(127 - byte): the factor that takes a value into e4m3's range (byte 0 .. 247 here: 2^127 .. 2^-120, all normal)
__device__ __forceinline__ float fp8_inverse(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }

// Largest of 16 neighbouring lanes (a DPP row), in every one of them.  Bits of non-negative floats order as integers.
__device__ __forceinline__ unsigned row16_max(unsigned v) {
  auto step = [](unsigned x, unsigned y) { return x > y ? x : y; };
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));    // quad_perm [1,0,3,2]
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));    // quad_perm [2,3,0,1]
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));   // row_half_mirror
  v = step(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));   // row_mirror
  return v;
}

// Magnitude bits of a finite value, 0 for infinities and NaN (they take no part in a block's exponent).
__device__ __forceinline__ unsigned fp8_finite_bits(float v) {
  const unsigned u = __float_as_uint(v) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// Eight values of one block -> eight e4m3 bytes, to nearest with ties to even.  |v| inv <= 448 by the choice of the
// exponent, so nothing saturates; infinities and NaN become NaN (a bad frame shows, it does not turn into a large value).
__device__ __forceinline__ u32x2 fp8_pack8(const float* v, float inv) {
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    t[i] = (__float_as_uint(v[i]) & 0x7fffffffu) < 0x7f800000u ? v[i] * inv : __uint_as_float(0x7fc00000u);
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[4], t[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[6], t[7], hi, true);
  return (u32x2){(unsigned)lo, (unsigned)hi};
}

// 16 bytes at the alignment of their elements: rows of odd widths and strides begin anywhere, and the hardware's global
// loads and stores take any address (one instruction either way).
typedef bf16x8 bf16x8_u __attribute__((aligned(2)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));
template <typename T, int N>
struct Run { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };

// What a lane read at element n - 8 of a row of n >= 8 elements, because its own 8 from element c on reach past the end ->
// those 8, zeros from n on.  The distance is 8 - n % 8 for the one lane with the row's last elements (a shift that is the same
// in the whole launch, in three steps); lanes wholly behind the row hold zeros.  (Read one by one,
// those elements made 48 000 x 511 bf16 rows cost 64 us instead of 42 in the join with two norms, 23 instead of 16 in the
// quantiser; 512 columns: 33 and 16.)
__device__ __forceinline__ void ragged_end(float* v, int c, int n) {
  if (c + 8 <= n) return;
  const int s = 8 - (n & 7);
  if (s & 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i + 1 < 8 ? v[i + 1] : 0.f;
  }
  if (s & 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i + 2 < 8 ? v[i + 2] : 0.f;
  }
  if (s & 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i + 4 < 8 ? v[i + 4] : 0.f;
  }
  if (c >= n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
}

// Eight consecutive elements from channel c on; those past `n` (the row's channels) read as 0.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int c, int n, float* v) {
  if (n < 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < n ? to_f32(p[c + i]) : 0.f;
    return;
  }
  p += min(c, n - 8);
  if constexpr (sizeof(T) == 2) {
    const bf16x8 t = *(const bf16x8_u*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  } else {
    const f32x4 t0 = *(const f32x4_u*)p, t1 = *(const f32x4_u*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = t0[i]; v[4 + i] = t1[i]; }
  }
  ragged_end(v, c, n);
}

// The first m (1 .. 7) of eight: runs of 4, 2 and 1.
template <typename T>
__device__ __forceinline__ void store_first(T* __restrict__ p, int m, typename Run<T, 8>::type t) {
  if (m & 4) *(typename Run<T, 4>::type*)p = t.lo;
  const typename Run<T, 4>::type r = m & 4 ? t.hi : t.lo;             // what is left: at most 3
  if (m & 2) *(typename Run<T, 2>::type*)(p + (m & 4)) = r.lo;
  const T last = m & 2 ? r.z : r.x;
  if (m & 1) p[m & 6] = last;
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int c, int n, const float* v) {
  typename Run<T, 8>::type t;
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(v[i]);
  if (c + 8 <= n) {
    if constexpr (sizeof(T) == 2) {
      *(bf16x8_u*)(p + c) = t;
    } else {
      *(f32x4_u*)(p + c) = t.lo;
      *(f32x4_u*)(p + c + 4) = t.hi;
    }
  } else if (c < n) {
    store_first(p + c, n & 7, t);
  }
}

// eight bf16 of a row of n channels from channel c on, as they lie in memory
__device__ __forceinline__ void store_bf16x8(bf16* __restrict__ y, int c, int n, bf16x8 o) {
  if (c + 8 <= n) *(bf16x8_u*)(y + c) = o;
  else if (c < n) store_first(y + c, n & 7, o);
}

// ---- products -------------------------------------------------------------------------------------------------------
// v_mfma_scale_f32_16x16x128_f8f6f4: lane (fr, fq) = (lane & 15, lane >> 4) holds 32 of the 128 K values of row fr of either
// operand (which 32 does not matter as long as both operands agree and the block has one scale); result: lane holds
// D[4 fq + i][fr].  Byte OP of the exponent dwords is applied.
// Precision, probed on the device: the products of 8 consecutive K values are aligned to the largest of them and cut off
// 2^-13 below its leading bit, then summed with the accumulator in f32.  On random operands (K = 1536) the result is
// 1.5e-5 off (2-norm), a hundredth of the 1.7e-3 that rounding it to bf16 costs: bf16 outputs take this instruction.
template <int OPA, int OPB>
__device__ __forceinline__ f32x4 mfma_fp8(i32x8 a, i32x8 b, f32x4 c, int ea, int eb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, OPA, ea, OPB, eb);
}

// float32 outputs: the same block as four 16-bit products on the values converted to bf16, block scale included (the
// conversion instruction applies a power of two; an e4m3 value times one is a bf16 value from bf16's smallest subnormal,
// 2^-133, up to 2^128, byte 255 gives NaN), whose sums are good to f32 (4.6e-8 off on the same operands), at half the rate.  Conversions are one
// instruction per two values and lie under the other wave's products.
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
__device__ __forceinline__ void fp8_to_bf16(i32x8 q, int byte, bf16x8 (&h)[4]) {
  const float sc = __uint_as_float((unsigned)(byte & 255) << 23);
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s + d], sc, false);
      const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[2 * s + d], sc, true);
      h[s][4 * d] = lo[0]; h[s][4 * d + 1] = lo[1]; h[s][4 * d + 2] = hi[0]; h[s][4 * d + 3] = hi[1];
    }
}
__device__ __forceinline__ f32x4 mfma_wide(const bf16x8 (&a)[4], const bf16x8 (&b)[4], f32x4 c) {
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[s], b[s], c, 0, 0, 0);
  return c;
}

struct Fp8Operand {        // [rows][ld] e4m3, [rows][lds] exponent bytes
  const uint8_t* q = nullptr;
  const uint8_t* e = nullptr;
  int64_t ldq = 0, lde = 0;
};

struct Fp8Weight {         // device-resident [n][k] operand of a layer (packed by pack_fp8)
  uint8_t* q = nullptr;
  uint8_t* e = nullptr;
  int n = 0, k = 0;
  Fp8Operand operand() const {
    Fp8Operand o;
    o.q = q; o.e = e; o.ldq = fp8_ldq(k); o.lde = fp8_lds(k);
    return o;
  }
};
// Reference-layout 1x1 conv weight [cout][cin] (host f32) -> [n][k] with out_map / in_map as pack_conv; the same values
// sugar_fp8_quant gives
int pack_fp8(Fp8Weight* w, const float* h_w, int cout, int cin, int n, const int* out_map, int k, const int* in_map);
void free_fp8(Fp8Weight* w);

struct Fp8Out {
  void* y = nullptr;       // [rows][ldy] dtype
  int64_t ldy = 0;
  int dtype = SUGAR_BF16;
  void* y2 = nullptr;      // optional second store (bf16 only) of columns >= y2_from, a multiple of 8 (pointer has NO column offset)
  int64_t ldy2 = 0;
  int y2_from = 0;
};

// y[r][o] = epilogue(sum_k a[r][k] w[o][k]), flags EPI_RELU | EPI_AFFINE (scale / shift [n], applied after the ReLU; one of them
// may be nullptr: 1 / 0)
int launch_fp8_linear(const Fp8Operand& a, int64_t rows, const Fp8Operand& w, int n, int k, const float* scale,
                      const float* shift, int flags, const Fp8Out& out, hipStream_t s);

// y [rows][ldy] dtype <- the first `cols` values of an operand (its exponent rows may begin anywhere)
int launch_fp8_dequant(const Fp8Operand& a, int64_t rows, int cols, void* d_y, int64_t ldy, int dtype, hipStream_t s);

// pad_exponents: also the padding bytes behind a row's last block (not where the 8-bit output is a column slice: the bytes
// behind it belong to the next slice or row)
int launch_block_join(const SugarBlockJoin& j, bool pad_exponents, hipStream_t s);

}  // namespace sugar
