// The join of a block with its residual stream (gfx950): the norm behind the block, the gate, the residual sum, the norm
// in front of the next block and, where that block multiplies in 8 bits, its operand -- one pass over the rows.
//
//   v = post(u);  s = residual + alpha * gate * v;  stream = s  (or residual + s);  z = pre(s)
//
// The SE-Res2 stack of DynamicTDNN.forward (sugar/models/dynamictdnn.py:98-100, 657-660) is the case without row norms:
// gate = the squeeze-excite scale of the row's utterance, out = y * gate + S, S += out.
// Everything between the loads and the stores is f32 in registers: a wave (several for wide rows, 16 or 32 lanes for narrow
// ones) holds its row, so a norm's mean and its sum of squares about that mean are two exact passes over registers, not over memory, and z
// comes from the unrounded s.  Bound: HBM (u and residual in, stream and z out).  Measured, bf16: 77 056 x 512 with two rms
// norms 59 us (5.3 TB/s), dense with 8-bit output 48 (5.7); 48 611 x 1024, layer / layer, float32 stream 115 (5.2); one row 3.5.
#include <type_traits>

#include "blockfp8.h"

namespace sugar {

namespace {

enum { NORM_NONE = SUGAR_NORM_NONE, NORM_AFFINE = SUGAR_NORM_AFFINE, NORM_RMS = SUGAR_NORM_RMS, NORM_LAYER = SUGAR_NORM_LAYER };

struct JoinArgs {
  SugarBlockJoin j;
  int run;                   // consecutive rows a wave (WPR = 1) or workgroup takes
  int e_bytes;               // exponent bytes of a row that are written (the blocks, and padding where the row is an operand of its own)
};

// Sum over LPR neighbouring lanes, the same in every one of them: within rows of 16 by DPP, across them by the row / half
// swaps (of a value with itself: the two results are the two halves, each in all lanes).
template <int LPR>
__device__ __forceinline__ float lane_total(float v) {
  v += dpp_row_f32<0xB1>(v);
  v += dpp_row_f32<0x4E>(v);
  v += dpp_row_f32<0x141>(v);
  v += dpp_row_f32<0x140>(v);
  if constexpr (LPR > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if constexpr (LPR > 32) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return v;
}

// Sum over the row.  Several waves a row exchange theirs through one half of `red` and the next total's through the other: a half
// is written again only behind the barrier of the total between.
template <int WPR, int LPR>
__device__ __forceinline__ float row_total(float v, float* red, int wv, int& half) {
  v = lane_total<LPR>(v);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) red[half + wv] = v;
    __syncthreads();
    v = red[half];
#pragma unroll
    for (int i = 1; i < WPR; ++i) v += red[half + i];
    half ^= 16;
  }
  return v;
}

// Eight channels as they lie in memory, fetched without a branch and without touching the values, so that every load of a
// row is on its way before the first is used: 16-byte loads, a lane that reaches past the row's end reads the row's last 8
// (ragged_end puts them right).  WIDE: rows of 8 channels and more; shorter ones are read one by one altogether.
template <typename T, bool WIDE>
struct Raw8 {
  typedef typename std::conditional<sizeof(T) == 2, bf16x8_u, f32x4_u>::type Chunk;
  Chunk q[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* __restrict__ p, int c, int n) {
    if constexpr (WIDE) {
      const Chunk* s = (const Chunk*)(p + min(c, n - 8));
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = s[i];
    }
  }
  __device__ __forceinline__ void get(const T* __restrict__ p, float* v, int c, int n) const {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(q[i * sizeof(T) / 16][i % (16 / sizeof(T))]);
      ragged_end(v, c, n);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < n ? to_f32(p[c + i]) : 0.f;
    }
  }
};

// weight and bias of a norm for this lane's channels: 1 and 0 where there is no vector, 0 past the row (so that what a
// norm leaves there is 0)
template <bool WIDE>
struct NormVec {
  float w[8], b[8];
  __device__ __forceinline__ void load(const float* __restrict__ pw, const float* __restrict__ pb, int c, int C) {
#pragma unroll
    for (int i = 0; i < 8; ++i) { w[i] = c + i < C ? 1.f : 0.f; b[i] = 0.f; }
    Raw8<float, WIDE> t;
    if (pw) { t.load(pw, c, C); t.get(pw, w, c, C); }
    if (pb) { t.load(pb, c, C); t.get(pb, b, c, C); }
  }
};

// x <- norm(x) over the row's C channels; lanes past the row hold zeros before and after.
template <int WPR, int LPR, bool WIDE>
__device__ __forceinline__ void row_norm(float (&x)[8], int kind, const NormVec<WIDE>& p, float eps, int C, float inv_c, int c,
                                         float* red, int wv, int& half) {
  if (kind == NORM_NONE) return;
  float mean = 0.f, mul = 1.f;
  if (kind == NORM_LAYER) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += x[i];
    mean = row_total<WPR, LPR>(t, red, wv, half) * inv_c;
  }
  if (kind != NORM_AFFINE) {
    float t = 0.f;
    if (C & 7) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = c + i < C ? x[i] - mean : 0.f;
        t = fmaf(d, d, t);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = x[i] - mean;
        t = fmaf(d, d, t);
      }
      t = c < C ? t : 0.f;
    }
    mul = 1.0f / sqrtf(fmaf(row_total<WPR, LPR>(t, red, wv, half), inv_c, eps));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf((x[i] - mean) * mul, p.w[i], p.b[i]);
}

// 8 channels a lane; LPR lanes of a wave a row, or (LPR = 64) WPR waves, which are the workgroup where they are more than one.
// Each group of lanes that holds a row takes a run of consecutive rows.
template <typename TU, typename TS, int WPR, int LPR, bool WIDE, bool NORMS>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void block_join_kernel(JoinArgs a) {
  __shared__ float red[WPR > 1 ? 32 : 1];
  int half = 0;
  const SugarBlockJoin& j = a.j;
  const int lane = threadIdx.x & (LPR - 1), wv = threadIdx.x >> 6;
  const int C = j.cols;
  const int c = (WPR > 1 ? wv * 512 : 0) + lane * 8;            // this lane's first channel
  const float inv_c = 1.0f / (float)C;
  constexpr int RPB = WPR > 1 ? 1 : 256 / LPR;                 // runs of rows a workgroup takes
  const int64_t first = ((int64_t)blockIdx.x * RPB + (WPR > 1 ? 0 : LPR == 64 ? __builtin_amdgcn_readfirstlane(wv) : (int)threadIdx.x / LPR)) * a.run;
  const int64_t last = first + a.run < j.rows ? first + a.run : j.rows;
  if (first >= last) return;
  int b = 0, b_end = 0, begin = 0;
  if (j.d_row_off) {                                           // last utterance that begins at or before the first row: LPR-ary search
    for (int n = j.n_utts; n > 1;) {
      const int step = (n + LPR - 1) / LPR, i = lane * step;
      uint64_t le = __ballot(i < n && j.d_row_off[b + i] <= first);
      if (LPR < 64) le = le >> (threadIdx.x & 63 & ~(LPR - 1)) & ((1ull << (LPR & 63)) - 1);
      const int k = max((int)__popcll(le) - 1, 0) * step;
      b += k;
      n = min(step, n - k);
    }
    b_end = j.d_row_off[b + 1];
    begin = j.d_row_off[0];
  }
  NormVec<WIDE> post, pre;                                     // in registers over the rows
  if (NORMS && j.post_kind) post.load(j.d_post_w, j.d_post_b, c, C);
  if (NORMS && j.pre_kind) pre.load(j.d_pre_w, j.d_pre_b, c, C);
  // the next row is fetched before this one is worked on; a gate per channel once, one per utterance when the utterance changes
  Raw8<TU, WIDE> nu, ng;
  Raw8<TS, WIDE> ns;
  auto fetch = [&](int64_t r) {
    nu.load((const TU*)j.d_u + r * j.ldu, c, C);
    ns.load((const TS*)j.d_residual + r * j.ldr, c, C);
    if (j.gate_kind == SUGAR_GATE_ROW) ng.load((const TU*)j.d_gate + r * j.ldg, c, C);
  };
  float g[8];
  auto fetch_gate = [&](const float* gp) {
    Raw8<float, WIDE> t;
    t.load(gp, c, C);
    t.get(gp, g, c, C);
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = 1.f;
  if (j.gate_kind == SUGAR_GATE_CHANNEL) fetch_gate((const float*)j.d_gate);
  int gate_of = -1;
  fetch(first);
  for (int64_t r = first; r < last; ++r) {
    const Raw8<TU, WIDE> ru = nu, rg = ng;
    const Raw8<TS, WIDE> rs = ns;
    if (r + 1 < last) fetch(r + 1);
    if (j.d_row_off) {
      while (r >= b_end && b + 1 < j.n_utts) { ++b; b_end = j.d_row_off[b + 1]; }
      if (r >= b_end || r < begin) continue;                   // a row of no utterance: left as it is
      if (j.gate_kind == SUGAR_GATE_UTTERANCE && b != gate_of) {
        fetch_gate((const float*)j.d_gate + b * j.ldg);
        gate_of = b;
      }
    }
    const TU* up = (const TU*)j.d_u + r * j.ldu;
    const TS* rp = (const TS*)j.d_residual + r * j.ldr;
    float v[8], s[8];
    ru.get(up, v, c, C);
    if (NORMS) row_norm<WPR, LPR, WIDE>(v, j.post_kind, post, j.post_eps, C, inv_c, c, red, wv, half);
    if (j.gate_kind == SUGAR_GATE_ROW) rg.get((const TU*)j.d_gate + r * j.ldg, g, c, C);
    rs.get(rp, s, c, C);
    float st[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float res = s[i];
      s[i] = fmaf(j.alpha * g[i], v[i], res);
      st[i] = j.dense ? res + s[i] : s[i];
    }
    if (j.d_stream) store8((TS*)j.d_stream + r * j.lds, c, C, st);
    if (!j.d_z && !j.d_q) continue;
    if (NORMS) row_norm<WPR, LPR, WIDE>(s, j.pre_kind, pre, j.pre_eps, C, inv_c, c, red, wv, half);
    if (j.d_z) {
      if (j.z_dtype == SUGAR_F32) store8((float*)j.d_z + r * j.ldz, c, C, s);
      else store8((bf16*)j.d_z + r * j.ldz, c, C, s);
    }
    if (j.d_q) {
      if (c + 8 > C) {                                         // the operand's padding columns are 0, whatever a norm of a bad row left there
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = c + i < C ? s[i] : 0.f;
      }
      unsigned big = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) { const unsigned u = fp8_finite_bits(s[i]); big = u > big ? u : big; }
      const int byte = fp8_exponent(row16_max(big)), kb = c / FP8_BLOCK, blocks = (C + FP8_BLOCK - 1) / FP8_BLOCK;
      if (kb < blocks) {
        *(u32x2*)(j.d_q + r * j.ldq + c) = fp8_pack8(s, fp8_inverse(byte));
        const int l16 = lane & 15;
        if (l16 == 0) j.d_e[r * j.lde + kb] = (uint8_t)byte;
        else if (kb == blocks - 1 && kb + l16 < a.e_bytes) j.d_e[r * j.lde + kb + l16] = 127;   // padding bytes
      }
    }
  }
}

template <typename TU, typename TS, int WPR, int LPR>
int launch_join(JoinArgs a, int n_cu, hipStream_t s) {
  constexpr int threads = WPR > 1 ? 64 * WPR : 256, RPB = WPR > 1 ? 1 : 256 / LPR;
  // Rows a group of lanes takes one after the other: they share the fetch of the norm vectors, the search of the utterance and its
  // gate, and each is fetched under the one before.  Many rows, us for runs of 1 / 2 / 4 / 8 (inputs from memory): 77 056 x 512 two rms
  // norms, gate per utterance 88 / 69 / 65 / 64; 48 611 x 1024 without norms 79 / 72 / 76 / 80, layer / layer into a 32-bit stream 134 /
  // 115 / 115 / 119 (3: 114); 30 000 x 1536 rms / rms 99 / 81 / 77 / 77; 40 000 x 2048 rms / rms 180 / 143 / 130 / 126.  Fewer rows: as many
  // waves as the chip holds at once, about three a SIMD, rather than a second round of them: 14 857 x 616 30 / 26 / 24 / 22, 12 000 x
  // 300 14.9 / 13.3 / 12.9 / 17.4, 35 438 x 120 12.2 / 11.9 / 12.1 / 15.9 (3: 10.4), 8000 x 200 6.5 / 6.7 / 9.0 / 13.8, 1480 x 592 5.2 / 5.5 / 7.6 /
  // 11.7, 301 x 512 4.0 / 4.8 / 6.8.
  const bool norms = a.j.post_kind || a.j.pre_kind;
  const int64_t most = !norms ? 2 : sizeof(TS) == 4 && LPR == 64 ? 3 : WPR > 3 ? 8 : 4;
  const int64_t waves = ceil_div(a.j.rows * WPR * LPR, 64), share = (waves + 6 * n_cu) / (12 * n_cu);
  const int64_t least = ceil_div(a.j.rows, RPB * ((1ll << 32) / threads - 1));            // a launch has fewer than 2^32 threads
  a.run = (int)(share >= most ? (most > least ? most : least) : share > 1 ? share : 1);
  const dim3 grid((unsigned)ceil_div(a.j.rows, (int64_t)a.run * RPB));
  if (a.j.cols < 8) {
    if constexpr (LPR == 16) hipLaunchKernelGGL((block_join_kernel<TU, TS, WPR, LPR, false, true>), grid, dim3(threads), 0, s, a);
  } else if (norms) {
    hipLaunchKernelGGL((block_join_kernel<TU, TS, WPR, LPR, true, true>), grid, dim3(threads), 0, s, a);
  } else {
    hipLaunchKernelGGL((block_join_kernel<TU, TS, WPR, LPR, true, false>), grid, dim3(threads), 0, s, a);
  }
  SUGAR_LAUNCH_CHECK();
  return SUGAR_OK;
}

// As many lanes as a row of 8 channels a lane fills: 30 000 x 1536 by three waves a row 74 us, by four 92; 1480 x 592 by two 5.4, by
// four 8.1; 22 180 x 11 by 16 lanes 8.7, by a wave 19.2.
template <typename TU, typename TS>
int launch_join_t(const JoinArgs& a, hipStream_t s) {
  int n_cu = 0;
  if (int rc = device_cu_count(&n_cu)) return rc;
  const int C = a.j.cols;
  if (C <= 128) return launch_join<TU, TS, 1, 16>(a, n_cu, s);
  if (C <= 256) return launch_join<TU, TS, 1, 32>(a, n_cu, s);
  if (C <= 512) return launch_join<TU, TS, 1, 64>(a, n_cu, s);
  if (C <= 1024) return launch_join<TU, TS, 2, 64>(a, n_cu, s);
  if (C <= 1536) return launch_join<TU, TS, 3, 64>(a, n_cu, s);
  if (C <= 2048) return launch_join<TU, TS, 4, 64>(a, n_cu, s);
  if (C <= 4096) return launch_join<TU, TS, 8, 64>(a, n_cu, s);
  return launch_join<TU, TS, 16, 64>(a, n_cu, s);
}

bool norm_ok(int kind) { return kind == NORM_NONE || kind == NORM_AFFINE || kind == NORM_RMS || kind == NORM_LAYER; }

}  // namespace

int launch_block_join(const SugarBlockJoin& j, bool pad_exponents, hipStream_t s) {
  JoinArgs a;
  a.j = j;
  a.e_bytes = (int)(pad_exponents ? fp8_lds(j.cols) : fp8_blocks(j.cols));
  if (j.u_dtype == SUGAR_F32) return launch_join_t<float, float>(a, s);
  return j.stream_dtype == SUGAR_F32 ? launch_join_t<bf16, float>(a, s) : launch_join_t<bf16, bf16>(a, s);
}

}  // namespace sugar

using namespace sugar;

extern "C" int sugar_block_join(const SugarBlockJoin* h, void* stream) {
  SUGAR_CHECK_ARG(h, "block_join: null descriptor");
  const SugarBlockJoin& j = *h;
  SUGAR_CHECK_ARG(j.rows >= 0 && j.rows < (1ll << 33) && j.cols > 0 && j.cols <= SUGAR_JOIN_MAX_COLS,
                  "block_join: rows %lld, columns %d out of range (1..%d)", (long long)j.rows, j.cols, SUGAR_JOIN_MAX_COLS);
  SUGAR_CHECK_ARG((j.u_dtype == SUGAR_F32 || j.u_dtype == SUGAR_BF16) && (j.stream_dtype == SUGAR_F32 || j.stream_dtype == SUGAR_BF16) &&
                      (j.z_dtype == SUGAR_F32 || j.z_dtype == SUGAR_BF16),
                  "block_join: bad dtype");
  SUGAR_CHECK_ARG(!(j.u_dtype == SUGAR_F32 && j.stream_dtype == SUGAR_BF16), "block_join: a 32-bit block output needs a 32-bit stream");
  SUGAR_CHECK_ARG(j.d_u && j.d_residual && (j.d_stream || j.d_z || j.d_q), "block_join: null pointer");
  SUGAR_CHECK_ARG(norm_ok(j.post_kind) && norm_ok(j.pre_kind), "block_join: unknown norm");
  SUGAR_CHECK_ARG(j.post_eps >= 0.f && j.pre_eps >= 0.f, "block_join: negative eps");
  SUGAR_CHECK_ARG(j.gate_kind >= SUGAR_GATE_NONE && j.gate_kind <= SUGAR_GATE_ROW && (j.gate_kind == SUGAR_GATE_NONE) == !j.d_gate,
                  "block_join: gate kind %d does not fit its pointer", j.gate_kind);
  SUGAR_CHECK_ARG(j.gate_kind != SUGAR_GATE_UTTERANCE || j.d_row_off, "block_join: a gate per utterance needs row offsets");
  SUGAR_CHECK_ARG(!j.d_row_off || j.n_utts > 0, "block_join: row offsets of no utterance");
  SUGAR_CHECK_ARG(j.ldu >= j.cols && j.ldr >= j.cols && (!j.d_stream || j.lds >= j.cols) && (!j.d_z || j.ldz >= j.cols) &&
                      (j.gate_kind < SUGAR_GATE_UTTERANCE || j.ldg >= j.cols),
                  "block_join: a row stride is shorter than the row");
  const uintptr_t eu = j.u_dtype == SUGAR_F32 ? 3 : 1, es = j.stream_dtype == SUGAR_F32 ? 3 : 1, ez = j.z_dtype == SUGAR_F32 ? 3 : 1;
  SUGAR_CHECK_ARG(!((uintptr_t)j.d_u & eu) && !((uintptr_t)j.d_residual & es) && !((uintptr_t)j.d_stream & es) &&
                      !((uintptr_t)j.d_z & ez) && !((uintptr_t)j.d_gate & (j.gate_kind == SUGAR_GATE_ROW ? eu : 3)) &&
                      !((uintptr_t)j.d_post_w & 3) && !((uintptr_t)j.d_post_b & 3) && !((uintptr_t)j.d_pre_w & 3) &&
                      !((uintptr_t)j.d_pre_b & 3) && !((uintptr_t)j.d_row_off & 3),
                  "block_join: a pointer is not aligned to its type");
  if (j.d_q)
    SUGAR_CHECK_ARG(j.d_e && !((uintptr_t)j.d_q & 15) && j.ldq % 16 == 0 && j.ldq >= fp8_ldq(j.cols) && j.lde >= fp8_lds(j.cols),
                    "block_join: bad 8-bit output");
  if (j.rows == 0) return SUGAR_OK;
  return launch_block_join(j, true, (hipStream_t)stream);
}
