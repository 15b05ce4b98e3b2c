// What the kernels with products of microscaled rows share: the matrix instruction and its operands, and the epilogue.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 elements and their scales, one scale byte per row
// and 32 columns. Lane l supplies row l % 16 of either operand. With g = l / 16 it holds, of 4-bit elements, columns
// 32 g .. 32 g + 31 (16 bytes), of 8-bit ones 16 g .. and 64 + 16 g .. (two times 16 bytes), and in both cases the
// scale of columns 32 g .. 32 g + 31. The result gives lane l column l % 16 and rows 4 g + i. W is the first operand, so
// a lane holds 4 channels of one row of X per product, and the channel that each of W's 16 rows stands for is free:
// channel(tile t, g, i) = (t / G) * 16 G + g * 4 G + (t % G) * 4 + i gives a lane 4 G consecutive channels over G tiles, so
// its stores are whole 16-byte pieces.
#pragma once
#include "mx.h"

namespace {
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kOOR = 0x80000000u;  // past every buffer below (at most 2^28 bytes), also with a step's offset added: reads as zeros

enum { OUT_16 = 0, OUT_F32 = 1, OUT_MX8 = 2, OUT_MX4 = 3 };

struct LinArgs {
  const uint8_t *x, *xs, *w, *ws;  // codes and scales
  const void *bias, *res;          // res: of out's type
  void* out;
  uint8_t* outs;
  i64 N;
  int K, O, bias_dt, act, f16;
  int xrow, wrow, srow, osrow;  // bytes of a row: X's and W's codes, their scales, out's scales
  int tiles_n, tiles_o, per, per_rest, band;
};

__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

template <int XB>
struct XFrag {  // 16 rows of X by 128 columns, this lane's part
  mx_u32x4 q[XB / 4];
};
template <>
struct XFrag<4> {
  mx_u32x4 q[1];
};
// The scales are byte IW of sw and byte IX of sx
template <int XB, int IW, int IX>
__device__ __forceinline__ f32x4 mfma(mx_u32x4 w, const XFrag<XB>& x, f32x4 c, int sw, int sx) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  if constexpr (XB == 8) {
    const i32x8 b = {(int)x.q[0][0], (int)x.q[0][1], (int)x.q[0][2], (int)x.q[0][3],
                     (int)x.q[1][0], (int)x.q[1][1], (int)x.q[1][2], (int)x.q[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, IW, sw, IX, sx);
  } else {
    const i32x8 b = {(int)x.q[0][0], (int)x.q[0][1], (int)x.q[0][2], (int)x.q[0][3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, IW, sw, IX, sx);
  }
}
// Of four e4m3 elements those of magnitude 4 and more (codes from 0x48), zeros for the others: a byte's low seven bits plus
// 0x38 carry into bit 7, which a byte permute spreads (selectors 8 and 9 repeat bits 15 and 31 of its second operand,
// 10 and 11 those of its first).
__device__ __forceinline__ uint32_t e4m3_large(uint32_t v) {
  const uint32_t t = (v & 0x7f7f7f7fu) + 0x38383838u;
  return v & __builtin_amdgcn_perm(t, t << 8, 0x0b090a08u);
}
// Epilogue of NV consecutive channels o .. of row n in v: bias, activation, residual (its words in r), store. Lanes l, l + 16, l + 32, l + 48
// hold neighbouring runs of one row; ok is the same for all lanes of a block of 32 channels. Runs of 64 bytes of a row are
// stored past the caches, which keep the operands ([8209, 2080] by [4128, 2080] 102 -> 94 us, [11467, 2048] by [512, 2048]
// 20.9 -> 20.2; fp32 level). Runs of 32 bytes are not (tail of 391007 rows, 128 channels: 193 us, 203 past the caches), nor are
// microscaled rows, which the next product reads at once (tail of 11467 rows, 512 channels: 63 us, 69 past the caches).
template <int OUT, int NV>
__device__ __forceinline__ void finish(const LinArgs& a, i64 n, int o, float (&v)[NV], const float (&bias)[NV],
                                       const uint32_t (&r)[4], bool ok) {
#pragma unroll
  for (int j = 0; j < NV; j++) v[j] += bias[j];
  if (a.act == ACT_SILU) {
#pragma unroll
    for (int j = 0; j < NV; j++) v[j] = silu(v[j]);
  }
  if constexpr (OUT == OUT_F32) {
    static_assert(NV == 4, "one 16-byte piece");
    if (!ok) return;
    if (a.res) {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += __uint_as_float(r[j]);
    }
    *(f32x4*)((float*)a.out + n * a.O + o) = f32x4{v[0], v[1], v[2], v[3]};
  } else if constexpr (OUT == OUT_16) {
    static_assert(NV == 8 || NV == 4, "one 16-byte piece, or half of one");
    if (!ok) return;
    uint32_t q[NV / 2];
    if (a.res) {
#pragma unroll
      for (int j = 0; j < NV / 2; j++) {
        v[2 * j] += a.f16 ? mx_lo<true>(r[j]) : mx_lo<false>(r[j]);
        v[2 * j + 1] += a.f16 ? mx_hi<true>(r[j]) : mx_hi<false>(r[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV / 2; j++) q[j] = a.f16 ? mx_pack2<true>(v[2 * j], v[2 * j + 1]) : mx_pack2<false>(v[2 * j], v[2 * j + 1]);
    uint32_t* y = (uint32_t*)((uint16_t*)a.out + n * a.O + o);
    if constexpr (NV == 8) __builtin_nontemporal_store(*(mx_u32x4*)q, (mx_u32x4*)y);
    else *(mx_u32x2*)y = *(mx_u32x2*)q;
  } else {
    static_assert(NV == 16 || NV == 8, "a half or a quarter of a block");
    constexpr int FMT = OUT == OUT_MX8 ? MX_E4M3 : MX_E2M1;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; j += 8) top = max(top, mx_top8(*(float(*)[8])&v[j]));
    top = mx_max_across16(top);
    if constexpr (NV == 8) top = mx_max_across32(top);
    const uint32_t byte = mx_scale_byte<FMT>(top);
    const float inv = mx_inverse(byte);
    const mx_u32x2 p = mx_encode8<FMT>(*(float(*)[8])&v[0], inv);
    if constexpr (NV == 16) {
      const mx_u32x2 q = mx_encode8<FMT>(*(float(*)[8])&v[8], inv);
      if (!ok) return;
      if constexpr (FMT == MX_E4M3) *(mx_u32x4*)((uint8_t*)a.out + n * a.O + o) = mx_u32x4{p[0], p[1], q[0], q[1]};
      else *(mx_u32x2*)((uint8_t*)a.out + (n * a.O + o) / 2) = mx_u32x2{p[0], q[0]};
    } else {
      if (!ok) return;
      if constexpr (FMT == MX_E4M3) *(mx_u32x2*)((uint8_t*)a.out + n * a.O + o) = p;
      else *(uint32_t*)((uint8_t*)a.out + (n * a.O + o) / 2) = p[0];
    }
    if (o % 32 == 0) {
      uint8_t* s = a.outs + n * a.osrow;
      s[o / 32] = (uint8_t)byte;
      if (o / 32 + 1 == a.O / 32)
        for (int k = a.O / 32; k < a.osrow; k++) s[k] = 0;
    }
  }
}

// The residual's words for NV channels of 16 or 32 bits
template <int OUT, int NV>
__device__ __forceinline__ void load_residual(const LinArgs& a, i64 n, int o, bool ok, uint32_t (&r)[4]) {
  if constexpr (OUT == OUT_16 && NV == 4) {
    const mx_u32x2 q = ok ? *(const mx_u32x2*)((const uint16_t*)a.res + n * a.O + o) : mx_u32x2{};
    r[0] = q[0];
    r[1] = q[1];
  } else if constexpr (OUT == OUT_16 || OUT == OUT_F32) {
    const mx_u32x4 q = ok ? *(const mx_u32x4*)((const char*)a.res + (n * a.O + o) * (OUT == OUT_16 ? 2 : 4)) : mx_u32x4{};
#pragma unroll
    for (int j = 0; j < 4; j++) r[j] = q[j];
  }
}

// The parts of e4m3 elements that SPLIT products take apart (see k_mx_gemm)
__device__ __forceinline__ void split(XFrag<8>& x, XFrag<8>& large) {  // x keeps the small ones
#pragma unroll
  for (int k = 0; k < 2; k++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      large.q[k][j] = e4m3_large(x.q[k][j]);
      x.q[k][j] ^= large.q[k][j];
    }
}
}  // namespace
