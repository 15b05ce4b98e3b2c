// Microscaled rows on the device: 32 consecutive values share the scale 2^(b - 127) of one byte b (255: the block holds
// an infinity or a NaN and reads as NaN); the elements are e4m3 (8 bits, largest 448, no infinity) or e2m1 (4 bits,
// largest 6, two per byte, the even one in the low half). Row-major codes; a row's scale bytes are padded to a multiple
// of 16, so that the 16 of 512 columns are one aligned load.
//
// Scale: the least power of two s for which amax / s, rounded to the element's precision as if its grid went on, is
// at most the largest element: amax / s <= 464 for e4m3 (464, halfway to 480, ties to 448), < 7 for e2m1 (7 ties to
// 8). Nothing is then off by more than a rounding. With s = 2^(floor(log2 amax) - emax) the top of the range is cut
// instead; with amax / s <= 448 or 6 the e2m1 blocks lose a step that they need not. Relative 2-norm error on normal
// values, on their SiLU, and with 1% of them ten times as large: e2m1 0.112, 0.124, 0.153 (floor 0.115, 0.128, 0.155;
// never cut 0.115, 0.134, 0.166), e4m3 0.0266 for all three (floor 0.029, 0.032, 0.035).
#pragma once
#include <hip/hip_runtime.h>

#include "spconv.h"

typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));

// The scale byte of a block whose largest magnitude has the bits `top` (sign cleared). One integer addition rounds the
// mantissa up over the border: 0x680000 is 464 / 256 - 1, 0x600000 is 7 / 4 - 1 in 23 bits.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const int b = (int)((top + (FMT == MX_E4M3 ? 0x17ffffu : 0x200000u)) >> 23) - (FMT == MX_E4M3 ? 8 : 2);
  return top >= 0x7f800000u ? 255u : (uint32_t)max(b, 0);
}
// 1 / scale, exact: bytes 0 ... 253 give 2^127 ... 2^-126. A block that reads as NaN gets zeros for elements.
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// 8 values -> their elements, each v * inv rounded to nearest, halves to even: 8 bytes (e4m3) or 4 (e2m1, in [0]). Where
// inv is 0 (a block with an infinity or NaN) the elements are zeros, whatever the conversion makes of the values.
template <int FMT>
__device__ __forceinline__ mx_u32x2 mx_encode8(const float (&v)[8], float inv) {
  mx_u32x2 r = {0, 0};
  const uint32_t keep = inv == 0.f ? 0u : ~0u;
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; j++) t[j] = v[j] * inv;
  if constexpr (FMT == MX_E4M3) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      int q = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * j], t[4 * j + 1], 0, false);
      r[j] = keep & (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[4 * j + 2], t[4 * j + 3], q, true);
    }
  } else {
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, t[0], t[1], 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, t[2], t[3], 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, t[4], t[5], 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, t[6], t[7], 1.0f, 3);
    r[0] = keep & q;
  }
  return r;
}

// Largest magnitude's bits (a NaN's are above infinity's) of 8 values
__device__ __forceinline__ uint32_t mx_top8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  return m;
}
// The maximum over the four lanes of a quad (quad_perm, full rate)
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));  // lanes 1, 0, 3, 2
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));  // lanes 2, 3, 0, 1
}

// In lanes that are multiples of 16: the bytes of lanes l, l + 4, l + 8, l + 12, lowest first (elsewhere: of no use)
__device__ __forceinline__ uint32_t mx_four_bytes(uint32_t b) {
  uint32_t w = b | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, 0x104, 0xf, 0xf, true) << 8;  // of four lanes on
  return w | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0x108, 0xf, 0xf, true) << 16;
}

// The maximum over lanes l and l ^ 16, and over l and l ^ 32: the swaps give every lane of a pair both values
__device__ __forceinline__ uint32_t mx_max_across16(uint32_t m) {
  const auto r = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}
__device__ __forceinline__ uint32_t mx_max_across32(uint32_t m) {
  const auto r = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}

// 16-bit storage <-> fp32, two values a word
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 mx_f16x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
template <bool F16>
__device__ __forceinline__ float mx_lo(uint32_t u) {
  if constexpr (F16) return (float)__builtin_bit_cast(mx_f16x2, u)[0];
  else return __uint_as_float(u << 16);
}
template <bool F16>
__device__ __forceinline__ float mx_hi(uint32_t u) {
  if constexpr (F16) return (float)__builtin_bit_cast(mx_f16x2, u)[1];
  else return __uint_as_float(u & 0xffff0000u);
}
template <bool F16>
__device__ __forceinline__ uint32_t mx_pack2(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_f32x2{a, b}, mx_f16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_f32x2{a, b}, mx_bf16x2));
}
template <bool F16>
__device__ __forceinline__ void mx_unpack8(mx_u32x4 q, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    v[2 * j] = mx_lo<F16>(q[j]);
    v[2 * j + 1] = mx_hi<F16>(q[j]);
  }
}
template <bool F16>
__device__ __forceinline__ mx_u32x4 mx_pack8(const float (&v)[8]) {
  return mx_u32x4{mx_pack2<F16>(v[0], v[1]), mx_pack2<F16>(v[2], v[3]), mx_pack2<F16>(v[4], v[5]), mx_pack2<F16>(v[6], v[7])};
}
// NV consecutive parameters p[i ...) of dtype dt (`none` without a pointer); the buffer need only be element-aligned
template <int NV>
__device__ __forceinline__ void mx_params(const void* p, int dt, i64 i, float none, float (&o)[NV]) {
#pragma unroll
  for (int q = 0; q < NV; q++) o[q] = none;
  if (!p) return;
  if (dt == F32) {
#pragma unroll
    for (int q = 0; q < NV; q++) o[q] = ((const float*)p)[i + q];
  } else if (dt == BF16) {
#pragma unroll
    for (int q = 0; q < NV; q++) o[q] = __uint_as_float((uint32_t)((const uint16_t*)p)[i + q] << 16);
  } else {
#pragma unroll
    for (int q = 0; q < NV; q++) o[q] = (float)((const _Float16*)p)[i + q];
  }
}

// mean and 1 / sqrt(variance + eps) of a row held by LPR lanes (this one has units sub, sub + LPR, ... below `units`, zeros
// else), or, without the mean, 1 / sqrt(mean square + eps); across: adds the lanes' sums over what LPR does not reach.
// s * (1 / c) is an ulp off s / c for a third of all c; a row of one large value, whose variance is 0, then has elements of that
// ulp, which 1 / sqrt(their square + eps) makes as large as 1. The mean gets the remainder's quotient (a division proper: [58321,
// 256] 12.8 -> 13.6 us).
template <int LPR, int CH, class F>
__device__ __forceinline__ void mx_row_stats(const float (&v)[CH][8], int sub, int units, float c, float inv_c, float eps, bool layer,
                                             float& mean, float& rstd, F&& across) {
  auto total = [&](float s) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 1; d < (LPR < 64 ? LPR : 64); d <<= 1) s += __shfl_xor(s, d, 64);
    return across(s);
  };
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < CH; k++)
#pragma unroll
    for (int j = 0; j < 8; j++) s += layer ? v[k][j] : v[k][j] * v[k][j];
  s = total(s);
  mean = 0.f;
  if (layer) {
    mean = s * inv_c;
    mean = fmaf(fmaf(-mean, c, s), inv_c, mean);
    s = 0.f;
#pragma unroll
    for (int k = 0; k < CH; k++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float d = k * LPR + sub < units ? v[k][j] - mean : 0.f;
        s += d * d;
      }
    s = total(s);
  }
  rstd = rsqrtf(s * inv_c + eps);
}
__device__ __forceinline__ void mx_norm8(const float (&v)[8], float mean, float rstd, const float (&g)[8], const float (&b)[8],
                                         float (&o)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++) o[j] = (v[j] - mean) * rstd * g[j] + b[j];
}
// f(integral_constant 0), f(1), ... f(N - 1)
template <class F, int... I>
__device__ __forceinline__ void mx_unroll_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void mx_unroll(F&& f) {
  mx_unroll_impl(f, std::make_integer_sequence<int, N>{});
}

// Host side, shared by the operators: argument checks
void mx_check(const MxTensor& q, const char* what);
void mx_check_apart(const MxTensor& q, const char* what);  // of a result: codes and scales share no byte
// Whether [a, a + na) and [b, b + nb) share a byte
inline bool mx_overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && na && nb && x < y + nb && y < x + na;
}
int mx_device_cus();

// The caller's workspace, or one of the library's own. The latter is refused while the stream is being captured: the graph
// would keep the address of a block that the library hands to other calls.
struct MxWorkspace {
  Tensor own;
  char* p;
  MxWorkspace(void* ws, i64 bytes, i64 need) {
    if (ws) {
      REQ((uintptr_t)ws % 16 == 0 && bytes >= need, "workspace of %lld bytes: %lld needed, 16-byte aligned", (long long)bytes,
          (long long)need);
      p = (char*)ws;
    } else if (need) {
      hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
      CK(hipStreamIsCapturing(stream(), &st));
      REQ(st == hipStreamCaptureStatusNone, "a captured call needs a workspace of its caller (%lld bytes)", (long long)need);
      own = empty({need}, U8);
      p = (char*)own.p;
    } else {
      p = nullptr;
    }
  }
  Tensor take(i64 bytes) {
    Tensor t = borrow(p, {bytes}, U8);
    p += (bytes + 255) / 256 * 256;
    return t;
  }
  MxTensor rows(int fmt, i64 n, i64 cols) {
    MxTensor q;
    q.fmt = fmt;
    q.rows = n;
    q.cols = cols;
    q.codes = take(n * mx_row_bytes(fmt, cols));
    q.scales = take(n * mx_scale_bytes(cols));
    return q;
  }
};
inline i64 mx_rows_bytes(int fmt, i64 n, i64 cols) {
  return (n * mx_row_bytes(fmt, cols) + 255) / 256 * 256 + (n * mx_scale_bytes(cols) + 255) / 256 * 256;
}

inline void mx_apart(const void* a, size_t na, const void* b, size_t nb, const char* what) {
  REQ(!mx_overlap(a, na, b, nb), "operands must not overlap %s", what);
}
inline void mx_out_apart(const Tensor* y, const MxTensor* yq, const Tensor& t, const char* what) {
  if (y) mx_apart(y->p, y->bytes(), t.p, t.bytes(), what);
  if (yq) {
    mx_apart(yq->codes.p, yq->codes.bytes(), t.p, t.bytes(), what);
    mx_apart(yq->scales.p, yq->scales.bytes(), t.p, t.bytes(), what);
  }
}

// mx_linear without its checks. xv: x's values (at most 16 rows), which the product quantises to x's format itself; else x's codes
void mx_product(const MxTensor& x, const MxTensor& w, const Tensor* bias, const Tensor* res, int act, Tensor* y, MxTensor* yq,
                const Tensor* xv = nullptr);
