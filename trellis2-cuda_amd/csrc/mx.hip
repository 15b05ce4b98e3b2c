// Rows into blocks of 32 values with a shared power-of-two scale and back (mx.h), and the norm that writes such rows:
// the residual's addition, root-mean-square or LayerNorm, the affine, and the quantisation in one pass.
#include "mx.h"

#include <algorithm>

#include "lnact.h"

i64 mx_row_bytes(int fmt, i64 cols) { return fmt == MX_E2M1 ? cols / 2 : cols; }
i64 mx_scale_bytes(i64 cols) { return (cols + 511) / 512 * 16; }

int mx_device_cus() {
  static int n[64] = {};
  int dev = 0;
  CK(hipGetDevice(&dev));
  if (dev < 0 || dev >= 64) return 256;
  if (!n[dev]) CK(hipDeviceGetAttribute(&n[dev], hipDeviceAttributeMultiprocessorCount, dev));
  return n[dev];
}

void mx_check(const MxTensor& q, const char* what) {
  REQ(q.fmt == MX_E4M3 || q.fmt == MX_E2M1, "%s: format %d", what, q.fmt);
  REQ(q.rows >= 0 && q.rows < (1ll << 31) && q.cols > 0 && q.cols % 32 == 0 && q.cols <= (1 << 20),
      "%s [%lld,%lld]: columns must be a multiple of 32, at most 2^20, rows below 2^31", what, (long long)q.rows,
      (long long)q.cols);
  REQ(q.codes.dt == U8 && q.scales.dt == U8 && q.codes.numel() == q.rows * mx_row_bytes(q.fmt, q.cols) &&
          q.scales.numel() == q.rows * mx_scale_bytes(q.cols),
      "%s: codes and scales must be the bytes of [%lld,%lld]", what, (long long)q.rows, (long long)q.cols);
  REQ(q.rows == 0 || (q.codes.p && q.scales.p), "%s: null codes or scales", what);
  REQ(((uintptr_t)q.codes.p | (uintptr_t)q.scales.p) % 16 == 0, "%s: codes and scales must be 16-byte aligned", what);
}
void mx_check_apart(const MxTensor& q, const char* what) {
  REQ(!mx_overlap(q.codes.p, q.codes.bytes(), q.scales.p, q.scales.bytes()), "%s: codes and scales must not overlap", what);
}

namespace {
// 8 consecutive values of unit u
template <int T>
__device__ __forceinline__ void load8(const void* x, i64 u, float (&v)[8]) {
  if constexpr (T == F32) {
    const mx_u32x4 a = ((const mx_u32x4*)x)[2 * u], b = ((const mx_u32x4*)x)[2 * u + 1];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      v[j] = __uint_as_float(a[j]);
      v[4 + j] = __uint_as_float(b[j]);
    }
  } else {
    mx_unpack8<T == F16>(((const mx_u32x4*)x)[u], v);
  }
}

// A block's scale byte, and zeros behind a row's last one up to the padded stride
__device__ __forceinline__ void put_scale(uint8_t* scales, i64 row, uint32_t col, uint32_t per, uint32_t stride,
                                          uint32_t byte) {
  uint8_t* s = scales + row * stride;
  s[col] = (uint8_t)byte;
  if (col + 1 == per)
    for (uint32_t k = per; k < stride; k++) s[k] = 0;
}

// One lane per 8 values, four lanes per block, four blocks' scale bytes a store. HBM-bound: bf16 [390503, 256] (253 MB with
// e2m1's) 43 us there, 38 back; [65536, 1024] with e4m3 38 and 31. Few values: a launch's latency (3 us).
constexpr int kQuantUnits = 4;
template <int FMT, int T>
__global__ void __launch_bounds__(256) k_mx_quantize(const void* __restrict__ x, i64 units, uint32_t per, uint32_t stride,
                                                     uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const i64 u0 = (i64)blockIdx.x * (256 * kQuantUnits) + threadIdx.x;
  float v[kQuantUnits][8];
#pragma unroll
  for (int k = 0; k < kQuantUnits; k++) load8<T>(x, min(u0 + k * 256, units - 1), v[k]);
#pragma unroll
  for (int k = 0; k < kQuantUnits; k++) {
    const i64 u = u0 + k * 256;
    const uint32_t byte = mx_scale_byte<FMT>(mx_quad_max(mx_top8(v[k])));
    const mx_u32x2 q = mx_encode8<FMT>(v[k], mx_inverse(byte));
    if (u >= units) break;  // a quad's four units are inside or outside together, and 16 lanes' where per % 4 == 0
    if constexpr (FMT == MX_E4M3) ((mx_u32x2*)codes)[u] = q;
    else ((uint32_t*)codes)[u] = q[0];
    const uint32_t b = (uint32_t)(u >> 2), row = b / per, col = b - row * per;
    if (per % 4 == 0) {  // four blocks' bytes are a word of one row
      const uint32_t w = mx_four_bytes(byte);
      if ((threadIdx.x & 15) == 0) {
        uint32_t* s = (uint32_t*)(scales + (i64)row * stride + col);
        *s = w;
        if (col + 4 == per)
          for (uint32_t k = 1; k < (stride - col) / 4; k++) s[k] = 0;
      }
    } else if ((threadIdx.x & 3) == 0) {
      put_scale(scales, row, col, per, stride, byte);
    }
  }
}

// The values are stored past the caches: bf16 [390503, 256], after mx_quantize, 97 -> 83 us for both.
template <int FMT, int T>
__global__ void __launch_bounds__(256) k_mx_dequantize(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                       i64 units, uint32_t per, uint32_t stride, void* __restrict__ y) {
  const i64 u0 = (i64)blockIdx.x * (256 * kQuantUnits) + threadIdx.x;
  mx_u32x2 q[kQuantUnits];
  uint32_t byte[kQuantUnits];
#pragma unroll
  for (int k = 0; k < kQuantUnits; k++) {
    const i64 u = min(u0 + k * 256, units - 1);
    if constexpr (FMT == MX_E4M3) q[k] = ((const mx_u32x2*)codes)[u];
    else q[k] = mx_u32x2{((const uint32_t*)codes)[u], 0};
    const uint32_t b = (uint32_t)(u >> 2), row = b / per;
    byte[k] = scales[(i64)row * stride + (b - row * per)];
  }
#pragma unroll
  for (int k = 0; k < kQuantUnits; k++) {
    const i64 u = u0 + k * 256;
    if (u >= units) break;
    const float s = mx_scale_value(byte[k]);
    float v[8];
    if constexpr (FMT == MX_E4M3) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const mx_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[k][j], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[k][j], true);
        v[4 * j] = a[0] * s;
        v[4 * j + 1] = a[1] * s;
        v[4 * j + 2] = b[0] * s;
        v[4 * j + 3] = b[1] * s;
      }
    } else {
      const mx_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k][0], 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k][0], 1.0f, 1),
                     c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k][0], 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[k][0], 1.0f, 3);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        v[j] = a[j] * s;
        v[2 + j] = b[j] * s;
        v[4 + j] = c[j] * s;
        v[6 + j] = d[j] * s;
      }
    }
    if constexpr (T == F32) {
      typedef float f32x4 __attribute__((ext_vector_type(4)));
      __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, (f32x4*)y + 2 * u);
      __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, (f32x4*)y + 2 * u + 1);
    } else {
      __builtin_nontemporal_store(mx_pack8<T == F16>(v), (mx_u32x4*)y + u);
    }
  }
}

template <class F>
void by_format(int fmt, F&& f) {
  if (fmt == MX_E4M3) f(std::integral_constant<int, MX_E4M3>{});
  else f(std::integral_constant<int, MX_E2M1>{});
}
template <class F>
void by_float(DT dt, F&& f) {
  if (dt == F32) f(std::integral_constant<int, F32>{});
  else if (dt == F16) f(std::integral_constant<int, F16>{});
  else f(std::integral_constant<int, BF16>{});
}
bool is_float(DT dt) { return dt == F32 || dt == F16 || dt == BF16; }
}  // namespace

void mx_quantize(const Tensor& x, MxTensor& q) {
  mx_check(q, "q");
  mx_check_apart(q, "q");
  REQ(is_float(x.dt) && x.dim() == 2 && x.size(0) == q.rows && x.size(1) == q.cols, "x must be fp32/fp16/bf16 [%lld,%lld]",
      (long long)q.rows, (long long)q.cols);
  REQ((uintptr_t)x.p % 16 == 0 && (x.p || q.rows == 0), "x must be 16-byte aligned and not null");
  REQ(!mx_overlap(x.p, x.bytes(), q.codes.p, q.codes.bytes()) && !mx_overlap(x.p, x.bytes(), q.scales.p, q.scales.bytes()),
      "codes and scales must not overlap x");
  const i64 units = q.rows * q.cols / 8;
  REQ(units / 4 < (1ll << 32), "%lld values: at most 2^37", (long long)(units * 8));
  if (!units) return;
  by_format(q.fmt, [&](auto FC) {
    by_float(x.dt, [&](auto TC) {
      k_mx_quantize<decltype(FC)::value, decltype(TC)::value><<<(unsigned)((units + 256 * kQuantUnits - 1) / (256 * kQuantUnits)), 256, 0, stream()>>>(
          x.p, units, (uint32_t)(q.cols / 32), (uint32_t)mx_scale_bytes(q.cols), q.codes.ptr<uint8_t>(), q.scales.ptr<uint8_t>());
    });
  });
  CK(hipGetLastError());
}

void mx_dequantize(const MxTensor& q, Tensor& y) {
  mx_check(q, "q");
  REQ(is_float(y.dt) && y.dim() == 2 && y.size(0) == q.rows && y.size(1) == q.cols, "y must be fp32/fp16/bf16 [%lld,%lld]",
      (long long)q.rows, (long long)q.cols);
  REQ((uintptr_t)y.p % 16 == 0 && (y.p || q.rows == 0), "y must be 16-byte aligned and not null");
  REQ(!mx_overlap(y.p, y.bytes(), q.codes.p, q.codes.bytes()) && !mx_overlap(y.p, y.bytes(), q.scales.p, q.scales.bytes()),
      "y must not overlap codes or scales");
  const i64 units = q.rows * q.cols / 8;
  REQ(units / 4 < (1ll << 32), "%lld values: at most 2^37", (long long)(units * 8));
  if (!units) return;
  by_format(q.fmt, [&](auto FC) {
    by_float(y.dt, [&](auto TC) {
      k_mx_dequantize<decltype(FC)::value, decltype(TC)::value><<<(unsigned)((units + 256 * kQuantUnits - 1) / (256 * kQuantUnits)), 256, 0, stream()>>>(
          q.codes.ptr<uint8_t>(), q.scales.ptr<uint8_t>(), units, (uint32_t)(q.cols / 32), (uint32_t)mx_scale_bytes(q.cols), y.p);
    });
  });
  CK(hipGetLastError());
}

// ---- norm -------------------------------------------------------------------------------------------------------
//   t = round(x + r) (r optional; the sum that a caller keeps is the sum that is normalised)
//   RMS    y = t / sqrt(mean(t^2) + eps) * gamma + beta        LAYER  y = (t - mean t) / sqrt(var t + eps) * gamma + beta
// and y's blocks quantised; statistics, norm and amax in fp32 registers, one rounding to the elements. A row is read
// once: LPR lanes hold it, 8 channels per lane and chunk, so a block of 32 is a quad of lanes (C / 8 is a multiple of 4:
// a quad has all of a block or nothing). LPR = 256: a workgroup per row, partial sums through LDS; LPR <= 64: a wavefront
// or part of one. HBM-bound: bf16 with a residual [32771, 4096] 177 us (5.3 TB/s), fp16 [58321, 256] 13 us (3.5;
// 7291 groups of rows on 4096 workgroups, half of which fit the card: most take two turns), one row 2.9.
// us with a wavefront / a workgroup per row, [20000, 512] 13.3 / 21.9, [40000, 1024] 52 / 56, [5000, 2048] 14.0 / 12.8,
// [20000, 2048] 51 / 53, [32771, 4096] 211 / 177, [2000, 4096] 17 / 11: a workgroup from more than 1024 channels on.
// The sum is stored past the caches (what reads it next is a block away): [32771, 4096] 183 -> 178.
namespace {
struct NormArgs {
  const uint16_t *x, *r;
  uint16_t* sum;
  const void *gamma, *beta;
  int gdt, bdt, kind, C;
  i64 n;
  float eps;
  uint8_t *codes, *scales;
  uint32_t stride;
};

template <bool F16, int FMT, int LPR, int CH>
__global__ void __launch_bounds__(256) k_add_norm_mx(NormArgs a) {
  constexpr int RPB = 256 / LPR;  // rows of a workgroup at a time
  __shared__ float part[2][4];
  int slot = 0;
  const int sub = threadIdx.x % LPR, units = a.C / 8;
  float g[CH][8], b[CH][8];
#pragma unroll
  for (int k = 0; k < CH; k++) {
    const int u = k * LPR + sub;
    mx_params<8>(u < units ? a.gamma : nullptr, a.gdt, u * 8, 1.f, g[k]);
    mx_params<8>(u < units ? a.beta : nullptr, a.bdt, u * 8, 0.f, b[k]);
  }
  const float c = (float)a.C, inv_c = 1.f / c;
  const i64 step = (i64)gridDim.x * RPB;
  // whole workgroups go round together (the reductions below need every lane): rows past the last repeat it
  for (i64 row0 = (i64)blockIdx.x * RPB; row0 < a.n; row0 += step) {
    const i64 row = min(row0 + threadIdx.x / LPR, a.n - 1);
    const bool live = row0 + threadIdx.x / LPR < a.n;
    const i64 base = row * units;
    mx_u32x4 q[CH], r[CH];
#pragma unroll
    for (int k = 0; k < CH; k++) {
      const int u = k * LPR + sub;
      q[k] = u < units ? ((const mx_u32x4*)a.x)[base + u] : mx_u32x4{};
      r[k] = a.r && u < units ? ((const mx_u32x4*)a.r)[base + u] : mx_u32x4{};
    }
    float v[CH][8];
#pragma unroll
    for (int k = 0; k < CH; k++) {
      mx_unpack8<F16>(q[k], v[k]);
      if (a.r) {
        float w[8];
        mx_unpack8<F16>(r[k], w);
#pragma unroll
        for (int j = 0; j < 8; j++) v[k][j] += w[j];
        q[k] = mx_pack8<F16>(v[k]);
        mx_unpack8<F16>(q[k], v[k]);
      }
    }
    float mean, rstd;
    mx_row_stats<LPR, CH>(v, sub, units, c, inv_c, a.eps, a.kind == MX_NORM_LAYER, mean, rstd, [&](float s) __attribute__((always_inline)) {
      if constexpr (LPR == 256) {  // two slots in turn: one is written again only past another barrier
        float* p = part[slot ^= 1];
        if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = s;
        __syncthreads();
        s = (p[0] + p[1]) + (p[2] + p[3]);
      }
      return s;
    });
#pragma unroll
    for (int k = 0; k < CH; k++) {
      const int u = k * LPR + sub;
      float o[8];
      mx_norm8(v[k], mean, rstd, g[k], b[k], o);
      const uint32_t byte = mx_scale_byte<FMT>(mx_quad_max(mx_top8(o)));
      const mx_u32x2 e = mx_encode8<FMT>(o, mx_inverse(byte));
      // scales, and zeros behind a row's last: 16 lanes' blocks are a word, a row of up to 256 channels fills 16 bytes by itself
      const uint32_t w = mx_four_bytes(u < units ? byte : 0u);
      const uint32_t w1 = LPR == 32 ? (uint32_t)__shfl_down((int)w, 16, 64) : 0u;
      if (!live) continue;
      if constexpr (LPR >= 64) {
        if (sub % 16 == 0 && u / 4 < (int)a.stride) *(uint32_t*)(a.scales + row * a.stride + u / 4) = w;
      } else {
        if (sub == 0) *(mx_u32x4*)(a.scales + row * a.stride) = mx_u32x4{LPR == 8 ? w & 0xffffu : w, w1, 0, 0};
      }
      if (u >= units) continue;
      if (a.sum) __builtin_nontemporal_store(q[k], (mx_u32x4*)a.sum + base + u);
      if constexpr (FMT == MX_E4M3) ((mx_u32x2*)a.codes)[base + u] = e;
      else ((uint32_t*)a.codes)[base + u] = e[0];
    }
  }
}
}  // namespace

void add_norm_mx(const Tensor& x, const Tensor* residual, const Tensor* gamma, const Tensor* beta, float eps, int kind,
                 Tensor* sum, MxTensor& q) {
  mx_check(q, "q");
  REQ(x.dim() == 2 && (x.dt == BF16 || x.dt == F16), "x must be bf16/fp16 [N,C]");
  const i64 n = x.size(0), C = x.size(1);
  REQ(C > 0 && C % 32 == 0 && C <= 16384, "C=%lld: a multiple of 32, at most 16384", (long long)C);
  REQ(q.rows == n && q.cols == C, "q must be [%lld,%lld]", (long long)n, (long long)C);
  mx_check_apart(q, "q");
  REQ(kind == MX_NORM_RMS || kind == MX_NORM_LAYER, "kind=%d", kind);
  if (residual) REQ(residual->dt == x.dt && residual->dim() == 2 && residual->size(0) == n && residual->size(1) == C, "residual must match x");
  if (sum) REQ(sum->dt == x.dt && sum->dim() == 2 && sum->size(0) == n && sum->size(1) == C, "sum must match x");
  REQ(!residual || sum, "a residual needs a sum to write");
  for (const Tensor* t : {gamma, beta}) REQ(!t || (is_float(t->dt) && t->numel() == C), "gamma/beta must have C elements");
  if (n == 0) return;
  const Tensor* rows[3] = {&x, residual, sum};
  for (const Tensor* t : rows) {
    if (!t) continue;
    REQ(t->p && (uintptr_t)t->p % 16 == 0, "x, residual and sum must be 16-byte aligned and not null");
    REQ(!mx_overlap(t->p, t->bytes(), q.codes.p, q.codes.bytes()) && !mx_overlap(t->p, t->bytes(), q.scales.p, q.scales.bytes()),
        "codes and scales must not overlap x, residual or sum");
  }
  for (const Tensor* t : {gamma, beta})
    if (t) mx_out_apart(sum, &q, *t, "gamma or beta");
  for (const Tensor* t : {&x, residual})  // in place is fine: a lane reads what it then writes
    REQ(!t || !sum || sum->p == t->p || !mx_overlap(t->p, t->bytes(), sum->p, sum->bytes()), "sum must be x, residual or apart from both");
  NormArgs a{};
  a.x = x.ptr<uint16_t>();
  a.r = residual ? residual->ptr<uint16_t>() : nullptr;
  a.sum = sum && (residual || sum->p != x.p) ? sum->ptr<uint16_t>() : nullptr;
  a.gamma = gamma ? gamma->p : nullptr;
  a.beta = beta ? beta->p : nullptr;
  a.gdt = gamma ? gamma->dt : F32;
  a.bdt = beta ? beta->dt : F32;
  a.kind = kind;
  a.C = (int)C;
  a.n = n;
  a.eps = eps;
  a.codes = q.codes.ptr<uint8_t>();
  a.scales = q.scales.ptr<uint8_t>();
  a.stride = (uint32_t)mx_scale_bytes(C);
  auto go = [&](auto L, auto K) {
    constexpr int LPR = decltype(L)::value, CH = decltype(K)::value;
    const i64 blocks = (n + 256 / LPR - 1) / (256 / LPR);
    const unsigned grid = (unsigned)std::min<i64>(blocks, (i64)mx_device_cus() * 16);
    by_format(q.fmt, [&](auto FC) {
      if (x.dt == F16) k_add_norm_mx<true, decltype(FC)::value, LPR, CH><<<grid, 256, 0, stream()>>>(a);
      else k_add_norm_mx<false, decltype(FC)::value, LPR, CH><<<grid, 256, 0, stream()>>>(a);
    });
  };
  using std::integral_constant;
  if (C <= 64) go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  else if (C <= 128) go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (C <= 256) go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  else if (C <= 512) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (C <= 1024) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (C <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (C <= 4096) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (C <= 8192) go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else go(integral_constant<int, 256>{}, integral_constant<int, 8>{});
  CK(hipGetLastError());
}
