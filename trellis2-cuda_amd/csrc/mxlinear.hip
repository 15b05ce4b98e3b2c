// Linear layers of microscaled rows (mx.h):  y = act(X . W^T + b) + r,  X [N,K] e4m3 or e2m1, W [O,K] e2m1, fp32 sums.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 elements and their scales, one scale byte per row
// and 32 columns. Lane l supplies row l % 16 of either operand. With g = l / 16 it holds, of 4-bit elements, columns
// 32 g .. 32 g + 31 (16 bytes), of 8-bit ones 16 g .. and 64 + 16 g .. (two times 16 bytes), and in both cases the
// scale of columns 32 g .. 32 g + 31. The result gives lane l column l % 16 and rows 4 g + i. W is the first operand, so
// a lane holds 4 channels of one row of X per product, and the channel that each of W's 16 rows stands for is free:
// channel(tile t, g, i) = (t / G) * 16 G + g * 4 G + (t % G) * 4 + i gives a lane 4 G consecutive channels over G tiles, so
// its stores are whole 16-byte pieces.
#include "mx.h"

#include <algorithm>

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
  int tiles_n, tiles_o, per, o_major;
};

__device__ __forceinline__ i32x4 rsrc4(const void* p, uint32_t bytes) {  // a raw buffer's descriptor, in SGPRs
  const uint64_t b = (uint64_t)(uintptr_t)p;
  return i32x4{(int32_t)__builtin_amdgcn_readfirstlane((uint32_t)b), (int32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)),
               (int32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// 16 bytes per lane, global -> LDS: lane l's land at dst + 16 l. Inline assembly, so that the compiler does not put a
// wait for it before every LDS read; the loop below counts them.
__device__ __forceinline__ void dma16(i32x4 r, uint32_t lds, uint32_t off, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               ::"s"(lds), "v"(off), "s"(r), "s"(soff) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

template <int XB>
__device__ __forceinline__ f32x4 mfma(mx_u32x4 w, const mx_u32x4 (&x)[XB / 4], f32x4 c, int sw, int sx) {
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  if constexpr (XB == 8) {
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, sw, 0, sx);
  } else {
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, sw, 0, sx);
  }
}
template <int OUT, int TO>
constexpr int run_tiles() {  // G above
  return OUT == OUT_F32 ? 1 : OUT == OUT_16 ? 2 : 4 < TO ? 4 : TO;
}

// Epilogue of 4 G consecutive channels o .. of row n in v: bias, activation, residual, store
template <int OUT, int NV>
__device__ __forceinline__ void finish(const LinArgs& a, i64 n, int o, float (&v)[NV], const float (&bias)[NV], bool ok, int g) {
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
      const f32x4 r = *(const f32x4*)((const float*)a.res + n * a.O + o);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += r[j];
    }
    *(f32x4*)((float*)a.out + n * a.O + o) = f32x4{v[0], v[1], v[2], v[3]};
  } else if constexpr (OUT == OUT_16) {
    static_assert(NV == 8, "one 16-byte piece");
    if (!ok) return;
    if (a.res) {
      const mx_u32x4 q = *(const mx_u32x4*)((const uint16_t*)a.res + n * a.O + o);
      float r[8];
      if (a.f16) mx_unpack8<true>(q, r);
      else mx_unpack8<false>(q, r);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += r[j];
    }
    *(mx_u32x4*)((uint16_t*)a.out + n * a.O + o) = a.f16 ? mx_pack8<true>(v) : mx_pack8<false>(v);
  } else {
    // 16 channels a lane, two lanes (g and g ^ 1) a block; both are inside or outside together
    static_assert(NV == 16, "half a block");
    constexpr int FMT = OUT == OUT_MX8 ? MX_E4M3 : MX_E2M1;
    float(&lo)[8] = *(float(*)[8])&v[0];
    float(&hi)[8] = *(float(*)[8])&v[8];
    uint32_t top = max(mx_top8(lo), mx_top8(hi));
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    const uint32_t byte = mx_scale_byte<FMT>(top);
    const float inv = mx_inverse(byte);
    const mx_u32x2 p = mx_encode8<FMT>(lo, inv), q = mx_encode8<FMT>(hi, inv);
    if (!ok) return;
    if constexpr (FMT == MX_E4M3) *(mx_u32x4*)((uint8_t*)a.out + n * a.O + o) = mx_u32x4{p[0], p[1], q[0], q[1]};
    else *(mx_u32x2*)((uint8_t*)a.out + (n * a.O + o) / 2) = mx_u32x2{p[0], q[0]};
    if ((g & 1) == 0) {
      uint8_t* s = a.outs + n * a.osrow;
      s[o / 32] = (uint8_t)byte;
      if (o / 32 + 1 == a.O / 32)
        for (int k = a.O / 32; k < a.osrow; k++) s[k] = 0;
    }
  }
}

// Tiled product. A workgroup of WO x WN wavefronts has BO = 16 TO WO channels by BN = 16 TN WN rows; K goes by steps of
// 128 through NS slots of LDS, filled by DMA NS - 1 steps ahead, with one barrier a step; the scales go by 512 columns
// (16 bytes a row), two slots. LDS rows are 64 (e2m1) or 128 bytes (e4m3) of a step, their 16-byte pieces permuted
// (piece c of row q at c ^ (q >> 2) % 4 or c ^ q % 8), so that eight lanes of neighbouring rows read from distinct banks.
template <int XB, int OUT, int TO, int TN, int WO, int WN, int NS>
__global__ void __launch_bounds__(64 * WO * WN) k_mx_gemm(LinArgs a) {
  constexpr int NW = WO * WN, BO = 16 * TO * WO, BN = 16 * TN * WN, D = NS - 1;
  constexpr int XR = XB == 8 ? 128 : 64;                                       // bytes of a row of X per step
  constexpr int XI = BN * XR / 1024 / NW, WI = BO * 64 / 1024 / NW, SI = (BO + BN) / 64 / NW;  // DMAs per wavefront
  static_assert(XI * 1024 * NW == BN * XR && WI * 1024 * NW == BO * 64 && SI * 64 * NW == BO + BN, "whole DMAs");
  constexpr int G = run_tiles<OUT, TO>();
  static_assert(TO % G == 0, "whole runs");
  __shared__ __attribute__((aligned(16))) mx_u32x4 lds[NS * (BN * XR + BO * 64) / 16 + 2 * (BO + BN)];
  constexpr uint32_t kSlot = BN * XR + BO * 64, kScales = NS * kSlot, kScaleSlot = (BO + BN) * 16;

  const int logical = (blockIdx.x % 8) * a.per + blockIdx.x / 8;  // each XCD walks one contiguous range of tiles
  if (logical >= a.tiles_n * a.tiles_o) return;
  const int tn = a.o_major ? logical % a.tiles_n : logical / a.tiles_o;
  const int to = a.o_major ? logical / a.tiles_n : logical % a.tiles_o;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wo = wave % WO, wn = wave / WO;
  const int S = (a.K + 127) / 128;
  const i64 n0 = (i64)tn * BN;
  const int o0 = to * BO;
  const int rows = (int)min((i64)BN, a.N - n0), chans = min(BO, a.O - o0);
  // descriptors of this tile's rows: anything past them reads as zero
  const i32x4 rx = rsrc4(a.x + n0 * a.xrow, (uint32_t)(rows * a.xrow)), rw = rsrc4(a.w + (i64)o0 * a.wrow, (uint32_t)(chans * a.wrow));
  const i32x4 rxs = rsrc4(a.xs + n0 * a.srow, (uint32_t)(rows * a.srow)), rws = rsrc4(a.ws + (i64)o0 * a.srow, (uint32_t)(chans * a.srow));
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) mx_u32x4*)&lds[0];

  // the channel of W's LDS row p
  auto channel = [&](int p) __attribute__((always_inline)) {
    const int t = p / 16 % TO, r = p % 16;
    return p / (16 * TO) * (16 * TO) + t / G * (16 * G) + r / 4 * (4 * G) + t % G * 4 + r % 4;
  };
  uint32_t xoff[XI], woff[WI], soff[SI];
  int xc[XI], wc[WI];  // first byte within the step, to cut a last step short
#pragma unroll
  for (int k = 0; k < XI; k++) {
    const int p = (wave * XI + k) * 64 + lane, q = p / (XR / 16), c = p % (XR / 16);
    xc[k] = XB == 8 ? (c ^ (q & 7)) * 16 : (c ^ ((q >> 2) & 3)) * 16;
    xoff[k] = q < rows ? (uint32_t)(q * a.xrow + xc[k]) : kOOR;
  }
#pragma unroll
  for (int k = 0; k < WI; k++) {
    const int p = (wave * WI + k) * 64 + lane, q = p / 4, c = p % 4, ch = channel(q);
    wc[k] = (c ^ ((q >> 2) & 3)) * 16;
    woff[k] = ch < chans ? (uint32_t)(ch * a.wrow + wc[k]) : kOOR;
  }
#pragma unroll
  for (int k = 0; k < SI; k++) {
    const int p = (wave * SI + k) * 64 + lane, ch = channel(p < BO ? p : 0);
    soff[k] = p < BO ? (ch < chans ? (uint32_t)(ch * a.srow) : kOOR) : p - BO < rows ? (uint32_t)((p - BO) * a.srow) : kOOR;
  }
  // fills step t's slot; past the last step the DMAs still run (the waits count them) but read nothing
  auto issue = [&](int t, int slot) __attribute__((always_inline)) {
    const bool live = t < S;
    if (t % 4 == 0) {
#pragma unroll
      for (int k = 0; k < SI; k++) {
        const int p0 = (wave * SI + k) * 64;  // BO is a multiple of 64: a DMA's rows are all W's or all X's
        const bool w = p0 < BO;
        dma16(w ? rws : rxs, lds0 + kScales + (t / 4 & 1) * kScaleSlot + p0 * 16, live ? soff[k] : kOOR, live ? t * 4 : 0);
      }
    }
    const bool cut = live && (t + 1) * 128 > a.K;
    const int xleft = cut ? a.xrow - t * XR : XR, wleft = cut ? a.wrow - t * 64 : 64;
#pragma unroll
    for (int k = 0; k < XI; k++)
      dma16(rx, lds0 + slot * kSlot + (wave * XI + k) * 1024, live && xc[k] < xleft ? xoff[k] : kOOR, live ? t * XR : 0);
#pragma unroll
    for (int k = 0; k < WI; k++)
      dma16(rw, lds0 + slot * kSlot + BN * XR + (wave * WI + k) * 1024, live && wc[k] < wleft ? woff[k] : kOOR, live ? t * 64 : 0);
  };

  f32x4 acc[TO][TN];
#pragma unroll
  for (int t = 0; t < TO; t++)
#pragma unroll
    for (int u = 0; u < TN; u++) acc[t][u] = f32x4{};

  // where this lane reads, in 16-byte units of a slot
  const int xq = wn * (16 * TN) + r16, wp = wo * (16 * TO) + r16;
  const int xa0 = XB == 8 ? xq * 8 + (g ^ (r16 & 7)) : xq * 4 + (g ^ (r16 >> 2)), xa1 = xq * 8 + ((g + 4) ^ (r16 & 7));
  const int wa = BN * XR / 16 + wp * 4 + (g ^ (r16 >> 2));
  const int blocks = a.K / 32;

  int fill = 0;
#pragma unroll
  for (int t = 0; t < D; t++) issue(t, fill++);
  int cur = 0;
  auto step = [&](auto I, int s) __attribute__((always_inline)) {
    constexpr int i = decltype(I)::value;
    // the D - 1 steps after this one may be in flight, and the scales that come with them
    constexpr int ahead = (D - 1) * (XI + WI) + SI * ((D > 1 && (i + 1) % 4 == 0) + (D > 2 && (i + 2) % 4 == 0));
    static_assert(D <= 3, "at most two steps after this one");
    wait_vm<ahead>();
    bare_barrier();
    issue(s + D, fill);
    fill = fill + 1 == NS ? 0 : fill + 1;
    const mx_u32x4* slot = lds + cur * (kSlot / 16);
    const uint8_t* sc = (const uint8_t*)lds + kScales + (s / 4 & 1) * kScaleSlot + i * 4 + g;
    const bool in = s * 4 + g < blocks;  // the padding behind a row's last scale is not read as a scale
    mx_u32x4 fx[TN][XB / 4];
    int sx[TN];
#pragma unroll
    for (int u = 0; u < TN; u++) {
      fx[u][0] = slot[xa0 + u * (XR)];
      if constexpr (XB == 8) fx[u][1] = slot[xa1 + u * XR];
      const int b = sc[(BO + xq + u * 16) * 16];
      sx[u] = in ? b : 0;
    }
#pragma unroll
    for (int t = 0; t < TO; t++) {
      const mx_u32x4 fw = slot[wa + t * 64];
      const int b = sc[(wp + t * 16) * 16];
      const int sw = in ? b : 0;
#pragma unroll
      for (int u = 0; u < TN; u++) acc[t][u] = mfma<XB>(fw, fx[u], acc[t][u], sw, sx[u]);
    }
    cur = cur + 1 == NS ? 0 : cur + 1;
  };
  for (int s = 0; s < S; s += 4) {
    step(std::integral_constant<int, 0>{}, s);
    if (s + 1 < S) step(std::integral_constant<int, 1>{}, s + 1);
    if (s + 2 < S) step(std::integral_constant<int, 2>{}, s + 2);
    if (s + 3 < S) step(std::integral_constant<int, 3>{}, s + 3);
  }
  wait_vm<0>();  // nothing lands in LDS after the workgroup has gone

#pragma unroll
  for (int t = 0; t < TO; t += G) {
    const int o = o0 + wo * (16 * TO) + t / G * (16 * G) + g * (4 * G);
    float bias[4 * G];
    mx_params<4 * G>(o < a.O ? a.bias : nullptr, a.bias_dt, o, 0.f, bias);
#pragma unroll
    for (int u = 0; u < TN; u++) {
      const i64 n = n0 + xq + u * 16;
      float v[4 * G];
#pragma unroll
      for (int j = 0; j < G; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) v[j * 4 + i] = acc[t + j][u][i];
      finish<OUT>(a, n, o, v, bias, n < a.N && o < a.O, g);
    }
  }
}

template <int XB, int OUT, int TO, int TN, int WO, int WN, int NS>
void launch(LinArgs a) {
  constexpr int BO = 16 * TO * WO, BN = 16 * TN * WN;
  const i64 tn = (a.N + BN - 1) / BN, to = (a.O + BO - 1) / BO;
  REQ(tn * to < (1ll << 30), "%lld rows by %d channels: too many tiles", (long long)a.N, a.O);
  a.tiles_n = (int)tn;
  a.tiles_o = (int)to;
  a.per = cdiv(tn * to, 8);
  a.o_major = (i64)a.O * a.wrow > (2 << 20);
  k_mx_gemm<XB, OUT, TO, TN, WO, WN, NS><<<a.per * 8, 64 * WO * WN, 0, stream()>>>(a);
  CK(hipGetLastError());
}

template <int XB, int OUT>
void gemm(const LinArgs& a) {
  const i64 cus = mx_device_cus();
  const i64 big = (i64)cdiv(a.N, 256) * cdiv(a.O, 256);
  if (big >= cus) launch<XB, OUT, 8, 4, 2, 4, XB == 8 ? 3 : 4>(a);
  else launch<XB, OUT, 4, 4, 2, 2, XB == 8 ? 3 : 4>(a);
}
}  // namespace

namespace {
// The caller's workspace, or one of the library's own. The latter is refused while the stream is being captured: the graph
// would keep the address of a block that the library hands to other calls.
struct Workspace {
  Tensor own;
  char* p;
  i64 left;
  Workspace(void* ws, i64 bytes, i64 need) {
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
    left = need;
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
i64 rows_bytes(int fmt, i64 n, i64 cols) {
  return (n * mx_row_bytes(fmt, cols) + 255) / 256 * 256 + (n * mx_scale_bytes(cols) + 255) / 256 * 256;
}

// shapes and types are checked by the callers
void product(const MxTensor& x, const MxTensor& w, const Tensor* bias, const Tensor* res, int act, Tensor* y, MxTensor* yq) {
  if (x.rows == 0) return;
  LinArgs a{};
  a.x = x.codes.ptr<uint8_t>();
  a.xs = x.scales.ptr<uint8_t>();
  a.w = w.codes.ptr<uint8_t>();
  a.ws = w.scales.ptr<uint8_t>();
  a.bias = bias ? bias->p : nullptr;
  a.bias_dt = bias ? bias->dt : F32;
  a.res = res ? res->p : nullptr;
  a.N = x.rows;
  a.K = (int)x.cols;
  a.O = (int)w.rows;
  a.act = act;
  a.xrow = (int)mx_row_bytes(x.fmt, x.cols);
  a.wrow = (int)mx_row_bytes(w.fmt, w.cols);
  a.srow = (int)mx_scale_bytes(x.cols);
  if (y) {
    a.out = y->p;
    a.f16 = y->dt == F16;
  } else {
    a.out = yq->codes.p;
    a.outs = yq->scales.ptr<uint8_t>();
    a.osrow = (int)mx_scale_bytes(a.O);
  }
  auto by_out = [&](auto X) {
    constexpr int XB = decltype(X)::value;
    if (!y) yq->fmt == MX_E4M3 ? gemm<XB, OUT_MX8>(a) : gemm<XB, OUT_MX4>(a);
    else if (y->dt == F32) gemm<XB, OUT_F32>(a);
    else gemm<XB, OUT_16>(a);
  };
  x.fmt == MX_E4M3 ? by_out(std::integral_constant<int, 8>{}) : by_out(std::integral_constant<int, 4>{});
}

void check_linear(i64 n, i64 K, const MxTensor& w, const Tensor* bias, const Tensor* res, int act, const Tensor* y, const MxTensor* yq) {
  mx_check(w, "w");
  REQ(w.fmt == MX_E2M1, "w must be e2m1 (format %d)", w.fmt);
  REQ(w.cols == K, "w has %lld columns, x %lld", (long long)w.cols, (long long)K);
  REQ(w.rows > 0 && w.rows % 32 == 0 && w.rows <= (1 << 20), "%lld output channels: a multiple of 32, at most 2^20", (long long)w.rows);
  REQ(act == ACT_NONE || act == ACT_SILU, "act=%d", act);
  REQ((y != nullptr) != (yq != nullptr), "one output");
  if (bias) REQ(bias->numel() == w.rows && bias->p && (bias->dt == F32 || bias->dt == F16 || bias->dt == BF16), "bias must have %lld elements", (long long)w.rows);
  if (y) {
    REQ((y->dt == F32 || y->dt == F16 || y->dt == BF16) && y->dim() == 2 && y->size(0) == n && y->size(1) == w.rows,
        "out must be fp32/fp16/bf16 [%lld,%lld]", (long long)n, (long long)w.rows);
    REQ((uintptr_t)y->p % 16 == 0 && (y->p || n == 0), "out must be 16-byte aligned and not null");
    if (res) {
      REQ(res->dt == y->dt && res->dim() == 2 && res->size(0) == n && res->size(1) == w.rows, "residual must match out");
      REQ((uintptr_t)res->p % 16 == 0 && (res->p || n == 0), "residual must be 16-byte aligned and not null");
      REQ(res->p == y->p || !mx_overlap(res->p, res->bytes(), y->p, y->bytes()), "out must be the residual or apart from it");
    }
  } else {
    mx_check(*yq, "out");
    REQ(yq->rows == n && yq->cols == w.rows, "out must be [%lld,%lld]", (long long)n, (long long)w.rows);
    REQ(!res, "a microscaled output takes no residual");
  }
}
void apart(const void* a, size_t na, const void* b, size_t nb, const char* what) {
  REQ(!mx_overlap(a, na, b, nb), "out must not overlap %s", what);
}
void out_apart(const Tensor* y, const MxTensor* yq, const Tensor& t, const char* what) {
  if (y) apart(y->p, y->bytes(), t.p, t.bytes(), what);
  if (yq) {
    apart(yq->codes.p, yq->codes.bytes(), t.p, t.bytes(), what);
    apart(yq->scales.p, yq->scales.bytes(), t.p, t.bytes(), what);
  }
}
}  // namespace

void mx_linear(const MxTensor& x, const MxTensor& w, const Tensor* bias, const Tensor* residual, int act, Tensor* y, MxTensor* yq) {
  mx_check(x, "x");
  check_linear(x.rows, x.cols, w, bias, residual, act, y, yq);
  for (const Tensor* t : {&x.codes, &x.scales, &w.codes, &w.scales}) out_apart(y, yq, *t, "x or w");
  if (bias) out_apart(y, yq, *bias, "bias");
  product(x, w, bias, residual, act, y, yq);
}

void mx_linear(const Tensor& x, int x_fmt, const MxTensor& w, const Tensor* bias, const Tensor* residual, int act, Tensor* y,
               MxTensor* yq, void* workspace, i64 workspace_bytes) {
  REQ(x.dim() == 2 && (x.dt == F32 || x.dt == F16 || x.dt == BF16), "x must be fp32/fp16/bf16 [N,K]");
  REQ(x_fmt == MX_E4M3 || x_fmt == MX_E2M1, "x_fmt=%d", x_fmt);
  const i64 n = x.size(0), K = x.size(1);
  check_linear(n, K, w, bias, residual, act, y, yq);
  REQ(n < (1ll << 31), "%lld rows", (long long)n);
  REQ((uintptr_t)x.p % 16 == 0 && (x.p || n == 0), "x must be 16-byte aligned and not null");
  out_apart(y, yq, x, "x");
  for (const Tensor* t : {&w.codes, &w.scales}) out_apart(y, yq, *t, "w");
  if (bias) out_apart(y, yq, *bias, "bias");
  if (n == 0) return;
  Workspace ws(workspace, workspace_bytes, mx_linear_workspace(n, K, x_fmt, w.rows));
  MxTensor q = ws.rows(x_fmt, n, K);
  mx_quantize(x, q);
  product(q, w, bias, residual, act, y, yq);
}

i64 mx_linear_workspace(i64 n, i64 K, int x_fmt, i64 O) {
  return n > 0 && K > 0 ? rows_bytes(x_fmt, n, K) : 0;
}

// ---- ConvNeXt tail ----------------------------------------------------------------------------------------------
//   y = x + W2 mx(silu(W1 mx(LayerNorm(h) * gamma + beta) + b1)) + b2
// norm pass, product with the SiLU and the quantisation in its epilogue, product with the residual. Many rows go in
// equal parts whose hidden units stay below kHidBytes, so that they are read back from the 256 MB cache.
namespace {
constexpr i64 kHidBytes = 128ll << 20;
i64 tail_rows(i64 n, i64 C, int fmt) {
  const i64 parts = (n * mx_row_bytes(fmt, 4 * C) + kHidBytes - 1) / kHidBytes;
  return n == 0 ? 0 : std::min(n, ((n + parts - 1) / parts + 255) / 256 * 256);
}
}  // namespace

i64 convnext_mlp_mx_workspace(i64 n, i64 C, int fmt) {
  if (n <= 0 || C <= 0) return 0;
  const i64 m = tail_rows(n, C, fmt);
  return rows_bytes(fmt, m, C) + rows_bytes(fmt, m, 4 * C);
}

void convnext_mlp_mx(const Tensor& h, const Tensor& x, const Tensor* gamma, const Tensor* beta, float eps, const MxTensor& w1,
                     const Tensor* b1, const MxTensor& w2, const Tensor* b2, int fmt, Tensor& y, void* workspace,
                     i64 workspace_bytes) {
  REQ(h.dim() == 2 && (h.dt == BF16 || h.dt == F16), "h must be bf16/fp16 [N,C]");
  const i64 n = h.size(0), C = h.size(1);
  REQ(C > 0 && C % 32 == 0 && C <= 4096, "C=%lld: a multiple of 32, at most 4096", (long long)C);
  REQ(n < (1ll << 31), "%lld rows", (long long)n);
  REQ(fmt == MX_E4M3 || fmt == MX_E2M1, "fmt=%d", fmt);
  mx_check(w1, "w1");
  mx_check(w2, "w2");
  REQ(w1.fmt == MX_E2M1 && w2.fmt == MX_E2M1, "w1 and w2 must be e2m1");
  REQ(w1.rows == 4 * C && w1.cols == C, "w1 must be [4C, C]");
  REQ(w2.rows == C && w2.cols == 4 * C, "w2 must be [C, 4C]");
  REQ(x.dt == h.dt && x.dim() == 2 && x.size(0) == n && x.size(1) == C, "x must match h");
  REQ(y.dt == h.dt && y.dim() == 2 && y.size(0) == n && y.size(1) == C, "y must match h");
  const Tensor* params[4] = {gamma, beta, b1, b2};
  for (int k = 0; k < 4; k++) {
    const Tensor* t = params[k];
    REQ(!t || (t->numel() == (k == 2 ? 4 * C : C) && (t->dt == F32 || t->dt == F16 || t->dt == BF16)), "gamma/beta/b2 must have C elements, b1 4C");
    if (t) out_apart(&y, nullptr, *t, "the parameters");
  }
  if (n == 0) return;
  REQ(h.p && x.p && y.p && ((uintptr_t)h.p | (uintptr_t)x.p | (uintptr_t)y.p) % 16 == 0, "h, x, y must be 16-byte aligned and not null");
  for (const Tensor* t : {&h, &x}) REQ(t->p == y.p || !mx_overlap(t->p, t->bytes(), y.p, y.bytes()), "y must be h, x or apart from both");
  for (const MxTensor* w : {&w1, &w2}) {
    out_apart(&y, nullptr, w->codes, "the weights");
    out_apart(&y, nullptr, w->scales, "the weights");
  }
  const i64 step = tail_rows(n, C, fmt);
  Workspace ws(workspace, workspace_bytes, convnext_mlp_mx_workspace(n, C, fmt));
  const MxTensor a = ws.rows(fmt, step, C), hid = ws.rows(fmt, step, 4 * C);
  auto first = [](const MxTensor& q, i64 m) {
    MxTensor r = q;
    r.rows = m;
    r.codes = borrow(q.codes.p, {m * mx_row_bytes(q.fmt, q.cols)}, U8);
    r.scales = borrow(q.scales.p, {m * mx_scale_bytes(q.cols)}, U8);
    return r;
  };
  for (i64 r0 = 0; r0 < n; r0 += step) {
    const i64 m = std::min(step, n - r0);
    MxTensor am = first(a, m), hm = first(hid, m);
    Tensor ym = y.slice0(r0, r0 + m);
    const Tensor xm = x.slice0(r0, r0 + m);
    add_norm_mx(h.slice0(r0, r0 + m), nullptr, gamma, beta, eps, MX_NORM_LAYER, nullptr, am);
    product(am, w1, b1, nullptr, ACT_SILU, nullptr, &hm);
    product(hm, w2, b2, &xm, ACT_NONE, &ym, nullptr);
  }
}
