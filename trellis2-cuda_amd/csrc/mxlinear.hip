// Linear layers of microscaled rows (mx.h):  y = act(X . W^T + b) + r,  X [N,K] e4m3 or e2m1, W [O,K] e2m1, fp32 sums.
#include "mxgemm.h"

#include <algorithm>

namespace {
__device__ __forceinline__ i32x4 rsrc4(const void* p, uint32_t bytes) {  // a raw buffer's descriptor, in SGPRs
  const uint64_t b = (uint64_t)(uintptr_t)p;
  return i32x4{(int32_t)__builtin_amdgcn_readfirstlane((uint32_t)b), (int32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)),
               (int32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// 16 bytes per lane, global -> LDS: lane l's land at dst + 16 l. Inline assembly, so that the compiler does not put a
// wait for it before every LDS read; the loop below counts them. M0 (dst) needs one wait state between its scalar write
// and the load that reads it, which the compiler does not insert in here.
__device__ __forceinline__ void dma16(i32x4 r, uint32_t lds, uint32_t off, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
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
template <int OUT, int TO>
constexpr int run_tiles() {  // G above
  return OUT == OUT_F32 ? 1 : OUT == OUT_16 ? 2 : 4 < TO ? 4 : TO;
}

// Few rows: W's bytes count, and that many of them are on their way at once. A workgroup of 8 wavefronts has 16 OT channels by 16
// NT rows; each wavefront takes a contiguous eighth of K, both operands straight into registers, and the eight sums meet in
// LDS in a fixed order. XT: x's type (fp32, fp16, bf16), quantised here by every workgroup for itself, which costs less
// than a launch of its own (NT = 1); or -1: x's codes.
// Bound by memory's latency, several times in a row: [1, 4096] by [4096, 4096] (8.9 MB: 1.7 us at the copy rate) 7.8 us as values,
// whose steps wait for their values and quantise them one after another, 5.5 as codes, whose four steps are on their way
// together; [77, 4096] by [8192, 4096] (17.8 MB) 16.8 us: one step at a time, which waits for its scales before its last codes
// are asked for (166 registers with 5 row tiles: one workgroup per CU, which could use 256).
template <int XB, int OUT, int XT, int OT, int NT>
__global__ void __launch_bounds__(512) k_mx_rows(LinArgs a) {
  constexpr bool SPLIT = XB == 8;
  constexpr int G = OUT == OUT_F32 ? 1 : OT;
  __shared__ f32x4 part[8][OT * NT][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S = (a.K + 127) / 128, blocks = a.K / 32, per = (S + 7) / 8;
  const int s0 = wave * per, s1 = min(s0 + per, S);
  const i64 n0 = (i64)blockIdx.y * (16 * NT);
  const int o0 = blockIdx.x * (16 * OT);
  int chan[OT];
#pragma unroll
  for (int t = 0; t < OT; t++) chan[t] = o0 + t / G * (16 * G) + r16 / 4 * (4 * G) + t % G * 4 + r16 % 4;
  f32x4 acc[OT][NT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int u = 0; u < NT; u++) acc[t][u] = f32x4{};
  struct Step {
    mx_u32x4 w[OT];
    int sw[OT], sx[NT];
    XFrag<XB> x[NT];
  };
  // Every load is a buffer load whose offset is past the end where there is nothing (a row past the last, columns past K).
  auto rsrc = [](const void* p, uint32_t bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
  };
  const int rows = (int)min((i64)(16 * NT), a.N - n0);
  constexpr int XS = XT == F32 ? 4 : 2;  // bytes of a value
  const auto rw = rsrc(a.w + (i64)o0 * a.wrow, 16 * OT * a.wrow), rws = rsrc(a.ws + (i64)o0 * a.srow, 16 * OT * a.srow);
  const auto rx = XT < 0 ? rsrc(a.x + n0 * a.xrow, rows * a.xrow) : rsrc(a.x + n0 * a.K * XS, rows * a.K * XS);
  const auto rxs = rsrc(XT < 0 ? a.xs + n0 * a.srow : nullptr, XT < 0 ? rows * a.srow : 0);
  // More row tiles: a load for every scale byte would be a third of the loads, so the scales of four steps come together. (The
  // compiler makes branches of the choice between their words, and waits for the scales ahead of each.)
  mx_u32x4 cw[OT], cx[NT];
  auto load_scales = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < OT; t++) cw[t] = __builtin_amdgcn_raw_buffer_load_b128(rws, (uint32_t)((chan[t] - o0) * a.srow), c * 16, 0);
#pragma unroll
    for (int u = 0; u < NT; u++) cx[u] = __builtin_amdgcn_raw_buffer_load_b128(rxs, (uint32_t)((u * 16 + r16) * a.srow), c * 16, 0);
  };
  auto scale_of = [&](mx_u32x4 q, int s) __attribute__((always_inline)) {  // block 4 s + g's, in byte 0
    const uint32_t w = s % 4 == 0 ? q[0] : s % 4 == 1 ? q[1] : s % 4 == 2 ? q[2] : q[3];
    return (int)(w >> (8 * g));
  };
  auto load = [&](Step& q, int s) __attribute__((always_inline)) {
    const bool in = s * 4 + g < blocks;  // columns past the last: zeros and scale 0
#pragma unroll
    for (int t = 0; t < OT; t++) {
      q.w[t] = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? (uint32_t)((chan[t] - o0) * a.wrow + g * 16) : kOOR, s * 64, 0);
      if constexpr (NT == 1) q.sw[t] = __builtin_amdgcn_raw_buffer_load_b8(rws, in ? (uint32_t)((chan[t] - o0) * a.srow + g) : kOOR, s * 4, 0);
      else q.sw[t] = in ? scale_of(cw[t], s) : 0;
    }
    if constexpr (XT < 0) {
#pragma unroll
      for (int u = 0; u < NT; u++) {
        const uint32_t x = (uint32_t)((u * 16 + r16) * a.xrow + g * 16);
        if constexpr (XB == 8) {  // block g / 2 for the first piece, 2 + g / 2 for the second
          q.x[u].q[0] = __builtin_amdgcn_raw_buffer_load_b128(rx, s * 4 + g / 2 < blocks ? x : kOOR, s * 128, 0);
          q.x[u].q[1] = __builtin_amdgcn_raw_buffer_load_b128(rx, s * 4 + 2 + g / 2 < blocks ? x + 64 : kOOR, s * 128, 0);
        } else {
          q.x[u].q[0] = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? x : kOOR, s * 64, 0);
        }
        if constexpr (NT == 1) q.sx[u] = __builtin_amdgcn_raw_buffer_load_b8(rxs, in ? (uint32_t)((u * 16 + r16) * a.srow + g) : kOOR, s * 4, 0);
        else q.sx[u] = in ? scale_of(cx[u], s) : 0;
      }
    } else {
      static_assert(NT == 1, "quantised once per workgroup");
      float v[32];  // e2m1: block g; e4m3: halves of blocks g / 2 and 2 + g / 2
      mx_u32x4 raw[XT == F32 ? 8 : 4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int c = XB == 4 ? g * 32 + k * 8 : k / 2 * 64 + g * 16 + k % 2 * 8;
        const uint32_t at = s * 128 + c < a.K ? (uint32_t)((r16 * a.K + c) * XS) : kOOR;
        if constexpr (XT == F32) {
          raw[2 * k] = __builtin_amdgcn_raw_buffer_load_b128(rx, at, s * 128 * XS, 0);
          raw[2 * k + 1] = __builtin_amdgcn_raw_buffer_load_b128(rx, at == kOOR ? kOOR : at + 16, s * 128 * XS, 0);
        } else {
          raw[k] = __builtin_amdgcn_raw_buffer_load_b128(rx, at, s * 128 * XS, 0);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float(&o)[8] = *(float(*)[8])&v[k * 8];
        if constexpr (XT == F32) {
#pragma unroll
          for (int j = 0; j < 8; j++) o[j] = __uint_as_float(raw[2 * k + j / 4][j % 4]);
        } else {
          mx_unpack8<XT == F16>(raw[k], o);
        }
      }
      uint32_t top[2];
#pragma unroll
      for (int h = 0; h < 2; h++) top[h] = max(mx_top8(*(float(*)[8])&v[h * 16]), mx_top8(*(float(*)[8])&v[h * 16 + 8]));
      if constexpr (XB == 8) {
        uint32_t byte[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          byte[h] = mx_scale_byte<MX_E4M3>(mx_max_across16(top[h]));
          const float inv = mx_inverse(byte[h]);
          const mx_u32x2 p = mx_encode8<MX_E4M3>(*(float(*)[8])&v[h * 16], inv), r = mx_encode8<MX_E4M3>(*(float(*)[8])&v[h * 16 + 8], inv);
          q.x[0].q[h] = mx_u32x4{p[0], p[1], r[0], r[1]};
        }
        // block g's scale is with lanes 32 (g % 2) + r16 of half g / 2
        const int from = (g & 1) * 32 + r16, b0 = __shfl((int)byte[0], from, 64), b1 = __shfl((int)byte[1], from, 64);
        q.sx[0] = g < 2 ? b0 : b1;
      } else {
        const uint32_t byte = mx_scale_byte<MX_E2M1>(max(top[0], top[1]));
        const float inv = mx_inverse(byte);
#pragma unroll
        for (int k = 0; k < 4; k++) q.x[0].q[0][k] = mx_encode8<MX_E2M1>(*(float(*)[8])&v[k * 8], inv)[0];
        q.sx[0] = (int)byte;
      }
    }
  };
  auto multiply = [&](const Step& q) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; u++) {
      if constexpr (SPLIT) {
        XFrag<8> small = q.x[u], large;
        split(small, large);
#pragma unroll
        for (int t = 0; t < OT; t++) {
          acc[t][u] = mfma<XB, 0, 0>(q.w[t], small, acc[t][u], q.sw[t], q.sx[u]);
          acc[t][u] = mfma<XB, 0, 0>(q.w[t], large, acc[t][u], q.sw[t], q.sx[u]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < OT; t++) acc[t][u] = mfma<XB, 0, 0>(q.w[t], q.x[u], acc[t][u], q.sw[t], q.sx[u]);
      }
    }
  };
  if constexpr (NT == 1) {
    constexpr int U = 4;  // steps loaded at once (codes; the quantisation of values waits within a step)
    int s = s0;
    for (; s + U <= s1; s += U) {
      Step q[U];
#pragma unroll
      for (int k = 0; k < U; k++) load(q[k], s + k);
#pragma unroll
      for (int k = 0; k < U; k++) multiply(q[k]);
    }
    for (; s < s1; s++) {
      Step q;
      load(q, s);
      multiply(q);
    }
  } else {
    for (int s = s0; s < s1; s++) {
      if (s == s0 || s % 4 == 0) load_scales(s / 4);
      Step q;
      load(q, s);
      multiply(q);
    }
  }
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int u = 0; u < NT; u++) part[wave][t * NT + u][lane] = acc[t][u];
  __syncthreads();
  // a wavefront finishes whole runs (G tiles) of the row tiles that fall to it
  constexpr int RUNS = OT / G * NT;
  for (int k = wave; k < RUNS; k += 8) {
    const int t = k / NT * G, u = k % NT;
    float v[4 * G], bias[4 * G];
#pragma unroll
    for (int j = 0; j < G; j++) {
      f32x4 c = part[0][(t + j) * NT + u][lane];
#pragma unroll
      for (int w = 1; w < 8; w++) c += part[w][(t + j) * NT + u][lane];
#pragma unroll
      for (int i = 0; i < 4; i++) v[j * 4 + i] = c[i];
    }
    const i64 n = n0 + u * 16 + r16;
    const int o = o0 + t / G * (16 * G) + g * (4 * G);
    mx_params<4 * G>(a.bias, a.bias_dt, o, 0.f, bias);
    uint32_t r[4] = {};
    if (a.res) load_residual<OUT, 4 * G>(a, n, o, n < a.N, r);
    finish<OUT>(a, n, o, v, bias, r, n < a.N);
  }
}

// Tiled product. A workgroup of WO x WN wavefronts has BO = 16 TO WO channels by BN = 16 TN WN rows; K goes by steps of
// 128, KS of them a stage, through NS slots of LDS, filled by DMA; the scales go by 512 columns (16 bytes a row), one slot. LDS rows are 64
// or 128 bytes of a stage (e2m1: of one or two steps, e4m3: of one), their 16-byte pieces permuted (piece c of row q at
// c ^ (q >> 1) % 4 or c ^ q % 8), so that eight lanes of neighbouring rows read from distinct banks.
//
// A step's products go in four quarters, halves of W's channel tiles by halves of X's row tiles, in the order (0, f), (0, 1 - f),
// (1, 1 - f), (1, f) with f = 0, 1 in turn: each quarter changes one operand's half, whose registers were free a quarter
// earlier, so every LDS read is issued one quarter before its use and a wavefront holds one step's operands only. In the
// middle all wavefronts meet: by then each has read the whole slot, so it is filled again at once. One barrier a stage,
// and NS - 1/2 stages for a DMA to land.
//
// Measured: [16411, 4096] by [4096, 4096] with a residual, 551 GFLOP, e2m1 235 us (2.3 PFLOP/s), e4m3 272. The DMA path bounds
// both (44 KB/us into a CU beside the products of e4m3, 53 of e2m1; alone 60 to 80 in segments of 64 bytes and 125 of 128, the
// reason for two steps of e2m1 a stage at 128 x 128), then the residual and the stores, which add their time at the copy rate.
//
// SPLIT (e4m3): the matrix unit adds eight neighbouring products at a time and drops what is below 2^-13 of the largest (of
// two to the sum of its factors' exponents). Taken for the elements of magnitude 4 and more and for the smaller ones apart,
// each step's products are exact: with e2m1 factors, of exponents -1 to 2, the ones span exponents 10 to -2, the others 3 to -10.
// That doubles the matrix work, so here it is done where the loss shows: fp32 results, and microscaled ones (an error that
// moves a value over a border between elements costs a whole step). A result of 16 bits is summed without it: off by 5e-6 of
// the results' root mean square on normal values, 4e-5 where one of eight is 60 times the others (worst 2e-4), without a
// bias, for K from 512 to 262144; fp16 itself rounds by up to 5e-4. With it [16411, 4096, 4096] 276 -> 415 us, [8209, 2080, 4128]
// 104 -> 140, [11467, 2048, 512] 21 -> 29. k_mx_rows always does it: 5.1 -> 5.4 us with one row, 16.0 -> 17.0 with 77.
template <int XB, int OUT, int TO, int TN, int WO, int WN, int KS, int NS>
__global__ void __launch_bounds__(64 * WO * WN, 2) k_mx_gemm(LinArgs a) {
  constexpr int NW = WO * WN, BO = 16 * TO * WO, BN = 16 * TN * WN, H = TO / 2, HX = TN / 2;
  constexpr bool SPLIT = XB == 8 && OUT != OUT_16;
  constexpr int XR = XB * 16 * KS, WR = 64 * KS;                                // bytes of a row of X and W per stage
  constexpr int XP = XR / 16, WP = WR / 16;                                     // 16-byte pieces of them
  constexpr int XI = BN * XR / 1024 / NW, WI = BO * WR / 1024 / NW, ST = (BO + BN) / 64, SI = (ST + NW - 1) / NW;  // DMAs per wavefront
  static_assert(XI * 1024 * NW == BN * XR && WI * 1024 * NW == BO * WR && BO % 64 == 0 && BN % 64 == 0, "whole DMAs");
  static_assert((XR == 64 || XR == 128) && (WR == 64 || WR == 128), "swizzles");
  constexpr int G = run_tiles<OUT, TO>();
  static_assert(TO % G == 0 && TO % 2 == 0 && TN % 2 == 0 && NS >= 2 && NS <= 4, "whole runs, two halves");
  __shared__ __attribute__((aligned(16))) mx_u32x4 lds[NS * (BN * XR + BO * WR) / 16 + (BO + BN)];
  constexpr uint32_t kSlot = BN * XR + BO * WR, kScales = NS * kSlot;

  // Whole tiles first, then those that the last rows or channels end in (they skip the products of what they lack): each
  // XCD takes a contiguous range of either, whole tiles in bands of `band` columns, row by row within a band.
  const int fn = (int)(a.N / BN), fo = a.O / BO, xcd = blockIdx.x % 8, k = blockIdx.x / 8;
  int tn, to;
  if (k < a.per) {
    const int l = xcd * a.per + k;
    if (l >= fn * fo) return;
    const int first = l / (a.band * fn) * a.band, width = min(a.band, fo - first), inside = l - first * fn;
    tn = inside / width;
    to = first + inside % width;
  } else {
    const int l = xcd * a.per_rest + k - a.per, below = (a.tiles_n - fn) * a.tiles_o;
    if (l >= below + (a.tiles_o - fo) * fn) return;
    tn = l < below ? fn : l - below;
    to = l < below ? l : fo;
  }
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wo = wave % WO, wn = wave / WO;
  const int S = (a.K + 127) / 128, stages = (S + KS - 1) / KS, blocks = a.K / 32;
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
  // where piece c of a row lies in the row's place in LDS, and (an involution) the piece that lies there
  auto place = [](auto PC, int row, int c) __attribute__((always_inline)) {
    return decltype(PC)::value == 8 ? c ^ (row & 7) : c ^ (row >> 1 & 3);
  };
  constexpr std::integral_constant<int, XP> XPC{};
  constexpr std::integral_constant<int, WP> WPC{};
  uint32_t xoff[XI], woff[WI], soff[SI];
#pragma unroll
  for (int k = 0; k < XI; k++) {
    const int p = (wave * XI + k) * 64 + lane, q = p / XP;
    xoff[k] = q < rows ? (uint32_t)(q * a.xrow + place(XPC, q, p % XP) * 16) : kOOR;
  }
#pragma unroll
  for (int k = 0; k < WI; k++) {
    const int p = (wave * WI + k) * 64 + lane, q = p / WP, ch = channel(q);
    woff[k] = ch < chans ? (uint32_t)(ch * a.wrow + place(WPC, q, p % WP) * 16) : kOOR;
  }
#pragma unroll
  for (int k = 0; k < SI; k++) {
    const int p = (k * NW + wave) * 64 + lane, ch = channel(p < BO ? p : 0);
    soff[k] = p < BO ? (ch < chans ? (uint32_t)(ch * a.srow) : kOOR) : p - BO < rows ? (uint32_t)((p - BO) * a.srow) : kOOR;
  }
  auto none_unless = [](i32x4 r, bool live) __attribute__((always_inline)) {
    r[2] = live ? r[2] : 0;
    return r;
  };
  auto issue_scales = [&](int c) __attribute__((always_inline)) {  // of columns 512 c .., past the last one nothing
    const bool live = c * 4 < S;
#pragma unroll
    for (int k = 0; k < SI; k++) {
      const int p0 = (k * NW + wave) * 64;  // BO is a multiple of 64: a DMA's rows are all W's or all X's
      if (p0 >= BO + BN) break;             // (the waits count ST / NW of them, which every wavefront has)
      dma16(none_unless(p0 < BO ? rws : rxs, live), lds0 + kScales + p0 * 16, soff[k], live ? c * 16 : 0);
    }
  };
  // fills stage t's slot; past the last one the DMAs still run (the waits count them) but read nothing
  auto issue = [&](int t, int slot) __attribute__((always_inline)) {
    const bool live = t < stages;
    const i32x4 fx = none_unless(rx, live), fw = none_unless(rw, live);
    const int xs = live ? t * XR : 0, ws = live ? t * WR : 0;
    const uint32_t at = lds0 + slot * kSlot;
    if (live && (t + 1) * (KS * 128) > a.K) {
      // the last stage ends inside its columns: pieces past them read as zeros. (Their places are computed here, from a
      // copy of the lane that the compiler cannot see through: kept in registers over the loop they would spill.)
      int l = lane;
      asm volatile("" : "+v"(l));
      const int xleft = a.xrow - xs, wleft = a.wrow - ws;
#pragma unroll
      for (int k = 0; k < XI; k++) {
        const int p = (wave * XI + k) * 64 + l;
        dma16(fx, at + (wave * XI + k) * 1024, place(XPC, p / XP, p % XP) * 16 < xleft ? xoff[k] : kOOR, xs);
      }
#pragma unroll
      for (int k = 0; k < WI; k++) {
        const int p = (wave * WI + k) * 64 + l;
        dma16(fw, at + BN * XR + (wave * WI + k) * 1024, place(WPC, p / WP, p % WP) * 16 < wleft ? woff[k] : kOOR, ws);
      }
    } else {
#pragma unroll
      for (int k = 0; k < XI; k++) dma16(fx, at + (wave * XI + k) * 1024, xoff[k], xs);
#pragma unroll
      for (int k = 0; k < WI; k++) dma16(fw, at + BN * XR + (wave * WI + k) * 1024, woff[k], ws);
    }
  };

  f32x4 acc[TO][TN];
#pragma unroll
  for (int t = 0; t < TO; t++)
#pragma unroll
    for (int u = 0; u < TN; u++) acc[t][u] = f32x4{};

  // where this lane reads, in 16-byte units of a slot: pieces of sub-step j
  const int xq = wn * (16 * TN) + r16, wp = wo * (16 * TO) + r16;
  auto xat = [&](int c) __attribute__((always_inline)) { return xq * XP + place(XPC, r16, c); };
  auto wat = [&](int c) __attribute__((always_inline)) { return BN * XP + wp * WP + place(WPC, r16, c); };
  int xa[XB == 8 ? 2 : KS], wa[KS];  // e4m3: its two pieces (KS = 1); e2m1: one per sub-step
#pragma unroll
  for (int j = 0; j < (XB == 8 ? 2 : KS); j++) xa[j] = xat(4 * j + g);
#pragma unroll
  for (int j = 0; j < KS; j++) wa[j] = wat(4 * j + g);
  static_assert(XB == 4 || KS == 1, "e4m3 rows are 128 bytes a step");
  XFrag<XB> fx[2][HX];
  mx_u32x4 fw[2][H];
  int sx[TN], sw[TO];  // scales of four steps: byte i is step i's
  auto read_x = [&](XFrag<XB>(&f)[HX], int slot, int j, int half) __attribute__((always_inline)) {
    const mx_u32x4* l = lds + slot * (kSlot / 16) + half * (HX * 16 * XP);
#pragma unroll
    for (int u = 0; u < HX; u++) {
      f[u].q[0] = l[xa[XB == 8 ? 0 : j] + u * (16 * XP)];
      if constexpr (XB == 8) f[u].q[1] = l[xa[1] + u * (16 * XP)];
    }
  };
  auto read_w = [&](mx_u32x4(&f)[H], int slot, int j, int half) __attribute__((always_inline)) {
    const mx_u32x4* l = lds + slot * (kSlot / 16) + wa[j] + half * (H * 16 * WP);
#pragma unroll
    for (int t = 0; t < H; t++) f[t] = l[t * (16 * WP)];
  };
  const uint32_t pick = (uint32_t)g * 0x0101u + 0x0400u;  // bytes g of two words, the second operand's first
  auto read_scales = [&](int c) __attribute__((always_inline)) {
    const mx_u32x4* l = lds + kScales / 16;
    auto gather = [&](mx_u32x4 q) __attribute__((always_inline)) {
      const uint32_t lo = __builtin_amdgcn_perm(q[1], q[0], pick), hi = __builtin_amdgcn_perm(q[3], q[2], pick);
      return (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
    };
#pragma unroll
    for (int t = 0; t < TO; t++) {
      sw[t] = gather(l[wp + t * 16]);
      if (t % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // few words at a time: the registers are short
    }
#pragma unroll
    for (int u = 0; u < TN; u++) {
      sx[u] = gather(l[BO + xq + u * 16]);
      if (u % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (c * 16 + 16 > blocks) {  // the padding behind a row's last scale is not read as a scale
      uint32_t keep = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) keep |= c * 16 + i * 4 + g < blocks ? 0xffu << (8 * i) : 0u;
#pragma unroll
      for (int t = 0; t < TO; t++) sw[t] &= keep;
#pragma unroll
      for (int u = 0; u < TN; u++) sx[u] &= keep;
    }
  };

  issue_scales(0);
#pragma unroll
  for (int t = 0; t < NS; t++) issue(t, t);
  wait_vm<(NS - 1) * (XI + WI)>();
  bare_barrier();
  read_x(fx[0], 0, 0, 0);
  read_w(fw[0], 0, 0, 0);
  read_scales(0);
  // which halves of this wavefront's part hold anything (a run of channels may lie across W's halves: then both or none)
  const bool xl[2] = {wn * (16 * TN) < rows, wn * (16 * TN) + 16 * HX < rows};
  const bool wl[2] = {wo * (16 * TO) < chans, wo * (16 * TO) + (H % G == 0 ? 16 * H : 0) < chans};
  int cur = 0;
  auto step = [&](auto IC, int s) __attribute__((always_inline)) {
    constexpr int I = decltype(IC)::value, J = I % KS, JN = (I + 1) % KS;  // sub-step of this and of the next one
    constexpr int f = I & 1;
    XFrag<XB> large[SPLIT ? 2 : 1][SPLIT ? HX : 1];
    auto take_apart = [&](auto XC) __attribute__((always_inline)) {
      constexpr int hx = decltype(XC)::value;
      if constexpr (SPLIT) {
#pragma unroll
        for (int u = 0; u < HX; u++) split(fx[hx][u], large[hx][u]);
      }
    };
    auto quarter = [&](auto WC, auto XC) __attribute__((always_inline)) {
      constexpr int hw = decltype(WC)::value, hx = decltype(XC)::value;
      if (!(xl[hx] && wl[hw])) return;
#pragma unroll
      for (int u = 0; u < HX; u++)
#pragma unroll
        for (int t = 0; t < H; t++) {
          f32x4& c = acc[hw * H + t][hx * HX + u];
          c = mfma<XB, I, I>(fw[hw][t], fx[hx][u], c, sw[hw * H + t], sx[hx * HX + u]);
          if constexpr (SPLIT) c = mfma<XB, I, I>(fw[hw][t], large[hx][u], c, sw[hw * H + t], sx[hx * HX + u]);
        }
    };
    constexpr std::integral_constant<int, 0> first{};
    constexpr std::integral_constant<int, 1> second{};
    constexpr std::integral_constant<int, f> xf{};
    constexpr std::integral_constant<int, 1 - f> xo{};
    read_x(fx[1 - f], cur, J, 1 - f);
    read_w(fw[1], cur, J, 1);
    take_apart(xf);
    quarter(first, xf);
    __builtin_amdgcn_sched_barrier(0);
    take_apart(xo);
    quarter(first, xo);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (JN == 0) {
      // The next stage has landed (the NS - 2 after it may be on their way, and scales issued with them), and this one is
      // in registers. The scales of the next four steps are asked for at the first meeting after all have read those of
      // these four; they are older than the stage that the last meeting of the four waits for.
      constexpr auto with_scales = [](int back) { return ((I - back * KS) & 3) == KS - 1; };
      wait_vm<(NS - 2) * (XI + WI) + ST / NW * ((NS > 2 && with_scales(1)) + (NS > 3 && with_scales(2)))>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      bare_barrier();
      if constexpr (I == KS - 1) issue_scales(s / 4 + 1);
      issue(s / KS + NS, cur);
      cur = cur + 1 == NS ? 0 : cur + 1;
    }
    read_w(fw[0], cur, JN, 0);
    quarter(second, xo);
    __builtin_amdgcn_sched_barrier(0);
    read_x(fx[1 - f], cur, JN, 1 - f);
    quarter(second, xf);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (I == 3) read_scales(s / 4 + 1);
  };
  for (int s = 0; s < S; s += 4) {
    step(std::integral_constant<int, 0>{}, s);
    if (s + 1 < S) step(std::integral_constant<int, 1>{}, s + 1);
    if (s + 2 < S) step(std::integral_constant<int, 2>{}, s + 2);
    if (s + 3 < S) step(std::integral_constant<int, 3>{}, s + 3);
  }
  wait_vm<0>();  // nothing lands in LDS after the workgroup has gone

  // The residual's loads go out together (a wavefront that waited for each in turn would spend the epilogue on latency):
  // of all runs for 16 bits, whose words fit where the operands were, else of one run's rows.
  constexpr bool RES = OUT == OUT_16 || OUT == OUT_F32;
  constexpr int RUNS = TO / G, AHEAD = OUT == OUT_16 ? RUNS : 1;
  uint32_t res[RES ? AHEAD : 1][RES ? TN : 1][4];
  auto channel_of = [&](int run) __attribute__((always_inline)) { return o0 + wo * (16 * TO) + run * (16 * G) + g * (4 * G); };
  auto load_run = [&](uint32_t(&r)[RES ? TN : 1][4], int run) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < TN; u++) {
      const i64 n = n0 + xq + u * 16;
      load_residual<OUT, 4 * G>(a, n, channel_of(run), n < a.N && channel_of(run) < a.O, r[u]);
    }
  };
  if constexpr (RES && AHEAD > 1) {
    if (a.res) {
#pragma unroll
      for (int run = 0; run < RUNS; run++) load_run(res[run], run);
    }
  }
#pragma unroll
  for (int run = 0; run < RUNS; run++) {
    const int o = channel_of(run);
    if constexpr (RES && AHEAD == 1) {
      if (a.res) load_run(res[0], run);
    }
    float bias[4 * G];
    mx_params<4 * G>(o < a.O ? a.bias : nullptr, a.bias_dt, o, 0.f, bias);
#pragma unroll
    for (int u = 0; u < TN; u++) {
      const i64 n = n0 + xq + u * 16;
      float v[4 * G];
#pragma unroll
      for (int j = 0; j < G; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) v[j * 4 + i] = acc[run * G + j][u][i];
      uint32_t none[4] = {};
      if constexpr (RES) finish<OUT>(a, n, o, v, bias, res[AHEAD > 1 ? run : 0][u], n < a.N && o < a.O);
      else finish<OUT>(a, n, o, v, bias, none, n < a.N && o < a.O);
    }
  }
}

template <int XB, int OUT, int TO, int TN, int WO, int WN, int KS, int NS>
void launch(LinArgs a) {
  constexpr int BO = 16 * TO * WO, BN = 16 * TN * WN;
  const i64 tn = (a.N + BN - 1) / BN, to = (a.O + BO - 1) / BO;
  REQ(tn * to <= (1ll << 24) - 16, "%lld rows by %d channels: more than 2^24 tiles", (long long)a.N, a.O);  // 2^32 threads a launch
  a.tiles_n = (int)tn;
  a.tiles_o = (int)to;
  const i64 whole = a.N / BN * (a.O / BO);
  a.per = cdiv(whole, 8);
  a.per_rest = cdiv(tn * to - whole, 8);
  a.band = 4;
  k_mx_gemm<XB, OUT, TO, TN, WO, WN, KS, NS><<<(a.per + a.per_rest) * 8, 64 * WO * WN, 0, stream()>>>(a);
  CK(hipGetLastError());
}

constexpr int kValueRows = 16, kFewRows = 128;  // rows that may come as values; rows up to which k_mx_rows is looked at
}  // namespace

// Few rows: k_mx_rows, 32 channels a workgroup (16 of values of up to 16 rows), in groups of the fewest row tiles whose
// workgroups are one round of the CUs: a workgroup's time grows with its row tiles, a second round doubles it. us with 2 / 3 / 4 /
// 5 / 6 / 8 row tiles / whole tiles of 128 x 64, e4m3 to 16 bits, [N, K, O]: [64, 4096, 4096] 10.0 / 12.0 / 13.8 / - / - / - / 16.6,
// [80, 4096, 4096] 15.1 / 12.0 / 14.1 / 16.1 / - / - / 16.3, [128, 4096, 4096] 16.9 / 19.2 / 14.2 / 16.4 / 18.4 / 22.8 / 16.8,
// [40, 4096, 8192] 14.5 / 11.5 / 12.3 / - / - / - / 16.3, [80, 4096, 8192] 21.6 / 19.2 / 21.3 / 16.1 / 17.3 / - / 16.5, [96, 4096, 8192]
// 22.9 / 20.5 / 22.3 / 25.6 / 18.6 / - / 16.5: more than 5 row tiles are the tiled kernel's. With e2m1, and where that kernel takes
// its products twice (SPLIT), they are not: e2m1 [128, 4096, 8192] 22.1 / 19.9 / 17.2 / 18.1 / 20.0 / 15.3 / 16.0, e4m3 to e4m3
// 30.1 / 27.9 / 25.4 / 27.5 / 29.4 / 23.8 / 25.3. Two rounds only with up to 32 rows: [24, 4096, 16384] 15.8 / 17.6 / - / - / - / - /
// 16.9, but [40, 4096, 16384] 25.8 / 19.8 / 21.7 / - / - / - / 16.7. (K in pieces over more workgroups, whose sums a second launch adds:
// [33, 4096, 4096] 12 us, [20, 1024, 4096] 14, against 9.6 and 4.6.)
// More rows: larger tiles read fewer operand bytes per product, smaller ones are more. Two workgroups of 256 channels by 128 rows
// fit a CU: they are taken where they fill most of these slots; 128 by 64 where 128 by 128 would leave a quarter of them free.
// us at 256 x 128 / 128 x 128 / 128 x 64, [N, K, O]: e4m3 [16411, 4096, 4096] 272 / 314 / 365, [8209, 2080, 4128] 94 / 103 / 114,
// [58321, 1024, 256] 29 / 32 / 32, [2048, 4096, 4096] 44 / 41 / 46, [1803, 4096, 1024] 41 / 26 / 18, [11467, 2048, 512] 28 / 23 / 21,
// [300, 1024, 1024] 20 / 12 / 9; e2m1 [16411, 4096, 4096] 236 / 242 / 306, [600, 2048, 2048] 23 / 15 / 12.
MxTile mx_linear_tile(i64 n, i64 o, int x_fmt, bool out16) {
  const i64 cus = mx_device_cus();
  if (n <= 16) return {16, 32};
  if (n <= kFewRows) {
    for (int t : {2, 3, 4, 5, 6, 8}) {
      if (t > 5 && x_fmt == MX_E4M3 && out16) break;
      if (cdiv(n, 16 * t) * (o / 32) <= cus || (n <= 32 && o / 32 <= 2 * cus)) return {16 * t, 32};
    }
  }
  const i64 n128 = cdiv(n, 128);
  if (n128 * cdiv(o, 256) * 2 >= 3 * cus) return {128, 256};
  if (n128 * cdiv(o, 128) * 2 > 3 * cus) return {128, 128};
  return {64, 128};
}

namespace {
template <int XB, int OUT, int XT, int NT>
void launch_rows(const LinArgs& a) {
  constexpr int OT = OUT == OUT_MX8 || OUT == OUT_MX4 ? 2 : NT == 1 ? 1 : 2;
  const dim3 grid(a.O / (16 * OT), (unsigned)((a.N + 16 * NT - 1) / (16 * NT)));
  k_mx_rows<XB, OUT, XT, OT, NT><<<grid, 512, 0, stream()>>>(a);
  CK(hipGetLastError());
}
template <int XB, int OUT>
void gemm(const LinArgs& a, int xt) {
  if (xt >= 0) {
    if (xt == F32) launch_rows<XB, OUT, F32, 1>(a);
    else if (xt == F16) launch_rows<XB, OUT, F16, 1>(a);
    else launch_rows<XB, OUT, BF16, 1>(a);
    return;
  }
  const MxTile t = mx_linear_tile(a.N, a.O, XB == 8 ? MX_E4M3 : MX_E2M1, OUT == OUT_16);
  if (t.channels <= 32) {
    switch (t.rows / 16) {
      case 1: return launch_rows<XB, OUT, -1, 1>(a);
      case 2: return launch_rows<XB, OUT, -1, 2>(a);
      case 3: return launch_rows<XB, OUT, -1, 3>(a);
      case 4: return launch_rows<XB, OUT, -1, 4>(a);
      case 5: return launch_rows<XB, OUT, -1, 5>(a);
    }
    if constexpr (XB == 4 || OUT != OUT_16) {
      if (t.rows == 96) return launch_rows<XB, OUT, -1, 6>(a);
      if (t.rows == 128) return launch_rows<XB, OUT, -1, 8>(a);
    }
    spc_fail("no kernel for %d rows", t.rows);
  }
  if (t.channels == 256) launch<XB, OUT, 8, 4, 2, 2, 1, XB == 8 ? 2 : 3>(a);
  else if (t.rows == 128) launch<XB, OUT, 4, 4, 2, 2, XB == 8 ? 1 : 2, XB == 8 ? 3 : 2>(a);
  else launch<XB, OUT, 4, 2, 2, 2, 1, 3>(a);
}
}  // namespace

// xv: x's values (at most 16 rows), which the product quantises to x's format itself; else x's codes
void mx_product(const MxTensor& x, const MxTensor& w, const Tensor* bias, const Tensor* res, int act, Tensor* y, MxTensor* yq,
                const Tensor* xv) {
  if (x.rows == 0) return;
  LinArgs a{};
  a.x = xv ? xv->ptr<uint8_t>() : x.codes.ptr<uint8_t>();
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
    const int xt = xv ? (int)xv->dt : -1;
    if (!y) yq->fmt == MX_E4M3 ? gemm<XB, OUT_MX8>(a, xt) : gemm<XB, OUT_MX4>(a, xt);
    else if (y->dt == F32) gemm<XB, OUT_F32>(a, xt);
    else gemm<XB, OUT_16>(a, xt);
  };
  x.fmt == MX_E4M3 ? by_out(std::integral_constant<int, 8>{}) : by_out(std::integral_constant<int, 4>{});
}

namespace {
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
    mx_check_apart(*yq, "out");
    REQ(yq->rows == n && yq->cols == w.rows, "out must be [%lld,%lld]", (long long)n, (long long)w.rows);
    REQ(!res, "a microscaled output takes no residual");
  }
}
}  // namespace

i64 mx_linear_workspace(i64 n, i64 K, int x_fmt) { return n > kValueRows && K > 0 ? mx_rows_bytes(x_fmt, n, K) : 0; }

void mx_linear(const MxTensor& x, const MxTensor& w, const Tensor* bias, const Tensor* residual, int act, Tensor* y, MxTensor* yq) {
  mx_check(x, "x");
  check_linear(x.rows, x.cols, w, bias, residual, act, y, yq);
  for (const Tensor* t : {&x.codes, &x.scales, &w.codes, &w.scales}) mx_out_apart(y, yq, *t, "x or w");
  if (bias) mx_out_apart(y, yq, *bias, "bias");
  mx_product(x, w, bias, residual, act, y, yq);
}

void mx_linear(const Tensor& x, int x_fmt, const MxTensor& w, const Tensor* bias, const Tensor* residual, int act, Tensor* y,
               MxTensor* yq, void* workspace, i64 workspace_bytes) {
  REQ(x.dim() == 2 && (x.dt == F32 || x.dt == F16 || x.dt == BF16), "x must be fp32/fp16/bf16 [N,K]");
  REQ(x_fmt == MX_E4M3 || x_fmt == MX_E2M1, "x_fmt=%d", x_fmt);
  const i64 n = x.size(0), K = x.size(1);
  check_linear(n, K, w, bias, residual, act, y, yq);
  REQ(n < (1ll << 31), "%lld rows", (long long)n);
  REQ((uintptr_t)x.p % 16 == 0 && (x.p || n == 0), "x must be 16-byte aligned and not null");
  mx_out_apart(y, yq, x, "x");
  for (const Tensor* t : {&w.codes, &w.scales}) mx_out_apart(y, yq, *t, "w");
  if (bias) mx_out_apart(y, yq, *bias, "bias");
  if (n == 0) return;
  const i64 need = mx_linear_workspace(n, K, x_fmt);
  if (workspace) {
    const Tensor room = borrow(workspace, {need}, U8);
    mx_out_apart(y, yq, room, "the workspace");
    for (const Tensor* t : {&x, &w.codes, &w.scales, bias, residual})
      if (t) mx_apart(t->p, t->bytes(), room.p, room.bytes(), "the workspace");
  }
  MxWorkspace ws(workspace, workspace_bytes, need);
  if (n <= kValueRows) {
    MxTensor q;
    q.fmt = x_fmt;
    q.rows = n;
    q.cols = K;
    return mx_product(q, w, bias, residual, act, y, yq, &x);
  }
  MxTensor q = ws.rows(x_fmt, n, K);
  mx_quantize(x, q);
  mx_product(q, w, bias, residual, act, y, yq);
}
