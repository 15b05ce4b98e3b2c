// ConvNeXt tail with microscaled products (beside mlp.hip's, whose products are in 16 bits):
//   y = x + W2 q(silu(W1 q(LayerNorm(h) * gamma + beta) + b1)) + b2,    q: blocks of e4m3 or e2m1 (mx.h), W1, W2 e2m1
//
// C = 128 and 256 with e4m3 activations and enough rows run in one kernel (k_mx_tail): the hidden units, which are what the
// three-pass form writes and reads most of, stay in LDS. Other widths and formats, and fewer rows, run as norm pass, product with the
// SiLU and the quantisation in its epilogue, product with the residual. The two forms give the same bits.
#include <algorithm>

#include "mxgemm.h"

namespace {
struct TailArgs {
  const uint16_t* h;
  const uint8_t *w1, *s1, *w2, *s2;
  const void *gamma, *beta, *b1;
  int gdt, bdt, b1dt;
  float eps;
  LinArgs out;  // the epilogue's: bias b2, residual x, y, N, O = C
};

// A workgroup of 8 wavefronts has 64 rows. It normalises and quantises them into LDS, already taken apart into elements of
// magnitude 4 and more and smaller ones (the first product is summed exactly: its results are quantised again). Then,
// 256 hidden units at a time: a wavefront computes 32 of them for all rows (one block of 32 per row: its largest magnitude
// is two lane exchanges away), SiLU, quantises them into LDS, and after a barrier multiplies all 256 into its C / 8
// channels of y. The weights go from L2 straight into registers, each to the one wavefront that needs it, read while
// the other product runs. Two slots of hidden units make it one barrier a round.
// us by graph replays, this kernel / three passes / the 16-bit tail: [15000, 256] 29 / 37 / 47, [58321, 256] 87 / 116 / 126, [391007, 128]
// 181 / 306 / 218. 61 GFLOP at the second size: with parts left out, about 20 us were norm, residual and stores, 27 the two products,
// 12 waits for weights, 6 SiLU and quantisation; the rest is their order in every wavefront, one after another. At 512 channels
// the sums of y leave room for 32 rows only, and each workgroup reads all weights for them: [11467, 512] 84 us with 8 wavefronts,
// 128 with 4, against 63 in three passes.
constexpr int kTailRows = 64;  // rows of a workgroup
template <bool F16, int C>
__global__ void __launch_bounds__(512, 4) k_mx_tail(TailArgs a) {
  constexpr int BN = kTailRows, S1 = C / 128, ROUNDS = C / 64, OT = C / 128, G = OT == 1 ? 1 : 2;
  constexpr int U = BN / 16, R1 = C / 2, R2 = 2 * C;         // row tiles; bytes of W1's and W2's rows
  constexpr int SR2 = C / 8;                                 // of W2's scale rows (W1's: 16)
  constexpr int LPR = C / 8, PASS = 512 / LPR;               // lanes of a row, rows of a pass
  __shared__ __attribute__((aligned(16))) mx_u32x4 xl[2][S1][BN * 8], hid[2][2][BN * 8];  // small, large; slots, steps
  __shared__ __attribute__((aligned(16))) float b1l[4 * C];
  __shared__ __attribute__((aligned(16))) uint8_t xsc[BN * S1 * 4], hsc[2][BN * 8];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const i64 n0 = (i64)blockIdx.x * BN;
  const int rows = (int)min((i64)BN, a.out.N - n0);
  auto rsrc = [](const void* p, uint32_t bytes) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
  };
  const auto rw1 = rsrc(a.w1, 4 * C * R1), rw2 = rsrc(a.w2, C * R2), rs1 = rsrc(a.s1, 4 * C * 16), rs2 = rsrc(a.s2, C * SR2);

  // This lane's row of W1 (of hidden unit round * 256 + ...) and of W2 in tile 0; tile t's is a constant number of rows on, and
  // steps and rounds go into the loads' scalar offset.
  const uint32_t c1 = (uint32_t)(wave * 32 + r16 / 4 * 8 + r16 % 4), c2 = (uint32_t)(wave * (16 * OT) + r16 / 4 * (4 * G) + r16 % 4);
  const uint32_t o1 = c1 * R1 + g * 16, os1 = c1 * 16, o2 = c2 * R2 + g * 16, os2 = c2 * SR2;
  mx_u32x4 w1[2][S1], w2[OT][2];
  uint32_t s1[2][S1], s2[OT][2];  // four blocks' scales each
  auto load1 = [&](int round) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int s = 0; s < S1; s++) {
        w1[t][s] = __builtin_amdgcn_raw_buffer_load_b128(rw1, o1, (round * 256 + t * 4) * R1 + s * 64, 0);
        s1[t][s] = __builtin_amdgcn_raw_buffer_load_b32(rs1, os1, (round * 256 + t * 4) * 16 + s * 4, 0);
      }
  };
  auto load2 = [&](int round) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < OT; t++)
#pragma unroll
      for (int s = 0; s < 2; s++) {
        w2[t][s] = __builtin_amdgcn_raw_buffer_load_b128(rw2, o2, (t / G * (16 * G) + t % G * 4) * R2 + round * 128 + s * 64, 0);
        s2[t][s] = __builtin_amdgcn_raw_buffer_load_b32(rs2, os2, (t / G * (16 * G) + t % G * 4) * SR2 + round * 8 + s * 4, 0);
      }
  };

  load1(0);
  {
    const auto rh = rsrc(a.h + n0 * C, rows * C * 2);
    const int sub = tid % LPR;
    mx_u32x4 q[BN / PASS];
#pragma unroll
    for (int p = 0; p < BN / PASS; p++) q[p] = __builtin_amdgcn_raw_buffer_load_b128(rh, (uint32_t)(((p * PASS + tid / LPR) * C + sub * 8) * 2), 0, 0);
    float gam[8], bet[8];
    mx_params<8>(a.gamma, a.gdt, sub * 8, 1.f, gam);
    mx_params<8>(a.beta, a.bdt, sub * 8, 0.f, bet);
#pragma unroll
    for (int k = 0; k < 4 * C / 512; k++) {
      float b[1];
      mx_params<1>(a.b1, a.b1dt, k * 512 + tid, 0.f, b);
      b1l[k * 512 + tid] = b[0];
    }
#pragma unroll
    for (int p = 0; p < BN / PASS; p++) {
      const int row = p * PASS + tid / LPR;
      float v[1][8], o[8];
      mx_unpack8<F16>(q[p], v[0]);
      float mean, rstd;
      mx_row_stats<LPR, 1>(v, sub, LPR, (float)C, 1.f / (float)C, a.eps, true, mean, rstd, [](float s) { return s; });
      mx_norm8(v[0], mean, rstd, gam, bet, o);
      const uint32_t byte = mx_scale_byte<MX_E4M3>(mx_quad_max(mx_top8(o)));
      const mx_u32x2 e = mx_encode8<MX_E4M3>(o, mx_inverse(byte)), large = {e4m3_large(e[0]), e4m3_large(e[1])};
      const int at = (row * 8 + (sub % 16 / 2 ^ (row & 7))) * 2 + sub % 2;
      ((mx_u32x2*)xl[0][sub / 16])[at] = e ^ large;
      ((mx_u32x2*)xl[1][sub / 16])[at] = large;
      if ((sub & 3) == 0) xsc[row * (S1 * 4) + sub / 4] = (uint8_t)byte;
      if (p % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // two rows' chains of lane sums at a time: all would not fit in registers
    }
  }
  __syncthreads();
  // where this lane reads 16-byte pieces g and 4 + g of a row of 128 bytes (the same place in every row tile)
  const int p0 = r16 * 8 + (g ^ (r16 & 7)), p1 = r16 * 8 + ((g + 4) ^ (r16 & 7));
  int sx[U];  // byte s: the scale of block 4 s + g
#pragma unroll
  for (int u = 0; u < U; u++) {
    sx[u] = 0;
#pragma unroll
    for (int s = 0; s < S1; s++) sx[u] |= xsc[(u * 16 + r16) * (S1 * 4) + s * 4 + g] << (8 * s);
  }
  f32x4 acc[OT][U];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int u = 0; u < U; u++) acc[t][u] = f32x4{};

#pragma unroll 1
  for (int round = 0; round < ROUNDS; round++) {
    const int slot = round & 1;
    // Row tile u + 1's products are issued beside row tile u's SiLU and quantisation.
    f32x4 hacc[2][2];
    auto product1 = [&](auto UC) __attribute__((always_inline)) {
      constexpr int u = decltype(UC)::value;
      f32x4(&c)[2] = hacc[u & 1];
      c[0] = c[1] = f32x4{};
      mx_unroll<S1 * 2>([&](auto IC) __attribute__((always_inline)) {
        constexpr int i = decltype(IC)::value, s = i / 2, part = i % 2;
        const mx_u32x4* l = xl[part][s] + u * 128;
        const XFrag<8> x = {{l[p0], l[p1]}};
        c[0] = mfma<8, 0, s>(w1[0][s], x, c[0], (int)(s1[0][s] >> (8 * g)), sx[u]);
        c[1] = mfma<8, 0, s>(w1[1][s], x, c[1], (int)(s1[1][s] >> (8 * g)), sx[u]);
      });
    };
    float bias[8];
#pragma unroll
    for (int j = 0; j < 2; j++) *(f32x4*)&bias[4 * j] = *(const f32x4*)&b1l[round * 256 + wave * 32 + g * 8 + 4 * j];
    product1(std::integral_constant<int, 0>{});
    __builtin_amdgcn_sched_barrier(0);
    mx_unroll<U>([&](auto UC) __attribute__((always_inline)) {
      constexpr int u = decltype(UC)::value;
      if constexpr (u + 1 < U) product1(std::integral_constant<int, u + 1>{});
      else load2(round);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = silu(hacc[u & 1][j / 4][j % 4] + bias[j]);
      const uint32_t byte = mx_scale_byte<MX_E4M3>(mx_max_across32(mx_max_across16(mx_top8(v))));
      const int row = u * 16 + r16;
      ((mx_u32x2*)hid[slot][wave / 4])[(row * 8 + ((wave % 4 * 2 + g / 2) ^ (row & 7))) * 2 + g % 2] = mx_encode8<MX_E4M3>(v, mx_inverse(byte));
      if (g == 0) hsc[slot][row * 8 + wave] = (uint8_t)byte;
      __builtin_amdgcn_sched_barrier(0);
    });
    // The hidden units are written. (A slot is written again two rounds on, past the next round's barrier, which no
    // wavefront reaches before it has read this one's.) The weights' loads stay on their way.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    auto read_h = [&](int i) __attribute__((always_inline)) {  // i = (step, row tile)
      const mx_u32x4* l = hid[slot][i / U] + i % U * 128;
      return XFrag<8>{{l[p0], l[p1]}};
    };
    auto read_hs = [&](int i) __attribute__((always_inline)) { return (int)hsc[slot][(i % U * 16 + r16) * 8 + i / U * 4 + g]; };
    XFrag<8> hf[2] = {read_h(0), {}};
    int hs[2] = {read_hs(0), 0};
    mx_unroll<2 * U>([&](auto IC) __attribute__((always_inline)) {
      constexpr int i = decltype(IC)::value, s = i / U, u = i % U;
      if constexpr (i + 1 < 2 * U) {
        hf[(i + 1) & 1] = read_h(i + 1);
        hs[(i + 1) & 1] = read_hs(i + 1);
      }
#pragma unroll
      for (int t = 0; t < OT; t++) acc[t][u] = mfma<8, 0, 0>(w2[t][s], hf[i & 1], acc[t][u], (int)(s2[t][s] >> (8 * g)), hs[i & 1]);
      __builtin_amdgcn_sched_barrier(0);
    });
    load1(min(round + 1, ROUNDS - 1));  // (the last round's again after it: a branch here costs registers)
  }

  uint32_t res[OT / G][U][4];
#pragma unroll
  for (int run = 0; run < OT / G; run++)
#pragma unroll
    for (int u = 0; u < U; u++) {
      const i64 n = n0 + u * 16 + r16;
      load_residual<OUT_16, 4 * G>(a.out, n, wave * (16 * OT) + run * (16 * G) + g * (4 * G), n < a.out.N, res[run][u]);
    }
#pragma unroll
  for (int run = 0; run < OT / G; run++) {
    const int o = wave * (16 * OT) + run * (16 * G) + g * (4 * G);
    float bias[4 * G];
    mx_params<4 * G>(a.out.bias, a.out.bias_dt, o, 0.f, bias);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const i64 n = n0 + u * 16 + r16;
      float v[4 * G];
#pragma unroll
      for (int j = 0; j < G; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) v[j * 4 + i] = acc[run * G + j][u][i];
      finish<OUT_16>(a.out, n, o, v, bias, res[run][u], n < a.out.N);
    }
  }
}

template <bool F16, int C>
void launch_tail(const TailArgs& a) {
  k_mx_tail<F16, C><<<(unsigned)((a.out.N + kTailRows - 1) / kTailRows), 512, 0, stream()>>>(a);
  CK(hipGetLastError());
}
// The widths and rows that k_mx_tail takes. Up to 128 rows are k_mx_rows', where K goes over a workgroup's wavefronts. A workgroup
// here takes as long for one row as for 64, and reads all weights: at 256 channels three passes, whose products have more
// workgroups, are faster until 64 rows each fill three eighths of the CUs. us, one kernel / three passes: 256 channels, 129 rows
// 25.8 / 16.6, 2000 26.2 / 18.2, 4000 26.2 / 21.4, 6000 26.5 / 25.6, 8000 26.9 / 30.0, 15000 29.1 / 37.3; 128 channels, 129 rows
// 11.7 / 14.3, 4000 12.1 / 15.2.
bool fused(i64 n, i64 C, int fmt) { return fmt == MX_E4M3 && ((C == 128 && n > 128) || (C == 256 && n > 6144)); }
}  // namespace

namespace {
constexpr i64 kHidBytes = 128ll << 20;
i64 tail_rows(i64 n, i64 C, int fmt) {
  const i64 parts = (n * mx_row_bytes(fmt, 4 * C) + kHidBytes - 1) / kHidBytes;
  return n == 0 ? 0 : std::min(n, ((n + parts - 1) / parts + 255) / 256 * 256);
}
}  // namespace

i64 convnext_mlp_mx_workspace(i64 n, i64 C, int fmt) {
  if (n <= 0 || C <= 0 || fused(n, C, fmt)) return 0;
  const i64 m = tail_rows(n, C, fmt);
  return mx_rows_bytes(fmt, m, C) + mx_rows_bytes(fmt, m, 4 * C);
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
    if (t) mx_out_apart(&y, nullptr, *t, "the parameters");
  }
  if (n == 0) return;
  REQ(h.p && x.p && y.p && ((uintptr_t)h.p | (uintptr_t)x.p | (uintptr_t)y.p) % 16 == 0, "h, x, y must be 16-byte aligned and not null");
  for (const Tensor* t : {&h, &x}) REQ(t->p == y.p || !mx_overlap(t->p, t->bytes(), y.p, y.bytes()), "y must be h, x or apart from both");
  for (const MxTensor* w : {&w1, &w2}) {
    mx_out_apart(&y, nullptr, w->codes, "the weights");
    mx_out_apart(&y, nullptr, w->scales, "the weights");
  }
  if (fused(n, C, fmt)) {
    TailArgs a{};
    a.h = h.ptr<uint16_t>();
    a.w1 = w1.codes.ptr<uint8_t>();
    a.s1 = w1.scales.ptr<uint8_t>();
    a.w2 = w2.codes.ptr<uint8_t>();
    a.s2 = w2.scales.ptr<uint8_t>();
    a.gamma = gamma ? gamma->p : nullptr;
    a.beta = beta ? beta->p : nullptr;
    a.b1 = b1 ? b1->p : nullptr;
    a.gdt = gamma ? gamma->dt : F32;
    a.bdt = beta ? beta->dt : F32;
    a.b1dt = b1 ? b1->dt : F32;
    a.eps = eps;
    a.out.bias = b2 ? b2->p : nullptr;
    a.out.bias_dt = b2 ? b2->dt : F32;
    a.out.res = x.p;
    a.out.out = y.p;
    a.out.N = n;
    a.out.O = (int)C;
    a.out.f16 = h.dt == F16;
    auto go = [&](auto CC) {
      constexpr int W = decltype(CC)::value;
      h.dt == F16 ? launch_tail<true, W>(a) : launch_tail<false, W>(a);
    };
    if (C == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return;
  }
  const i64 step = tail_rows(n, C, fmt);
  if (workspace)
    for (const Tensor* t : {&h, &x, (const Tensor*)&y, &w1.codes, &w1.scales, &w2.codes, &w2.scales, gamma, beta, b1, b2})
      if (t) mx_apart(t->p, t->bytes(), workspace, (size_t)convnext_mlp_mx_workspace(n, C, fmt), "the workspace");
  MxWorkspace ws(workspace, workspace_bytes, convnext_mlp_mx_workspace(n, C, fmt));
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
    mx_product(am, w1, b1, nullptr, ACT_SILU, nullptr, &hm);
    mx_product(hm, w2, b2, &xm, ACT_NONE, &ym, nullptr);
  }
}
