// Products of groups of rows with a weight matrix each, and their gradients. Rows ends[g-1] .. ends[g] - 1 are group g's.
//   forward  y[n] = W_g x[n] + b_g        dx[n] = W_g^T dy[n]        dW_g = sum over g's rows of dy[n] x[n]^T, db_g = sum of dy[n]
#include "mx.h"

#include <algorithm>

namespace {
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { FORWARD = 0, DX = 1, DW = 2 };
struct GroupArgs {
  const void *a, *b, *bias;  // forward: x, w; dx: dy, w; dw: dy, x
  const int32_t* ends;
  void *out, *db;
  i64 N;
  int G, K, O, bias_dt, out_f32;
};

template <bool F16>
__device__ __forceinline__ f32x4 mfma(mx_u32x4 a, mx_u32x4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Group g's rows: [first, first + count), inside [0, N) whatever ends holds
__device__ __forceinline__ void rows_of(const GroupArgs& a, int g, i64& first, i64& count) {
  const i64 s = g ? min((i64)max(a.ends[g - 1], 0), a.N) : 0, e = min((i64)max(a.ends[g], 0), a.N);
  first = s;
  count = max(e - s, (i64)0);
}

// 64 x 64 results per workgroup of 4 wavefronts, operands element by element through LDS
template <int OP, bool F16>
__global__ void __launch_bounds__(256) k_group(GroupArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t la[64][40], lb[64][40];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = blockIdx.x * 64;  // first column of the result
  i64 first, count, m0 = 0;
  int g = 0, depth = OP == FORWARD ? a.K : a.O;
  if (OP == DW) {
    g = blockIdx.z;
    rows_of(a, g, first, count);
    m0 = blockIdx.y * 64;
    depth = 0;
  } else {
    i64 t = blockIdx.y;
    for (; g < a.G; g++) {
      rows_of(a, g, first, count);
      const i64 tiles = (count + 63) / 64;
      if (t < tiles) break;
      t -= tiles;
    }
    if (g == a.G) return;
    m0 = t * 64;
  }
  const i64 inner = OP == DW ? count : depth, rows = OP == DW ? a.O : count;
  const int cols = OP == FORWARD ? a.O : a.K;
  const uint16_t *pa = (const uint16_t*)a.a, *pb = (const uint16_t*)a.b;
  const i64 wbase = (i64)g * a.O * a.K;
  f32x4 acc[4] = {};
  float sum = 0.f;
  for (i64 k0 = 0; k0 < inner; k0 += 32) {
    for (int i = tid; i < 64 * 32; i += 256) {
      const int r = OP == DW ? i % 64 : i / 32, k = OP == DW ? i / 64 : i % 32;
      const bool in = m0 + r < rows && k0 + k < inner;
      la[r][k] = !in ? 0 : OP == DW ? pa[(first + k0 + k) * a.O + m0 + r] : pa[(first + m0 + r) * depth + k0 + k];
    }
    for (int i = tid; i < 64 * 32; i += 256) {
      const int c = OP == FORWARD ? i / 32 : i % 64, k = OP == FORWARD ? i % 32 : i / 64;
      const bool in = c0 + c < cols && k0 + k < inner;
      lb[c][k] = !in ? 0 : OP == FORWARD ? pb[wbase + (i64)(c0 + c) * a.K + k0 + k] : OP == DX ? pb[wbase + (k0 + k) * a.K + c0 + c]
                                                                                         : pb[(first + k0 + k) * a.K + c0 + c];
    }
    __syncthreads();
    const mx_u32x4 fb = *(const mx_u32x4*)&lb[wave * 16 + lane % 16][lane / 16 * 8];
    for (int t = 0; t < 4; t++) acc[t] = mfma<F16>(fb, *(const mx_u32x4*)&la[t * 16 + lane % 16][lane / 16 * 8], acc[t]);
    if (OP == DW && tid < 64)
      for (int k = 0; k < 32; k++) sum += mx_lo<F16>(la[tid][k]);
    __syncthreads();
  }
  for (int t = 0; t < 4; t++)
    for (int i = 0; i < 4; i++) {
      const i64 m = m0 + t * 16 + lane % 16;
      const int c = c0 + wave * 16 + lane / 16 * 4 + i;
      if (m >= rows || c >= cols) continue;
      float bias[1];
      mx_params<1>(a.bias, a.bias_dt, (i64)g * a.O + c, 0.f, bias);
      const float v = acc[t][i] + bias[0];
      const i64 at = OP == DW ? wbase + m * a.K + c : (first + m) * cols + c;
      if (a.out_f32) ((float*)a.out)[at] = v;
      else ((uint16_t*)a.out)[at] = (uint16_t)mx_pack2<F16>(v, 0.f);
    }
  if (OP == DW && a.db && blockIdx.x == 0 && tid < 64 && m0 + tid < rows) {
    const i64 at = (i64)g * a.O + m0 + tid;
    if (a.out_f32) ((float*)a.db)[at] = sum;
    else ((uint16_t*)a.db)[at] = (uint16_t)mx_pack2<F16>(sum, 0.f);
  }
}

template <int OP>
void launch(const GroupArgs& a, DT dt) {
  const int cols = OP == FORWARD ? a.O : a.K;
  const i64 tiles = a.N / 64 + a.G;  // the sum over groups of ceil(rows / 64) is at most this
  REQ(OP == DW || tiles <= 65535, "%lld rows", (long long)a.N);
  const dim3 grid(cdiv(cols, 64), OP == DW ? cdiv(a.O, 64) : (unsigned)tiles, OP == DW ? a.G : 1);
  if (dt == F16) k_group<OP, true><<<grid, 256, 0, stream()>>>(a);
  else k_group<OP, false><<<grid, 256, 0, stream()>>>(a);
  CK(hipGetLastError());
}

constexpr i64 kWidest = 1 << 20, kMostGroups = 1 << 16;
void check_rows(const Tensor& t, const char* what, DT dt, i64 rows, i64 cols) {
  REQ(t.dt == dt && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, "%s must be %s [%lld,%lld]", what, dname(dt), (long long)rows,
      (long long)cols);
  REQ((uintptr_t)t.p % 16 == 0 && (t.p || rows == 0), "%s must be 16-byte aligned and not null", what);
}
void check_weights(const Tensor& t, const char* what, i64& groups, i64& O, i64& K) {
  REQ(t.dim() == 3, "%s must be [G,O,K]", what);
  groups = t.size(0), O = t.size(1), K = t.size(2);
  REQ(groups > 0 && groups <= kMostGroups, "%lld groups: 1 to 2^16", (long long)groups);
  for (i64 c : {O, K}) REQ(c > 0 && c % 8 == 0 && c <= kWidest, "%lld channels: a positive multiple of 8, at most 2^20", (long long)c);
  REQ(t.p && (uintptr_t)t.p % 16 == 0, "%s must be 16-byte aligned and not null", what);
}
void check_ends(const Tensor& ends, i64 groups) {
  REQ(ends.dt == I32 && ends.numel() == groups && ends.p && (uintptr_t)ends.p % 4 == 0, "ends must be int32 [%lld] and not null",
      (long long)groups);
}
void check_16(const Tensor& t, const char* what) { REQ(t.dt == F16 || t.dt == BF16, "%s must be bf16/fp16, not %s", what, dname(t.dt)); }
i64 rows_in(const Tensor& t, const char* what) {
  REQ(t.dim() == 2, "%s must be a matrix", what);
  REQ(t.size(0) < (1ll << 31), "%lld rows", (long long)t.size(0));
  return t.size(0);
}
void apart(const Tensor& out, const Tensor* t, const char* what) {
  if (t) mx_apart(out.p, out.bytes(), t->p, t->bytes(), what);
}
}  // namespace

void group_linear(const Tensor& x, const Tensor& w, const Tensor& ends, const Tensor* bias, Tensor& y) {
  i64 G, O, K;
  check_16(x, "x");
  const i64 N = rows_in(x, "x");
  check_weights(w, "w", G, O, K);
  REQ(w.dt == x.dt, "w must be of x's type");
  check_rows(x, "x", x.dt, N, K);
  check_rows(y, "out", x.dt, N, O);
  check_ends(ends, G);
  if (bias)
    REQ(bias->numel() == G * O && bias->p && (bias->dt == F32 || bias->dt == F16 || bias->dt == BF16), "bias must have %lld elements", (long long)(G * O));
  for (const Tensor* t : {&x, &w, &ends, bias}) apart(y, t, "out");
  if (N == 0) return;
  GroupArgs a{x.p, w.p, bias ? bias->p : nullptr, ends.ptr<int32_t>(), y.p, nullptr, N, (int)G, (int)K, (int)O, bias ? bias->dt : F32, 0};
  launch<FORWARD>(a, x.dt);
}

void group_linear_dx(const Tensor& dy, const Tensor& w, const Tensor& ends, Tensor& dx) {
  i64 G, O, K;
  check_16(dy, "dy");
  const i64 N = rows_in(dy, "dy");
  check_weights(w, "w", G, O, K);
  REQ(w.dt == dy.dt, "w must be of dy's type");
  check_rows(dy, "dy", dy.dt, N, O);
  check_rows(dx, "out", dy.dt, N, K);
  check_ends(ends, G);
  for (const Tensor* t : {&dy, &w, &ends}) apart(dx, t, "out");
  if (N == 0) return;
  GroupArgs a{dy.p, w.p, nullptr, ends.ptr<int32_t>(), dx.p, nullptr, N, (int)G, (int)K, (int)O, F32, 0};
  launch<DX>(a, dy.dt);
}

void group_linear_dw(const Tensor& dy, const Tensor& x, const Tensor& ends, Tensor& dw, Tensor* db) {
  i64 G, O, K;
  check_16(dy, "dy");
  const i64 N = rows_in(dy, "dy");
  check_weights(dw, "out", G, O, K);
  REQ(dw.dt == F32 || dw.dt == dy.dt, "out must be fp32 or of dy's type");
  check_rows(dy, "dy", dy.dt, N, O);
  check_rows(x, "x", dy.dt, N, K);
  check_ends(ends, G);
  for (const Tensor* t : {&dy, &x, &ends}) apart(dw, t, "out");
  if (db) {
    REQ(db->dt == dw.dt && db->numel() == G * O && db->p && (uintptr_t)db->p % 16 == 0, "the bias' gradient must have %lld elements of out's type, 16-byte aligned",
        (long long)(G * O));
    for (const Tensor* t : std::initializer_list<const Tensor*>{&dy, &x, &ends, &dw}) apart(*db, t, "the bias' gradient");
  }
  GroupArgs a{dy.p, x.p, nullptr, ends.ptr<int32_t>(), dw.p, db ? db->p : nullptr, N, (int)G, (int)K, (int)O, F32, dw.dt == F32};
  launch<DW>(a, dy.dt);
}
