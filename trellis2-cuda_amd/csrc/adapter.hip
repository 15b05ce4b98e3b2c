// Low-rank adapters of many requests beside one shared projection: with s = slots[n], row n gets scale[s] B_s (A_s x[n]) added to its
// projection; a slot outside [0, L) is no adapter.
#include "mx.h"

namespace {
struct AdapterArgs {
  const void *x, *w, *a, *b, *y, *bias;
  const int32_t* slots;
  const float* scale;
  void* out;
  i64 N;
  int L, R, K, O, bias_dt;
};

// One workgroup a row: h = A_s x[n] by wavefronts, then every thread its channels
template <bool F16>
__global__ void __launch_bounds__(256) k_adapter(AdapterArgs a) {
  __shared__ float h[256];
  const i64 n = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, s = a.slots[n];
  const bool has = s >= 0 && s < a.L;
  const uint16_t* x = (const uint16_t*)a.x + n * a.K;
  if (has)
    for (int r = wave; r < a.R; r += 4) {
      const uint16_t* row = (const uint16_t*)a.a + ((i64)s * a.R + r) * a.K;
      float v = 0.f;
      for (int k = lane; k < a.K; k += 64) v += mx_lo<F16>(x[k]) * mx_lo<F16>(row[k]);
      for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
      if (lane == 0) h[r] = v * (a.scale ? a.scale[s] : 1.f);
    }
  __syncthreads();
  for (int o = tid; o < a.O; o += 256) {
    float v[1] = {0.f}, acc = 0.f;
    mx_params<1>(a.bias, a.bias_dt, o, 0.f, v);
    if (a.w)
      for (int k = 0; k < a.K; k++) acc += mx_lo<F16>(x[k]) * mx_lo<F16>(((const uint16_t*)a.w)[(i64)o * a.K + k]);
    else acc = mx_lo<F16>(((const uint16_t*)a.y)[n * a.O + o]);
    acc += v[0];
    if (has)
      for (int r = 0; r < a.R; r++) acc += h[r] * mx_lo<F16>(((const uint16_t*)a.b)[((i64)s * a.O + o) * a.R + r]);
    ((uint16_t*)a.out)[n * a.O + o] = (uint16_t)mx_pack2<F16>(acc, 0.f);
  }
}

constexpr int kHighestRank = 256;
void check(const Tensor& t, const char* what, DT dt, std::vector<i64> sh) {
  std::string s;
  for (i64 v : sh) s += (s.empty() ? "" : ",") + std::to_string(v);
  REQ(t.dt == dt && t.sh == sh, "%s must be %s [%s]", what, dname(dt), s.c_str());
  REQ((uintptr_t)t.p % 16 == 0 && (t.p || t.numel() == 0), "%s must be 16-byte aligned and not null", what);
}
void adapter(const Tensor& x, const Tensor* w, const Tensor* y, const Tensor& a, const Tensor& b, const Tensor& slots, const Tensor* scale,
             const Tensor* bias, Tensor& out, void* workspace, i64 workspace_bytes) {
  REQ(x.dt == F16 || x.dt == BF16, "x must be bf16/fp16, not %s", dname(x.dt));
  REQ(x.dim() == 2 && a.dim() == 3 && b.dim() == 3, "x must be [N,K], a [L,R,K], b [L,O,R]");
  const i64 N = x.size(0), K = x.size(1), L = a.size(0), R = a.size(1), O = b.size(1);
  REQ(N < (1ll << 31), "%lld rows", (long long)N);
  REQ(L > 0 && L <= (1 << 16), "%lld adapters: 1 to 2^16", (long long)L);
  REQ(R > 0 && R % 8 == 0 && R <= kHighestRank, "rank %lld: a positive multiple of 8, at most %d", (long long)R, kHighestRank);
  for (i64 c : {O, K}) REQ(c > 0 && c % 8 == 0 && c <= (1 << 20), "%lld channels: a positive multiple of 8, at most 2^20", (long long)c);
  check(x, "x", x.dt, {N, K});
  check(a, "a", x.dt, {L, R, K});
  check(b, "b", x.dt, {L, O, R});
  if (w) check(*w, "w", x.dt, {O, K});
  if (y) check(*y, "y", x.dt, {N, O});
  check(out, "out", x.dt, {N, O});
  REQ(slots.dt == I32 && slots.numel() == N && (slots.p || N == 0) && (uintptr_t)slots.p % 4 == 0, "slots must be int32 [%lld] and not null", (long long)N);
  if (scale) REQ(scale->dt == F32 && scale->numel() == L && scale->p, "scale must be F32 [%lld]", (long long)L);
  if (bias) REQ(bias->numel() == O && bias->p && (bias->dt == F32 || bias->dt == F16 || bias->dt == BF16), "bias must have %lld elements", (long long)O);
  for (const Tensor* t : {&x, &a, &b, &slots, w, scale, bias})
    if (t) mx_apart(out.p, out.bytes(), t->p, t->bytes(), "out");
  if (y) REQ(y->p == out.p || !mx_overlap(y->p, y->bytes(), out.p, out.bytes()), "out must be y or apart from it");
  if (N == 0) return;
  const i64 need = adapter_workspace(N, K, R);
  if (workspace) {
    for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &a, &b, &slots, w, y, scale, bias, &out})
      if (t) mx_apart(t->p, t->bytes(), workspace, (size_t)need, "the workspace");
  }
  MxWorkspace ws(workspace, workspace_bytes, need);
  AdapterArgs g{x.p, w ? w->p : nullptr, a.p, b.p, y ? y->p : nullptr, bias ? bias->p : nullptr, slots.ptr<int32_t>(),
                scale ? scale->ptr<float>() : nullptr, out.p, N, (int)L, (int)R, (int)K, (int)O, bias ? bias->dt : F32};
  if (x.dt == F16) k_adapter<true><<<(unsigned)N, 256, 0, stream()>>>(g);
  else k_adapter<false><<<(unsigned)N, 256, 0, stream()>>>(g);
  CK(hipGetLastError());
}
}  // namespace

i64 adapter_workspace(i64 N, i64 K, i64 R) { return 0; }

void adapter_linear(const Tensor& x, const Tensor& w, const Tensor& a, const Tensor& b, const Tensor& slots, const Tensor* scale,
                    const Tensor* bias, Tensor& out, void* workspace, i64 workspace_bytes) {
  adapter(x, &w, nullptr, a, b, slots, scale, bias, out, workspace, workspace_bytes);
}
void adapter_add(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& slots, const Tensor* scale, Tensor& out,
                 void* workspace, i64 workspace_bytes) {
  adapter(x, nullptr, &y, a, b, slots, scale, nullptr, out, workspace, workspace_bytes);
}
