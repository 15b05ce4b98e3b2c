// Low-rank adapters of many requests beside one shared projection: with s = slots[n], row n gets scale[s] B_s (A_s x[n]) added to its
// projection; a slot outside [0, L) is no adapter.
#include "group.h"

#include <algorithm>
#include <type_traits>

namespace {
// Four ranks of a row's first product, the first of them rank r of row n of N, into memory in halves (group.h)
template <bool F16>
__device__ __forceinline__ void store_inner(uint16_t* h, i64 n, i64 N, int R, int r, f32x4 c, float to) {
  mx_u32x2 high, low;
#pragma unroll
  for (int j = 0; j < 2; j++) {
    uint32_t hi, lo;
    halves<F16>(c[2 * j] * to, c[2 * j + 1] * to, hi, lo);
    high[j] = hi;
    low[j] = lo;
  }
  const i64 n0 = n / 16 * 16;
  const int m = (int)min((i64)16, N - n0);
  uint16_t* p = h + n0 * R * 2 + inner_tile_place((int)(n - n0), m, r);
  *(mx_u32x2*)p = high;
  *(mx_u32x2*)(p + inner_to_low(m, r, R)) = low;
}
__device__ __forceinline__ uint32_t top4(f32x4 c) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) m = max(m, finite_bits(c[j]));
  return m;
}

// The first product, h = scale[s] x a[s]^T per row, one row per workgroup: the reading of a is shared by nobody but the caches, and no row waits for
// another's adapter. The 8 wavefronts share the depth out, and their sums meet in LDS in a fixed order. 16 RT ranks (blockIdx.y: which).
// Bound by latency: [77, 4096], 16 ranks of 32 adapters 5.2 us, slots and then one load of all that a wavefront needs.
template <bool F16, int RT>
__global__ void __launch_bounds__(512) k_adapter_in_rows(const uint16_t* x, const uint16_t* a, const int32_t* slots, const float* scale, uint16_t* h,
                                                         float* back, int L, int R, int K) {
  constexpr int NW = 8;
  __shared__ f32x4 sums[NW][RT][4];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const i64 n = blockIdx.x;
  const int s = slots[n], r0 = blockIdx.y * (16 * RT), ranks = min(16 * RT, R - r0);
  if (s < 0 || s >= L) return;
  const int S = (K + 63) / 64, s0 = S * wave / NW, s1 = S * (wave + 1) / NW;
  const auto rx = buffer(x + n * K, (uint32_t)(K * 2)), ra = buffer(a + ((i64)s * R + r0) * K, (uint32_t)(ranks * K * 2));
  const uint32_t off = line_offset(lane, K * 2);
  const int depth = line_depth(lane);
  f32x4 acc[RT] = {};
  constexpr int AT = RT == 1 ? 8 : RT == 2 ? 4 : 2;  // steps on their way together
  for (int k = s0; k < s1; k += AT) {
    Lines qa[AT][RT], qx[AT];
#pragma unroll
    for (int i = 0; i < AT; i++) {
      const bool in = k + i < s1 && (k + i) * 64 + depth < K;
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const uint32_t at = off + t * 16 * K * 2;
        const int r = t * 16 + (r16 & 14);
        qa[i][t].even = __builtin_amdgcn_raw_buffer_load_b128(ra, in && r < ranks ? at : kOOR, (k + i) * 128, 0);
        qa[i][t].odd = __builtin_amdgcn_raw_buffer_load_b128(ra, in && r + 1 < ranks ? at + K * 2 : kOOR, (k + i) * 128, 0);
      }
      qx[i].even = __builtin_amdgcn_raw_buffer_load_b128(rx, in && r16 < 2 ? off : kOOR, (k + i) * 128, 0);
      qx[i].odd = mx_u32x4{};
    }
    __builtin_amdgcn_sched_barrier(0);  // the loads stay together
#pragma unroll
    for (int i = 0; i < AT; i++) {
      mx_u32x4 x0, x1, a0, a1;
      operands(qx[i], lane, x0, x1);
#pragma unroll
      for (int t = 0; t < RT; t++) {
        operands(qa[i][t], lane, a0, a1);
        acc[t] = mfma<F16>(a0, x0, acc[t]);
        acc[t] = mfma<F16>(a1, x1, acc[t]);
      }
    }
  }
  if (r16 == 0) {
#pragma unroll
    for (int t = 0; t < RT; t++) sums[wave][t][g] = acc[t];
  }
  __syncthreads();
  if (wave == 0) {  // the first 16 lanes have 4 ranks each
    const bool in = lane < RT * 4 && lane * 4 < ranks;
    f32x4 c{};
    if (in) {
#pragma unroll
      for (int w = 0; w < NW; w++) c += sums[w][lane / 4][lane % 4];
      c *= scale ? scale[s] : 1.f;
    }
    float to = 1.f;
    if constexpr (F16) {
      uint32_t top = mx_quad_max(top4(c));
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x124, 0xf, 0xf, true));  // of 4 lanes on, of the 16
      top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x128, 0xf, 0xf, true));
      float from;
      inner_factors(top, to, from);
      if (lane == 0) back[n * ((R + 63) / 64) + r0 / 64] = from;
    }
    if (in) store_inner<F16>(h, n, gridDim.x, R, r0 + lane * 4, c, to);
  }
}

// The same for many rows: 16 U of them per workgroup. Each XCD takes neighbouring rows, whose adapters are the same ones. Every adapter that
// some of the rows have takes its turn, and the lanes whose row has it keep the sums; `turns` workgroups share the adapters out, so that one
// with a request's border among its rows takes no longer than the others (those without a turn end at once). Bound by how many loads a CU has
// on their way: [8209, 4096], 64 ranks, 30 - 37 us (x alone 13 at a copy's rate); [8209, 2080], 24 ranks, 16 us.
template <bool F16, int U, int RT>
__global__ void __launch_bounds__(256, 2) k_adapter_in(const uint16_t* x, const uint16_t* a, const int32_t* slots, const float* scale, uint16_t* h,
                                                       float* back, i64 N, int L, int R, int K, int turns) {
  constexpr int NW = 4;
  __shared__ f32x4 sums[NW][U * RT][64];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const i64 n0 = ((i64)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8) * (16 * U);
  if (n0 >= N) return;
  const int rows = (int)min((i64)(16 * U), N - n0), r0 = blockIdx.y / turns * (16 * RT), ranks = min(16 * RT, R - r0);
  int mine = lane < rows && lane < 16 * U ? slots[n0 + lane] : -1;
  mine = mine < L ? mine : -1;
  int slot[U];
#pragma unroll
  for (int u = 0; u < U; u++) slot[u] = __shfl(mine, u * 16 + r16, 64);
  const int S = (K + 63) / 64, s0 = S * wave / NW, s1 = S * (wave + 1) / NW;
  const auto rx = buffer(x + n0 * K, (uint32_t)(rows * K * 2));
  const uint32_t off = line_offset(lane, K * 2);
  const int depth = line_depth(lane);
  uint64_t done = 0;  // rows whose adapters this workgroup took
  int turn = 0;
  for (uint64_t left = __ballot(mine >= 0); left; turn++) {
    const int s = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t same = __ballot(mine == s);
    left &= ~same;
    if (turn % turns != blockIdx.y % turns) continue;
    done |= same;
    const auto ra = buffer(a + ((i64)s * R + r0) * K, (uint32_t)(ranks * K * 2));
    f32x4 acc[U][RT];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int t = 0; t < RT; t++) acc[u][t] = f32x4{};
    struct Step {
      Lines a[RT], x[U];
    } q[2];  // one is loaded while the other is multiplied
    auto load = [&](Step& q, int k) __attribute__((always_inline)) {
      const bool in = k < s1 && k * 64 + depth < K;
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const uint32_t at = off + t * 16 * K * 2;
        const int r = t * 16 + (r16 & 14);
        q.a[t].even = __builtin_amdgcn_raw_buffer_load_b128(ra, in && r < ranks ? at : kOOR, k * 128, 0);
        q.a[t].odd = __builtin_amdgcn_raw_buffer_load_b128(ra, in && r + 1 < ranks ? at + K * 2 : kOOR, k * 128, 0);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t at = off + u * 16 * K * 2;
        const int n = u * 16 + (r16 & 14);
        q.x[u].even = __builtin_amdgcn_raw_buffer_load_b128(rx, in && n < rows ? at : kOOR, k * 128, 0);
        q.x[u].odd = __builtin_amdgcn_raw_buffer_load_b128(rx, in && n + 1 < rows ? at + K * 2 : kOOR, k * 128, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // the loads stay together
    };
    auto multiply = [&](const Step& q) __attribute__((always_inline)) {
      mx_u32x4 x[U][2];
#pragma unroll
      for (int u = 0; u < U; u++) operands(q.x[u], lane, x[u][0], x[u][1]);
#pragma unroll
      for (int t = 0; t < RT; t++) {
        mx_u32x4 a[2];
        operands(q.a[t], lane, a[0], a[1]);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < 2; j++) acc[u][t] = mfma<F16>(a[j], x[u][j], acc[u][t]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    load(q[0], s0);
    for (int k = s0; k < s1; k += 2) {
      load(q[1], k + 1);
      multiply(q[0]);
      load(q[0], k + 2);
      multiply(q[1]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (slot[u] != s) continue;
#pragma unroll
      for (int t = 0; t < RT; t++) sums[wave][u * RT + t][lane] = acc[u][t];
    }
  }
  if (!done) return;
  __syncthreads();
  for (int u = wave; u < U; u += NW) {
    const int n = u * 16 + r16;
    const bool mine_too = done >> n & 1;
    const float by = mine_too && scale ? scale[slots[n0 + n]] : 1.f;
    f32x4 c[RT];
    uint32_t top = 0;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      c[t] = f32x4{};
      if (!mine_too || t * 16 + g * 4 >= ranks) continue;
#pragma unroll
      for (int w = 0; w < NW; w++) c[t] += sums[w][u * RT + t][lane];
      c[t] *= by;
      top = max(top, top4(c[t]));
    }
    float to = 1.f;
    if constexpr (F16) {
      float from;
      inner_factors(mx_max_across32(mx_max_across16(top)), to, from);
      if (mine_too && g == 0) back[(n0 + n) * ((R + 63) / 64) + r0 / 64] = from;
    }
#pragma unroll
    for (int t = 0; t < RT; t++)
      if (mine_too && t * 16 + g * 4 < ranks) store_inner<F16>(h, n0 + n, N, R, r0 + t * 16 + g * 4, c[t], to);
  }
}

// out = y + scale b[s] h: 16 TM rows by 16 TC channels per wavefront, four wavefronts beside each other; or (SHARE) all four at the same
// place, sharing out the rows' adapters, for few rows that differ in theirs; FUSED, they make the first product, too. Bound by y's reading and
// writing: [8209, 4128] fp16, 24 ranks, 31.4 us, 4.3 TB/s; few rows by latency ([77, 4096], 16 ranks of 32 adapters, 5.8 us).
template <bool F16, int TC, int TM, bool SHARE, bool FUSED>
__global__ void __launch_bounds__(256) k_adapter_add(GroupArgs a) {
  constexpr int NW = 4;
  __shared__ f32x4 part[SHARE ? NW : 1][SHARE ? TC * TM : 1][64];
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const i64 n0 = (i64)(blockIdx.x / a.tiles_c) * (16 * TM);
  const int rows = (int)min((i64)(16 * TM), a.N - n0), tile = blockIdx.x % a.tiles_c * (SHARE ? 1 : NW) + (SHARE ? 0 : wave);
  const int c0 = tile * (16 * TC), cols = min(16 * TC, a.O - c0);
  if (cols <= 0) return;
  const auto ry = buffer((const uint16_t*)a.m + n0 * a.O + c0, (uint32_t)(((rows - 1) * a.O + cols) * 2));
  mx_u32x4 y[TC / 2][TM];
#pragma unroll
  for (int t = 0; t < TC / 2; t++)
#pragma unroll
    for (int u = 0; u < TM; u++) {
      const int c = t * 32 + g * 8, m = u * 16 + r16;
      y[t][u] = __builtin_amdgcn_raw_buffer_load_b128(ry, c < cols && m < rows ? (uint32_t)((m * a.O + c) * 2) : kOOR, 0, 0);
    }
  f32x4 acc[TC][TM];
#pragma unroll
  for (int t = 0; t < TC; t++)
#pragma unroll
    for (int u = 0; u < TM; u++) acc[t][u] = f32x4{};
  auto chan = [](int t, int r) __attribute__((always_inline)) { return t / 2 * 32 + r / 4 * 8 + t % 2 * 4 + r % 4; };
  if constexpr (FUSED) {
    __shared__ __attribute__((aligned(16))) InnerSums inner[NW];
    inner_products<F16, NW>(a, lane, wave, inner[wave]);
    __syncthreads();
    add_adapters<F16>(a, acc, n0, rows, c0, cols, lane, chan, summed_inner<F16, NW>(a, inner, lane), wave, NW);
  } else {
    add_adapters<F16>(a, acc, n0, rows, c0, cols, lane, chan, stored_inner<F16>(a, n0, rows, lane), SHARE ? wave : 0, SHARE ? NW : 1);
  }
  if constexpr (SHARE) {
#pragma unroll
    for (int t = 0; t < TC; t++)
#pragma unroll
      for (int u = 0; u < TM; u++) part[wave][t * TM + u][lane] = acc[t][u];
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < TC / 2; t++)
#pragma unroll
    for (int u = 0; u < TM; u++) {
      if (SHARE && (t * TM + u) % NW != wave) continue;
      if constexpr (SHARE) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
          acc[t * 2 + k][u] = part[0][(t * 2 + k) * TM + u][lane];
#pragma unroll
          for (int w = 1; w < NW; w++) acc[t * 2 + k][u] += part[w][(t * 2 + k) * TM + u][lane];
        }
      }
      const int c = t * 32 + g * 8, m = u * 16 + r16;
      if (c >= cols || m >= rows) continue;
      float v[8];
      mx_unpack8<F16>(y[t][u], v);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += acc[t * 2 + j / 4][u][j % 4];
      *(mx_u32x4*)((uint16_t*)a.out + (n0 + m) * a.O + c0 + c) = mx_pack8<F16>(v);
    }
}

// us with one, two and four workgroups, [8209, 4096] to 64 channels, 64 ranks: 64 requests of 16 adapters 57, 40 and 37, 24 requests 44, 40 and
// 36, one 23 each; of 16 ranks, 64 requests, 29, 25 and 25; adapter_linear to 4096 channels, 24 requests, 299, 290 and 290
constexpr int kTurns = 2;
// One workgroup a row reads 2 R K bytes of a for each; 16 U rows share them, but wait for every adapter among them in turn. us of adapter_add,
// by row / in tiles, [N, 4096] to 64 channels, four adapters in runs; every row another than its neighbour: 256 rows of 64 ranks 16 / 24;
// 23 / 127, 512 of 64 24 / 21; 34 / 134, 1024 of 16 15 / 15; 19 / 68, of 64 39 / 18; 59 / 135, 2048 of 16 25 / 15; 36 / 80. The order is not
// known here, so rows in runs pay up to 10 us for what others save.
bool by_row(i64 N, i64 R) { return N <= 2048 && N * R <= 32768; }
template <bool F16>
void launch_in(const AdapterPart& p, i64 N, int K, uint16_t* h, float* back) {
  const int L = p.L, R = p.R;
  auto go = [&](auto UC, auto RC) {
    constexpr int U = decltype(UC)::value, RT = decltype(RC)::value;
    const i64 tiles = U ? ((N + 16 * U - 1) / (16 * (U ? U : 1)) + 7) / 8 * 8 : N;
    const dim3 grid((unsigned)tiles, cdiv(R, 16 * RT) * (U ? kTurns : 1));
    const uint16_t *px = (const uint16_t*)p.x, *pa = (const uint16_t*)p.a;
    if constexpr (U == 0) k_adapter_in_rows<F16, RT><<<grid, 512, 0, stream()>>>(px, pa, p.slots, p.scale, h, back, L, R, K);
    else k_adapter_in<F16, U, RT><<<grid, 256, 0, stream()>>>(px, pa, p.slots, p.scale, h, back, N, L, R, K, kTurns);
    CK(hipGetLastError());
  };
  auto by = [&](auto UC) {
    if constexpr (decltype(UC)::value <= 2) {  // (more rows a workgroup only where it has 64 ranks)
      if (R <= 16) return go(UC, std::integral_constant<int, 1>{});
      if (R <= 32) return go(UC, std::integral_constant<int, 2>{});
    }
    go(UC, std::integral_constant<int, 4>{});
  };
  // Workgroups of 16 u rows. With more than 32 ranks one takes some u + 2 (its rows of x, and a) and fills a CU; a second one doubles the time
  // ([8209, 4096], 64 ranks of 16 adapters: 41 us with 32 rows, whose 257 workgroups are one too many; [8192, 4096] 28)
  const i64 cus = mx_device_cus();
  int u = 2;
  i64 least = 0;
  for (int t = 2; t <= (R > 32 ? 4 : 2); t++) {
    const i64 rounds = cdiv(cdiv(cdiv(N, 16 * t), 8) * 8, cus), cost = rounds * (t + 2);
    if (t == 2 || cost < least) u = t, least = cost;
  }
  if (by_row(N, R)) by(std::integral_constant<int, 0>{});
  else if (u == 2) by(std::integral_constant<int, 2>{});
  else if (u == 3) by(std::integral_constant<int, 3>{});
  else by(std::integral_constant<int, 4>{});
}
// Up to as many rows four wavefronts share a place's adapters out. us of adapter_add, so / not, [N, 64] to 4096 channels, every row another of
// 32 adapters than its neighbour (the first product in tiles for 1024 rows and more): 512 rows 15.8 / 16.3, 1024 29 / 27, 2048 42 / 38
constexpr i64 kSharedRows = 512;
template <bool F16>
void launch_add(const GroupArgs& a) {
  auto go = [&](auto TCC, auto TMC, auto share, auto fused) {
    constexpr int TC = decltype(TCC)::value, TM = decltype(TMC)::value;
    constexpr bool SHARE = decltype(share)::value, FUSED = decltype(fused)::value;
    const i64 tiles = (a.N + 16 * TM - 1) / (16 * TM);
    GroupArgs p = a;
    p.tiles_c = cdiv(a.O, (SHARE ? 16 : 64) * TC);
    const i64 blocks = tiles * p.tiles_c;
    REQ(blocks * 256 < (1ll << 32), "%lld rows by %d channels: too many for a launch", (long long)a.N, a.O);
    k_adapter_add<F16, TC, TM, SHARE, FUSED><<<(unsigned)blocks, 256, 0, stream()>>>(p);
    CK(hipGetLastError());
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  constexpr std::integral_constant<int, 4> four{};
  if (!a.ad.h) go(four, one, std::true_type{}, std::true_type{});
  else if (a.N <= kSharedRows) go(four, one, std::true_type{}, std::false_type{});
  else go(two, four, std::false_type{}, std::false_type{});
}

// Of a row's first product: its halves and its factors
i64 inner_row_bytes(i64 R) { return R * 4 + (R + 63) / 64 * 4; }
i64 inner_bytes(i64 N, i64 R) { return adapter_fused(N, R) ? 0 : (N * inner_row_bytes(R) + 15) / 16 * 16; }
constexpr i64 kWhole = 1 << 28;  // of a workspace of the library's own: more than 256 MB, and rows go in parts of some 10^5 and more
constexpr int kHighestRank = 256;
constexpr i64 kMostRows = 1 << 27;  // whose launches hold fewer than 2^32 threads in any direction
void check(const Tensor& t, const char* what, DT dt, std::initializer_list<i64> sh) {
  bool same = t.dt == dt && t.dim() == (int)sh.size();
  if (same) {
    int i = 0;
    for (i64 v : sh) same &= t.sh[i++] == v;
  }
  if (!same) {  // (the message is put together only now: a call takes some microseconds in all)
    std::string s;
    for (i64 v : sh) s += (s.empty() ? "" : ",") + std::to_string(v);
    REQ(same, "%s must be %s [%s]", what, dname(dt), s.c_str());
  }
  REQ((uintptr_t)t.p % 16 == 0 && (t.p || t.numel() == 0), "%s must be 16-byte aligned and not null", what);
}
void adapter(const Tensor& x, const Tensor* w, const Tensor* y, const Tensor& a, const Tensor& b, const Tensor& slots, const Tensor* scale,
             const Tensor* bias, Tensor& out, void* workspace, i64 workspace_bytes) {
  REQ(x.dt == F16 || x.dt == BF16, "x must be bf16/fp16, not %s", dname(x.dt));
  REQ(x.dim() == 2 && a.dim() == 3 && b.dim() == 3, "x must be [N,K], a [L,R,K], b [L,O,R]");
  const i64 N = x.size(0), K = x.size(1), L = a.size(0), R = a.size(1), O = b.size(1);
  REQ(N <= kMostRows, "%lld rows: at most 2^27", (long long)N);
  REQ(L > 0 && L <= (1 << 16), "%lld adapters: 1 to 2^16", (long long)L);
  REQ(R > 0 && R % 8 == 0 && R <= kHighestRank, "rank %lld: a positive multiple of 8, at most %d", (long long)R, kHighestRank);
  for (i64 c : {O, K}) REQ(c > 0 && c % 8 == 0 && c <= (1 << 20), "%lld channels: a positive multiple of 8, at most 2^20", (long long)c);
  check(x, "x", x.dt, {N, K});
  check(a, "a", x.dt, {L, R, K});
  check(b, "b", x.dt, {L, O, R});
  if (w) check(*w, "w", x.dt, {O, K});
  if (y) check(*y, "y", x.dt, {N, O});
  check(out, "out", x.dt, {N, O});
  REQ(slots.dt == I32 && slots.numel() == N && (slots.p || N == 0) && (uintptr_t)slots.p % 4 == 0, "slots must be int32 [%lld] and not null",
      (long long)N);
  if (scale) REQ(scale->dt == F32 && scale->numel() == L && scale->p, "scale must be F32 [%lld]", (long long)L);
  if (bias)
    REQ(bias->numel() == O && bias->p && (bias->dt == F32 || bias->dt == F16 || bias->dt == BF16), "bias must have %lld elements", (long long)O);
  for (const Tensor* t : {&x, &a, &b, &slots, w, scale, bias})
    if (t) mx_apart(out.p, out.bytes(), t->p, t->bytes(), "out");
  if (y) REQ(y->p == out.p || !mx_overlap(y->p, y->bytes(), out.p, out.bytes()), "out must be y or apart from it");
  if (N == 0) return;
  // Rows go in as many parts as it takes for the workspace to hold a part's first product; where all of it would be large, parts lose nothing
  const i64 product = w ? adapter_product_bytes(N, K, O) : 0, all = inner_bytes(N, R) + product, least = adapter_workspace(N, R, w ? K : 0, O);
  const i64 given = workspace ? workspace_bytes : all <= kWhole ? all : least, need = given < all ? std::max(least, given) : all;
  if (workspace) {
    for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &a, &b, &slots, w, y, scale, bias, &out})
      if (t) mx_apart(t->p, t->bytes(), workspace, (size_t)need, "the workspace");
  }
  MxWorkspace ws(workspace, workspace_bytes, need);
  const i64 part = need < all ? (need - product) / 16 * 16 / inner_row_bytes(R) : N;
  for (i64 n = 0; n < N; n += part) {
    const i64 rows = std::min(part, N - n), inner = inner_bytes(rows, R);
    GroupArgs g{};
    g.m = w ? x.ptr<uint16_t>() + n * K : y->ptr<uint16_t>() + n * O;
    g.c = w ? w->p : nullptr;
    g.bias = bias ? bias->p : nullptr;
    g.bias_dt = bias ? bias->dt : F32;
    g.out = out.ptr<uint16_t>() + n * O;
    g.N = rows;
    g.G = 1;
    g.K = (int)K;
    g.O = (int)O;
    uint16_t* h = inner ? (uint16_t*)ws.p : nullptr;
    float* back = inner ? (float*)(h + rows * R * 2) : nullptr;
    g.ad = AdapterPart{b.p, h, back, slots.ptr<int32_t>() + n, (int)L, (int)R, x.ptr<uint16_t>() + n * K, a.p, scale ? scale->ptr<float>() : nullptr};
    if (h) x.dt == F16 ? launch_in<true>(g.ad, rows, (int)K, h, back) : launch_in<false>(g.ad, rows, (int)K, h, back);
    if (w) {
      const i64 deep = adapter_product_bytes(rows, K, O);  // (that of a part may be more than all rows': undivided then)
      adapter_product(g, x.dt, deep && deep <= product ? ws.p + inner : nullptr);
    } else if (x.dt == F16) {
      launch_add<true>(g);
    } else {
      launch_add<false>(g);
    }
  }
}
}  // namespace

i64 adapter_workspace(i64 N, i64 R, i64 K, i64 O) {
  // half of the rows, and at least one
  const i64 some = adapter_fused(N, R) ? 0 : (std::max((N + 1) / 2 * R * 4, inner_row_bytes(R)) + 255) / 256 * 256;
  return some + (K ? adapter_product_bytes(N, K, O) : 0);
}

void adapter_linear(const Tensor& x, const Tensor& w, const Tensor& a, const Tensor& b, const Tensor& slots, const Tensor* scale,
                    const Tensor* bias, Tensor& out, void* workspace, i64 workspace_bytes) {
  adapter(x, &w, nullptr, a, b, slots, scale, bias, out, workspace, workspace_bytes);
}
void adapter_add(const Tensor& y, const Tensor& x, const Tensor& a, const Tensor& b, const Tensor& slots, const Tensor* scale, Tensor& out,
                 void* workspace, i64 workspace_bytes) {
  adapter(x, nullptr, &y, a, b, slots, scale, nullptr, out, workspace, workspace_bytes);
}
