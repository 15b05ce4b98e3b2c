// What the kernels of linear layers with many weights share: the products of groups of rows (group.hip) and the low-rank
// adapters beside one projection (adapter.hip).
//
// v_mfma_f32_16x16x32 multiplies 16 x 32 by 32 x 16 values: lane l supplies row l % 16 of either operand, depths 8 (l / 16) .. + 7, and gets
// column l % 16 and rows 4 (l / 16) + i of the result. The channels' operand (w) is the first and the rows' (x) the second, so a lane has
// 4 channels of one row per product.
#pragma once
#include "ldsdma.h"
#include "mx.h"

namespace {
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr uint32_t kOOR = 0x80000000u;  // past every buffer of these kernels, also with a step's offset added: reads as zeros

template <bool F16>
__device__ __forceinline__ f32x4 mfma(mx_u32x4 a, mx_u32x4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

// 16 rows of 64 depths straight from memory into operands. A load instruction that takes 64 bytes of each of 16 rows gets half of what one that
// takes 128 bytes of each of 8 gets (x and a of 8192 rows by 4096, 64 ranks: 28 us and 17), so one loads the even rows' lines and one the
// odd ones', two lanes beside each other 64 bytes of either row, and change halves afterwards.
struct Lines {
  mx_u32x4 even, odd;
};
// Byte offset of this lane's 16 bytes of the even rows' lines, `row` bytes apart; the odd ones' are a row further
__device__ __forceinline__ uint32_t line_offset(int lane, int row) {
  return (uint32_t)((lane & 14) * row + ((lane & 1) * 4 + (lane >> 4)) * 16);
}
__device__ __forceinline__ int line_depth(int lane) { return ((lane & 1) * 4 + (lane >> 4)) * 8; }  // its first depth of the 64
// Operands of the first and the last 32 depths: lane l has row l % 16, depths 8 (l / 16) .. + 7
__device__ __forceinline__ void operands(const Lines& q, int lane, mx_u32x4& first, mx_u32x4& last) {
  const bool odd = lane & 1;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t away = odd ? q.even[j] : q.odd[j];
    const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)away, 0xB1, 0xf, 0xf, true);  // of lanes 1, 0, 3, 2
    first[j] = odd ? got : q.even[j];
    last[j] = odd ? q.odd[j] : got;
  }
}
}  // namespace

// Adapters of a product's rows: the second of their two products is added to the result
struct AdapterPart {
  const void* b;         // [L,O,R]
  const uint16_t* h;     // the first product, scaled, in halves (inner_tile_place says where; rows without an adapter: anything)
  const float* back;     // what their products are multiplied by: [N,ceil(R/64)] (fp16 only)
  const int32_t* slots;  // [N]
  int L, R;
  const void *x, *a;     // what h is made of where the same kernel makes it (h null): [N,K], [L,R,K]
  const float* scale;    // [L] or null
};
// Where that is: so few rows and ranks that every workgroup reads a for itself, in about the time that it waits for the weights, rather than
// wait for a kernel of its own. us so / in two kernels, 4096 to 4096 channels, bf16: adapter_linear 1 row of 16 ranks 12.2 / 16.6, 1 of 32
// 14.2 / 16.8, 2 of 16 12.9 / 16.2, 4 of 8 16.1 / 15.8; adapter_add 10.2 - 10.3 / 15.8, 4 of 8 11.5 / 15.8. InnerSums holds no more.
constexpr int kFusedRows = 4, kFusedRanks = 32;
inline bool adapter_fused(i64 N, i64 R) { return N <= kFusedRows && N * R <= kFusedRanks; }
struct GroupArgs {
  const void *m, *c, *bias;  // operands of the result's rows and columns: x, w (forward); dy, w (dx); dy, x (dw)
  const int32_t* ends;
  void *out, *db;
  i64 N;
  int G, K, O, bias_dt;
  int tiles_m, tiles_c, per, band, width;
  AdapterPart ad;
  int split;  // parts of the depth, of `elems` results each
  i64 elems;
};

namespace {
// The first product is a sum in fp32 and a factor of the second, whose instructions take 16-bit operands: it goes there as two, a high and a
// low half, whose sum it is to 2^-15 of itself (bf16; one operand alone 2^-8) or 2^-22 (fp16; one alone 2^-11, up to 65504 only).
//
// In fp16 the 64 ranks of a row that share a factor are brought to below 2^15 by a power of two, which their products are multiplied back
// with; their low halves end at 2^-39 of the largest. `largest`: the bits of the largest finite magnitude (an infinity stays one, and must not
// make zeros of the others, which may meet an infinity of the second product).
__device__ __forceinline__ void inner_factors(uint32_t largest, float& to, float& back) {
  const uint32_t e = max(largest >> 23, 15u);
  to = __uint_as_float((268 - e) << 23);  // 2^14 / the largest's power of two; both are normal
  back = __uint_as_float((e - 14) << 23);
}
__device__ __forceinline__ uint32_t finite_bits(float v) {  // of its magnitude; zero for an infinity or NaN
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// Two values. The high half is cut in bf16, where rounding would make infinities of the largest. An infinity or NaN is the high half's alone.
template <bool F16>
__device__ __forceinline__ void halves(float x, float y, uint32_t& high, uint32_t& low) {
  high = F16 ? mx_pack2<F16>(x, y) : __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
  const float dx = x - mx_lo<F16>(high), dy = y - mx_hi<F16>(high);
  low = mx_pack2<F16>(dx == dx ? dx : 0.f, dy == dy ? dy : 0.f);
}
// 16-bit values with zeros for infinities and NaN: what the low half is multiplied by, so that the high half's product alone decides
// what comes of an infinity
template <bool F16>
__device__ __forceinline__ mx_u32x4 finite_only(mx_u32x4 q) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  constexpr uint32_t kExponent = F16 ? 0x7c007c00u : 0x7f807f80u, kStep = F16 ? 0x04000400u : 0x00800080u;
#pragma unroll
  for (int j = 0; j < 4; j++) q[j] &= ~__builtin_bit_cast(uint32_t, __builtin_bit_cast(s16x2, (q[j] & kExponent) + kStep) >> (short)15);
  return q;
}
// Where the high half of rank r of row n stands among the 2 R of all N rows: as the operands are loaded, 16 rows at a time (m where fewer
// are left) and of these 32 ranks' high halves, then their low ones, eight ranks of each row together (64 bytes of 16 rows a load: adapter_add
// [8209, 4096] to 4096 channels, 64 ranks, 92 -> 77 us)
__device__ __forceinline__ int inner_tile_place(int i, int m, int r) { return r / 32 * 64 * m + (r % 32 / 8 * m + i) * 8 + r % 8; }
__device__ __forceinline__ int inner_to_low(int m, int r, int R) { return m * min(32, R - r / 32 * 32); }
// The first product of a wavefront's rows, from row n0 on, from memory: row i's high[c], low[c] are ranks r0 + 32 c + 8 (lane / 16) .. + 7,
// anything where the row has no adapter, so that the loads do not wait for the slots. (Loads past a buffer's end, not branches: around the
// lanes' branches the compiler, short of registers in the tiles' kernel, has copied a value of all lanes for some of them only.)
template <bool F16>
__device__ __forceinline__ auto stored_inner(const GroupArgs& a, i64 n0, int rows, int lane) {
  const int R = a.ad.R, blocks = (R + 63) / 64, n = max(min(rows, 64), 0);
  const auto rh = buffer(a.ad.h + n0 * R * 2, (uint32_t)(n * R * 4));
  const auto rf = buffer(F16 ? a.ad.back + n0 * blocks : nullptr, F16 ? (uint32_t)(n * blocks * 4) : 0u);
  return [=](int i, int r0, int, auto& high, auto& low, float& back) __attribute__((always_inline)) {
    constexpr int RC = sizeof(high) / sizeof(high[0]);
#pragma unroll
    for (int c = 0; c < RC; c++) {
      const int r = r0 + c * 32 + (lane >> 4) * 8;
      const bool in = r < R;
      const int m = min(16, n - i / 16 * 16);
      const uint32_t at = (uint32_t)((i / 16 * 16 * R * 2 + inner_tile_place(i % 16, m, r)) * 2);
      high[c] = __builtin_amdgcn_raw_buffer_load_b128(rh, in ? at : kOOR, 0, 0);
      low[c] = __builtin_amdgcn_raw_buffer_load_b128(rh, in ? at + inner_to_low(m, r, R) * 2 : kOOR, 0, 0);
    }
    if constexpr (F16) back = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rf, (uint32_t)((i * blocks + r0 / 64) * 4), 0, 0));
  };
}
// The first product of up to kFusedRows rows, by NW wavefronts, of which this is number w: its part of the sums, to be added over w
typedef float InnerSums[kFusedRows][kFusedRanks];
template <bool F16, int NW>
__device__ __forceinline__ void inner_products(const GroupArgs& a, int lane, int w, InnerSums& sums) {
  const AdapterPart& p = a.ad;
  const int r16 = lane & 15, g = lane >> 4, S = (a.K + 63) / 64, s0 = S * w / NW, s1 = S * (w + 1) / NW, depth = line_depth(lane), even = r16 & 14;
  const uint32_t off = line_offset(lane, a.K * 2);
  for (int n = 0; n < (int)a.N; n++) {
    const int slot = p.slots[n];
    if (slot < 0 || slot >= p.L) continue;
    const auto rx = buffer((const char*)p.x + (i64)n * a.K * 2, (uint32_t)(a.K * 2));
    const auto ra = buffer((const char*)p.a + (i64)slot * p.R * a.K * 2, (uint32_t)(p.R * a.K * 2));
    for (int r0 = 0; r0 < p.R; r0 += 16) {
      f32x4 acc{};
      constexpr int AT = 8;  // steps on their way together
      for (int k = s0; k < s1; k += AT) {
        Lines qa[AT], qx[AT];
#pragma unroll
        for (int i = 0; i < AT; i++) {
          const bool in = k + i < s1 && (k + i) * 64 + depth < a.K;
          const uint32_t at = off + r0 * a.K * 2;
          qa[i].even = __builtin_amdgcn_raw_buffer_load_b128(ra, in && r0 + even < p.R ? at : kOOR, (k + i) * 128, 0);
          qa[i].odd = __builtin_amdgcn_raw_buffer_load_b128(ra, in && r0 + even + 1 < p.R ? at + a.K * 2 : kOOR, (k + i) * 128, 0);
          qx[i].even = __builtin_amdgcn_raw_buffer_load_b128(rx, in && r16 < 2 ? off : kOOR, (k + i) * 128, 0);
          qx[i].odd = mx_u32x4{};
        }
        __builtin_amdgcn_sched_barrier(0);  // the loads stay together
#pragma unroll
        for (int i = 0; i < AT; i++) {
          mx_u32x4 a0, a1, x0, x1;
          operands(qa[i], lane, a0, a1);
          operands(qx[i], lane, x0, x1);
          acc = mfma<F16>(a0, x0, acc);
          acc = mfma<F16>(a1, x1, acc);
        }
      }
      if (r16 == 0) *(f32x4*)&sums[n][r0 + g * 4] = acc;
    }
  }
}
// The same of rows 0 .. kFusedRows - 1 from the sums of NW wavefronts
template <bool F16, int NW>
__device__ __forceinline__ auto summed_inner(const GroupArgs& a, const InnerSums* sums, int lane) {
  return [&a, sums, lane](int i, int, int slot, auto& high, auto& low, float& back) __attribute__((always_inline)) {
    constexpr int RC = sizeof(high) / sizeof(high[0]), FC = kFusedRanks / 32;  // (there are no ranks past these)
    const float scale = a.ad.scale ? a.ad.scale[max(slot, 0)] : 1.f;
    float v[FC][8];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < FC; c++) {
      const int r = c * 32 + (lane >> 4) * 8;
      const bool in = r < a.ad.R && slot >= 0;
      const int n = in ? i : 0, from = in ? r : 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) t += sums[w][n][from + j];
        v[c][j] = in ? t * scale : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) top = max(top, finite_bits(v[c][j]));
    }
    float to = 1.f;
    if constexpr (F16) inner_factors(mx_max_across32(mx_max_across16(top)), to, back);
#pragma unroll
    for (int c = 0; c < RC; c++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t hi = 0, lo = 0;
        if (c < FC) halves<F16>(v[c][2 * j] * to, v[c][2 * j + 1] * to, hi, lo);
        high[c][j] = hi;
        low[c][j] = lo;
      }
  };
}

// The adapters' second product for up to 64 rows of one wavefront (16 TM rows, the first of them row n0, `rows` of which exist):
// acc[t][u] += b h over tiles t of 16 channels and u of 16 rows. Every adapter that some row has takes its turn, of whose products a
// lane takes its row's (rows of zeros for the others would let an infinity in b reach them), so rows come in any order; those that share
// an adapter share its reading. chan(t, r): the channel of the first operand's row r in tile t, counted from c0, `cols` of which exist.
// inner: a row's first product (stored_inner, summed_inner). Turns first, first + every, ...
template <bool F16, int TC, int TM, class Chan, class Inner>
__device__ __forceinline__ void add_adapters(const GroupArgs& a, f32x4 (&acc)[TC][TM], i64 n0, int rows, int c0, int cols, int lane, Chan&& chan,
                                             Inner&& inner, int first = 0, int every = 1) {
  static_assert(TM <= 4, "a lane a row");
  const AdapterPart& p = a.ad;
  const int r16 = lane & 15, g = lane >> 4;
  const bool here = lane < 16 * TM && lane < rows;
  const auto rs = buffer(p.slots + n0, (uint32_t)(max(min(rows, 64), 0) * 4));
  int mine = (int)__builtin_amdgcn_raw_buffer_load_b32(rs, here ? (uint32_t)(lane * 4) : kOOR, 0, 0);
  mine = here && mine < p.L ? mine : -1;
  int slot[TM];
#pragma unroll
  for (int u = 0; u < TM; u++) slot[u] = __shfl(mine, u * 16 + r16, 64);
  const uint64_t all = __ballot(mine >= 0);
  // 64 ranks and 4 channel tiles at a time; for 64 rows half of either, as registers allow ([8209, 4096] by [4096, 4096], 64 ranks, fp16 306 us;
  // with 4 tiles 310, with 64 ranks 1060)
  constexpr int RC = TM <= 2 ? 2 : 1, TP = TC < 4 ? TC : TM > 2 ? 2 : 4;
  mx_u32x4 high[TM][RC], low[TM][RC];
  float back[TM];
#pragma unroll
  for (int u = 0; u < TM; u++) inner(u * 16 + r16, 0, slot[u], high[u], low[u], back[u]);
  for (int r0 = 0;;) {
    int turn = 0;
    for (uint64_t left = all; left; turn++) {
      const int s = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
      const uint64_t same = __ballot(mine == s);
      left &= ~same;
      if (turn % every != first) continue;
      const auto rb = buffer((const char*)p.b + ((i64)s * a.O + c0) * p.R * 2, (uint32_t)(cols * p.R * 2));
#pragma unroll
      for (int t0 = 0; t0 < TC; t0 += TP) {
        mx_u32x4 b[RC][TP], bf[RC][TP];
#pragma unroll
        for (int c = 0; c < RC; c++) {
          const int r = r0 + c * 32 + g * 8;
          if (c && r0 + c * 32 >= p.R) {
#pragma unroll
            for (int t = 0; t < TP; t++) b[c][t] = bf[c][t] = mx_u32x4{};
            continue;
          }
#pragma unroll
          for (int t = 0; t < TP; t++) {
            const int ch = chan(t0 + t, r16);
            b[c][t] = __builtin_amdgcn_raw_buffer_load_b128(rb, ch < cols && r < p.R ? (uint32_t)((ch * p.R + r) * 2) : kOOR, 0, 0);
          }
        }
#pragma unroll
        for (int c = 0; c < RC; c++)
          if (c == 0 || r0 + c * 32 < p.R) {
#pragma unroll
            for (int t = 0; t < TP; t++) bf[c][t] = finite_only<F16>(b[c][t]);
          }
#pragma unroll
        for (int u = 0; u < TM; u++) {
          if (!(same >> (16 * u) & 0xffff)) continue;
#pragma unroll
          for (int t = 0; t < TP; t++) {
            f32x4 d{};
#pragma unroll
            for (int c = 0; c < RC; c++) {
              if (c && r0 + c * 32 >= p.R) continue;
              d = mfma<F16>(bf[c][t], low[u][c], d);
              d = mfma<F16>(b[c][t], high[u][c], d);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) acc[t0 + t][u][i] += slot[u] == s ? (F16 ? d[i] * back[u] : d[i]) : 0.f;
          }
        }
      }
    }
    r0 += 32 * RC;
    if (r0 >= p.R) break;
#pragma unroll
    for (int u = 0; u < TM; u++) inner(u * 16 + r16, r0, slot[u], high[u], low[u], back[u]);
  }
}
}  // namespace

// out = x w^T + bias + adapters over all N rows (group.hip), without checks; workspace: of that many bytes
void adapter_product(const GroupArgs& a, DT dt, void* workspace);
i64 adapter_product_bytes(i64 N, i64 K, i64 O);
