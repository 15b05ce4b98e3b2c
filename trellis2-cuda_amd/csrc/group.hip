// Products of groups of rows with a weight matrix each, and their gradients. Rows ends[g-1] .. ends[g] - 1 are group g's.
//   forward  y[n] = W_g x[n] + b_g        dx[n] = W_g^T dy[n]        dW_g = sum over g's rows of dy[n] x[n]^T, db_g = sum of dy[n]
#include "group.h"

#include <algorithm>
#include <type_traits>

namespace {
enum { FORWARD = GROUP_FORWARD, DX = GROUP_DX, DW = GROUP_DW };
enum { OUT_16 = 0, OUT_F32 = 1 };
// A workgroup's tiles, one after another. Every wavefront finds them for itself, with a lane a group, 64 groups at a time.
//
// Rows' products: the tiles of all groups stand in one list, a group's in bands of `band` columns, row by row within a band. Each XCD
// takes a contiguous eighth of it, its workgroups every W-th tile of that, so that the tiles that run beside each other on it share
// operands in its L2.
// dw: tiles are as deep as their group is long, so the longest groups come first (up to 64 groups; more are short), in rounds of W tiles
// a XCD that run to and fro; each XCD takes a contiguous eighth of every group's tiles (where they are many, and whole in depth).
//
// The last round of an XCD's W workgroups may have few tiles left: where at most a quarter of them would have one, these are taken in
// QUARTERS (of half the rows and columns) after the whole ones, which take two fifths of a whole one's time, and where at most half of them
// would, in HALVES (of the rows), which take three fifths ([2560, 2048] by [2048, 2048]: 32 us,
// 40 in quarters; [4099, 1416] by 16 groups of [1416, 1032], dx: 28 and 37).
//
// A few deep tiles are each taken in `split` parts of the depth, whose fp32 sums a second kernel adds (split_of says when).
enum { WHOLE = 0, HALVES = 1, QUARTERS = 2, ALL = 3 };
struct TilePlace {
  i64 first = 0;  // the group's first row
  int count = 0, g = 0, tm = 0, tc = 0;
  int part = 0;  // of the depth
};
template <int OP, int BM, bool ONE, int PART>  // ONE: one group, of all rows; BM: rows of a whole tile (at counts pieces)
struct Tiles {
  const GroupArgs& a;
  int lane, first, count, key;  // of the lane's group among the first 64; key: tiles up to its end, or (dw) its place in the order
  int W, round = 0;
  i64 begin;     // this XCD's first part of a tile
  i64 end, cut;  // how many it has, and where those begin that are taken in pieces

  __device__ __forceinline__ Tiles(const GroupArgs& a_, int lane_) : a(a_), lane(lane_), W(gridDim.x / 8) {
    key = chunk(0);
    if constexpr (OP == DW) {
      int place = 0;
      for (int i = 0; i < min(a.G, 64); i++) {
        const int c = __builtin_amdgcn_readlane(count, i);
        place += c > count || (c == count && i < lane) ? 1 : 0;
      }
      key = lane < a.G ? place : -1;
      const i64 per = (i64)a.tiles_m * a.tiles_c;
      begin = 0;
      end = a.per ? (i64)a.per * a.G : (per * a.G * a.split + 7) / 8;
    } else {
      i64 total = __builtin_amdgcn_readlane(key, 63);
      if (a.G > 64) {
        for (int g0 = 64; g0 < a.G; g0 += 64) total += __builtin_amdgcn_readlane(chunk(g0), 63);
        key = chunk(0);
      }
      total = min(total, a.N / BM + a.G);  // (only ends that fall, which is not allowed, have groups of more)
      const i64 all = total * a.tiles_c * a.split, per = (all + 7) / 8;
      begin = blockIdx.x % 8 * per;
      end = max(min(per, all - begin), (i64)0);
    }
    const i64 rest = end % W;
    cut = end;
    if (PART == WHOLE ? rest * 2 <= W : PART == HALVES ? rest * 4 > W && rest * 2 <= W : PART == QUARTERS && rest * 4 <= W) cut -= rest;
    if constexpr (PART == WHOLE) end = cut;
  }
  __device__ __forceinline__ bool any() const { return PART == WHOLE || PART == ALL ? end > 0 : cut < end; }
  // The lane's group of those from g0 on, its rows inside [0, N) whatever ends holds; the tiles of all up to it
  __device__ __forceinline__ int chunk(int g0) {
    const int g = g0 + lane, N = (int)a.N;
    if constexpr (ONE) {
      first = 0;
      count = lane ? 0 : N;
      return (int)(((i64)N + BM - 1) / BM);
    }
    first = g > 0 && g < a.G ? min(max(a.ends[g - 1], 0), N) : 0;
    count = max((g < a.G ? min(max(a.ends[g], 0), N) : 0) - first, 0);
    int sum = (int)(((i64)count + BM - 1) / BM);
    if constexpr (OP == DW) return sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int below = __shfl_up(sum, d, 64);
      sum += lane >= d ? below : 0;
    }
    return sum;
  }
  __device__ __forceinline__ void group(TilePlace& at, int g0, int who) {
    at.g = g0 + who;
    at.first = __builtin_amdgcn_readlane(first, who);
    at.count = __builtin_amdgcn_readlane(count, who);
  }
  __device__ __forceinline__ bool next(TilePlace& at) {  // (the same in every lane, which the compiler does not see)
    const bool more = __builtin_amdgcn_readfirstlane(find(at));
    round = __builtin_amdgcn_readfirstlane(round);
    at.first = __builtin_amdgcn_readfirstlane((int)at.first);
    at.count = __builtin_amdgcn_readfirstlane(at.count);
    at.g = __builtin_amdgcn_readfirstlane(at.g);
    at.tm = __builtin_amdgcn_readfirstlane(at.tm);
    at.tc = __builtin_amdgcn_readfirstlane(at.tc);
    at.part = __builtin_amdgcn_readfirstlane(at.part);
    return more;
  }
  __device__ __forceinline__ bool find(TilePlace& at) {
    const int k = blockIdx.x / 8;
    for (;;) {
      const i64 start = (i64)round * W;
      i64 l = start + k;
      int which = 0;
      if constexpr (PART == HALVES || PART == QUARTERS) {
        const int across = PART == HALVES || (OP == FORWARD ? a.O : a.K) <= a.width / 2 ? 1 : 2;  // (a narrow result has none to the right)
        which = (int)(l % (2 * across));
        l = cut + l / (2 * across);
        if (cut + start / (2 * across) >= end) return false;
        which = across == 1 ? which * 2 : which;
      } else {
        if (OP == DW && (round & 1)) l = start + W - 1 - k;
        if (start >= end) return false;
      }
      round++;
      if (l >= end) continue;
      if (!place(at, begin + l)) continue;
      if constexpr (PART == HALVES || PART == QUARTERS) {
        at.tm = at.tm * 2 + (which >> 1);
        if constexpr (PART == QUARTERS) at.tc = at.tc * 2 + (which & 1);
        if (at.tm * (BM / 2) >= (OP == DW ? a.O : at.count) ||
            (PART == QUARTERS && at.tc * (a.width / 2) >= (OP == FORWARD ? a.O : a.K)))
          continue;
      }
      return true;
    }
  }
  __device__ __forceinline__ bool place(TilePlace& at, i64 l) {
    if constexpr (OP == DW) {
      const int tiles = a.tiles_m * a.tiles_c;
      const i64 u = l * 8 + blockIdx.x % 8, b = u / a.split;
      at.part = a.per ? 0 : (int)(u % a.split);  // (a list of eighths has whole depths)
      const int order = (int)(a.per ? l / a.per : b / tiles);
      const int inside = (int)(a.per ? blockIdx.x % 8 * a.per + l % a.per : b % tiles);
      if (order >= a.G || inside >= tiles) return false;
      at.tm = inside / a.tiles_c;
      at.tc = inside % a.tiles_c;
      if (a.G <= 64) {
        group(at, 0, __builtin_ctzll(__ballot(key == order)));
      } else {
        at.g = order;
        const int N = (int)a.N, s = order ? min(max(a.ends[order - 1], 0), N) : 0;
        at.first = s;
        at.count = max(min(max(a.ends[order], 0), N) - s, 0);
      }
      return true;
    } else {
      at.part = (int)(l % a.split);
      l /= a.split;
      const int row_tile = (int)(l / a.tiles_c);
      int before = 0, upto = key;
      for (int g0 = 0;; g0 += 64) {
        if (g0) upto = chunk(g0);
        const uint64_t past = __ballot(before + upto > row_tile);
        if (past) {
          const int who = __builtin_ctzll(past);
          group(at, g0, who);
          if (who) before += __builtin_amdgcn_readlane(upto, who - 1);
          break;
        }
        if (g0 + 64 >= a.G) return false;
        before += __builtin_amdgcn_readlane(upto, 63);
      }
      if (a.G > 64) chunk(0);  // back to the first groups
      const int tiles = (int)(((i64)at.count + BM - 1) / BM), inside = (int)(l - (i64)before * a.tiles_c);
      const int band = inside / (a.band * tiles) * a.band, width = min(a.band, a.tiles_c - band), rest = inside - band * tiles;
      at.tm = rest / width;
      at.tc = band + rest % width;
      return inside >= 0 && at.tm < tiles;
    }
  }
};

// Tiled products of all three kinds. A workgroup of WC x WM wavefronts has BC = 16 TC WC columns of the result by BM = 16 TM WM rows;
// the depth goes by stages of 64 through slots of LDS (two; three of a half's, five of a quarter's), filled by DMA. An operand whose depth
// is contiguous (x and w of the forward product, dy of dx) lies there as rows of 64 values, its 16-byte pieces permuted (piece c of row q at
// c ^ q % 8), so that eight lanes of neighbouring rows read from distinct banks; one whose depth runs over rows (w of dx, dy and x of dw) as 64 rows, and
// is transposed on its way into registers (ds_read_b64_tr_b16: 16 lanes give the addresses of 4 rows by four pieces of 4 values, lane i gets
// column i of the four rows); piece c of row q is at c ^ (4 (q % 4) + 2 (q / 8 % 2)) there.
//
// The columns' operand is the matrix instruction's first, so a lane has 4 columns of one row of the result per product, and
// which channel each of its 16 rows stands for is free: RUN tiles give a lane 4 RUN consecutive columns.
//
// A step's (32 deep) products go in four quarters, halves of the column tiles by halves of the row tiles, in the order (0, f),
// (0, 1 - f), (1, 1 - f), (1, f) with f = 0, 1 in turn: each quarter changes one operand's half, whose registers were free a quarter
// earlier, so every LDS read is issued one quarter before its use and a wavefront holds one step's operands only. In the
// middle of a stage's second step all wavefronts meet: by then each has read the whole slot, so it is filled again at once.
//
// Bound by the matrix unit at the clock that the card's power leaves (1.7 - 2.0 GHz under this load), and between tiles by the stores, which
// come from all CUs at once and stand before the next tile's DMAs in the counter that both wait for. Measured, bf16: [8192, 8192] by
// [8192, 8192] 0.80 ms, 1.37 PFLOP/s forward and dx, 1.24 dw into fp32, matrix unit busy 70 - 74%; 16411 rows by 8 groups of [4096, 2048] 267 us (1.03 PFLOP/s,
// busy 53%), dx 266, dw into fp32 278.
constexpr int kTileLds = 163840;
template <int OP, bool F16, int OUT, int TC, int TM, int WC, int WM, bool ADAPT, int PART>
__device__ __forceinline__ void multiply_tiles(const GroupArgs& a, uint8_t* lds) {
  constexpr bool MT = OP == DW, CT = OP != FORWARD;  // transposed: the rows' operand, the columns'
  constexpr int NW = WC * WM, BC = 16 * TC * WC, BM = 16 * TM * WM, HC = TC / 2, HM = TM / 2;
  constexpr int RUN = OUT == OUT_F32 ? 1 : 2;
  constexpr int MI = BM / 8 / NW, CI = BC / 8 / NW;  // DMAs per wavefront and stage
  static_assert(MI * 8 * NW == BM && CI * 8 * NW == BC && TC % 2 == 0 && TM % 2 == 0 && HC % RUN == 0, "whole DMAs, halves of whole runs");
  constexpr uint32_t kC = BM * 128, kSlot = (BM + BC) * 128;
  constexpr int NS = kTileLds / kSlot;  // slots

  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wc = wave % WC, wm = wave / WC;
  const int ncols = OP == FORWARD ? a.O : a.K;
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t*)lds;
  struct Part {  // what of the result a tile is
    int m0, c0, rows, cols, from, depth, stages;  // from: its first depth
  };
  auto part_of = [&](const TilePlace& at) __attribute__((always_inline)) {
    Part p;
    p.depth = OP == FORWARD ? a.K : OP == DX ? a.O : at.count;
    p.stages = (int)(((i64)p.depth + 63) / 64);
    const int s0 = (int)((i64)p.stages * at.part / a.split), s1 = (int)((i64)p.stages * (at.part + 1) / a.split);
    p.from = s0 * 64;
    p.depth = max((int)min((i64)p.depth, (i64)s1 * 64) - p.from, 0);
    p.stages = s1 - s0;
    p.m0 = at.tm * BM;
    p.c0 = at.tc * BC;
    p.rows = min(BM, (OP == DW ? a.O : at.count) - p.m0);
    p.cols = min(BC, ncols - p.c0);
    return p;
  };
  Tiles<OP, PART == WHOLE ? BM : 2 * BM, ADAPT, PART> tiles(a, lane), ahead = tiles;
  if (!tiles.any()) return;

  // the channel of the first operand's row p (direct) or of its columns' piece q of tile t
  auto channel = [&](int p) __attribute__((always_inline)) {
    const int t = p / 16 % TC, r = p % 16;
    return p / (16 * TC) * (16 * TC) + t / RUN * (16 * RUN) + r / 4 * (4 * RUN) + t % RUN * 4 + r % 4;
  };
  auto swizzle = [](int row) __attribute__((always_inline)) { return (row & 3) << 2 | (row >> 3 & 1) << 1; };
  // The stages of all tiles are asked for one after another, NS ahead of the products, across the tiles' borders: descriptors and
  // offsets of the one asked for. An operand's first byte, bytes of a row; direct operands have a descriptor of the tile's rows,
  // transposed ones one of the stage's. Past the last tile the DMAs still run but read nothing.
  const int mrow = (OP == FORWARD ? a.K : a.O) * 2, crow = a.K * 2;
  Part asked{};
  int stage = 0;  // of the tile `asked`, next
  const char *mp = nullptr, *cp = nullptr;
  uint32_t moff[MI], coff[CI];
  i32x4 nm{}, nc{};
  int soff = 0;
  uint32_t fill_m = lds0 + wave * (MI * 1024), fill_c = lds0 + kC + wave * (CI * 1024);  // the slot that is filled, where this wavefront's parts go
  auto enter = [&](const TilePlace& at) __attribute__((always_inline)) {
    const Part& p = asked;
    mp = (const char*)a.m + (OP == DW ? (at.first + p.from) * mrow + p.m0 * 2 : (at.first + p.m0) * mrow + p.from * 2);
    cp = (const char*)a.c + (OP == FORWARD ? ((i64)at.g * a.O + p.c0) * crow + p.from * 2
                             : OP == DX    ? ((i64)at.g * a.O + p.from) * crow + p.c0 * 2
                                           : (at.first + p.from) * crow + p.c0 * 2);
    int l = lane;
    asm volatile("" : "+v"(l));  // (computed here, not kept in registers over the loop)
#pragma unroll
    for (int k = 0; k < MI; k++) {
      const int u = (wave * MI + k) * 64 + l;
      if constexpr (MT) {
        const int q = u / (BM / 8), c = u % (BM / 8) ^ swizzle(q);
        moff[k] = c * 8 < p.rows ? (uint32_t)(q * mrow + c * 16) : kOOR;
      } else {
        const int q = u / 8;
        moff[k] = q < p.rows ? (uint32_t)(q * mrow + (u % 8 ^ (q & 7)) * 16) : kOOR;
      }
    }
#pragma unroll
    for (int k = 0; k < CI; k++) {
      const int u = (wave * CI + k) * 64 + l;
      if constexpr (CT) {
        const int q = u / (BC / 8), c = u % (BC / 8) ^ swizzle(q);
        coff[k] = c * 8 < p.cols ? (uint32_t)(q * crow + c * 16) : kOOR;
      } else {
        const int q = u / 8, ch = channel(q);
        coff[k] = ch < p.cols ? (uint32_t)(ch * crow + (u % 8 ^ (q & 7)) * 16) : kOOR;
      }
    }
    if constexpr (!MT) nm = rsrc4(mp, (uint32_t)(p.rows * mrow - p.from * 2));
    if constexpr (!CT) nc = rsrc4(cp, (uint32_t)(p.cols * crow - p.from * 2));
  };
  auto ask = [&]() __attribute__((always_inline)) {
    if (stage == asked.stages) {
      stage = 0;
      TilePlace at;
      bool more;
      do {
        more = ahead.next(at);
        if (more) asked = part_of(at);
      } while (more && !asked.stages);  // an empty group's gradient has none
      if (more) {
        enter(at);
      } else {
        asked.depth = 0;
        asked.stages = -1;  // never again
        nm[2] = nc[2] = 0;
      }
    }
    const int left = min(64, asked.depth - stage * 64);  // of the depth
    auto aim = [&](auto TC_, auto NC, const char* p, int row, int width, uint32_t* off, i32x4& r) __attribute__((always_inline)) {
      constexpr int N = decltype(NC)::value;
      if constexpr (decltype(TC_)::value) {  // rows stage * 64 ..: `left` of them
        r = rsrc4(p + (i64)stage * 64 * row, left > 0 ? (uint32_t)((left - 1) * row + width * 2) : 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = __builtin_amdgcn_readfirstlane(r[i]);  // (in SGPRs, whatever the compiler makes of the branches)
        if (left > 0 && left < 64) {  // the last stage: pieces past the last column read as zeros
#pragma unroll
          for (int k = 0; k < N; k++) {
            const int u = (wave * N + k) * 64 + lane;
            off[k] = (u % 8 ^ (u / 8 & 7)) * 8 < left ? off[k] : kOOR;
          }
        }
      }
    };
    aim(std::bool_constant<MT>{}, std::integral_constant<int, MI>{}, mp, mrow, asked.rows, moff, nm);
    aim(std::bool_constant<CT>{}, std::integral_constant<int, CI>{}, cp, crow, asked.cols, coff, nc);
    soff = __builtin_amdgcn_readfirstlane(left > 0 ? stage * 128 : 0);
    if (asked.stages >= 0) stage++;
  };
  constexpr int DI = MI + CI;  // DMAs of a stage
  auto issue = [&](auto KC) __attribute__((always_inline)) {  // number k of the stage asked for
    constexpr int K = decltype(KC)::value;
    if constexpr (K < MI) dma16_at<K * 1024>(nm, fill_m, moff[K], MT ? 0 : soff);
    else dma16_at<(K - MI) * 1024>(nc, fill_c, coff[K - MI], CT ? 0 : soff);
  };

  f32x4 acc[TC][TM], accb[OP == DW ? TM : 1];
  bool with_db = false;

  // LDS addresses. Direct: row (tile, r16), piece 4 j + g. Transposed: rows 32 j + 8 g + r16 / 4 and 4 further, the piece of 4 columns
  // r16 % 4 of the tile, whose place the swizzle scatters: one address per tile (pair of tiles where a piece holds columns of both).
  const int mq = wm * (16 * TM) + r16, cq = wc * (16 * TC) + r16;
  uint32_t ma[MT ? TM : 2], ca[CT ? TC / RUN : 2];
  auto transposed = [&](int width, int col) __attribute__((always_inline)) {  // col: the lane's first column in the operand's tile
    const int row = 8 * g + r16 / 4;
    return (uint32_t)(row * width * 2 + ((col / 8) ^ swizzle(row)) * 16 + col % 8 * 2);
  };
  if constexpr (MT) {
#pragma unroll
    for (int t = 0; t < TM; t++) ma[t] = lds0 + transposed(BM, wm * (16 * TM) + t * 16 + r16 % 4 * 4);
  } else {
#pragma unroll
    for (int j = 0; j < 2; j++) ma[j] = lds0 + (mq * 8 + ((4 * j + g) ^ (r16 & 7))) * 16;
  }
  if constexpr (CT) {
#pragma unroll
    for (int t = 0; t < TC / RUN; t++) ca[t] = lds0 + kC + transposed(BC, wc * (16 * TC) + t * (16 * RUN) + r16 % 4 * (4 * RUN));
  } else {
#pragma unroll
    for (int j = 0; j < 2; j++) ca[j] = lds0 + kC + (cq * 8 + ((4 * j + g) ^ (r16 & 7))) * 16;
  }
  auto read16 = [](uint32_t at) __attribute__((always_inline)) { return *(__attribute__((address_space(3))) mx_u32x4*)(size_t)at; };
  auto read_tr = [](uint32_t at) __attribute__((always_inline)) {
    return __builtin_bit_cast(mx_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)at));
  };
  auto read_m = [&](mx_u32x4& f, int j, int t) __attribute__((always_inline)) {
    if constexpr (MT) {
      const uint32_t p = ma[t] + j * (32 * BM * 2);
      const mx_u32x2 lo = read_tr(p), hi = read_tr(p + 4 * BM * 2);
      f = mx_u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      f = read16(ma[j] + t * 2048);
    }
  };
  auto read_c = [&](mx_u32x4& f, int j, int t) __attribute__((always_inline)) {
    if constexpr (CT) {
      const uint32_t p = ca[t / RUN] + j * (32 * BC * 2) + t % RUN * 8;
      const mx_u32x2 lo = read_tr(p), hi = read_tr(p + 4 * BC * 2);
      f = mx_u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      f = read16(ca[j] + t * 2048);
    }
  };

  mx_u32x4 fm[2][HM], fc[2][HC];
  constexpr uint32_t kOnes = F16 ? 0x3c003c00u : 0x3f803f80u;
  const mx_u32x4 ones = {kOnes, kOnes, kOnes, kOnes};
  // A quarter's products, with READS LDS reads and DMAS DMAs between them: a wavefront that has its SIMD to itself (or shares it with
  // one at the same place) feeds the matrix unit only if few instructions stand between two products.
  auto quarter = [&](auto BC_, auto CC, auto MC, auto RC, auto&& read, auto DC, auto&& dma) __attribute__((always_inline)) {
    constexpr bool BUSY = decltype(BC_)::value;
    constexpr int hc = decltype(CC)::value, hm = decltype(MC)::value, R = decltype(RC)::value, D = decltype(DC)::value, P = HC * HM;
    if constexpr (BUSY) {
      mx_unroll<P>([&](auto IC) __attribute__((always_inline)) {
        constexpr int i = decltype(IC)::value, u = i / HC, t = i % HC;
        mx_unroll<R>([&](auto KC) __attribute__((always_inline)) {
          if constexpr (decltype(KC)::value * P / 2 / (R ? R : 1) == i) read(decltype(KC)::value);  // the first half: they land by the quarter's end
        });
        mx_unroll<D>([&](auto KC) __attribute__((always_inline)) {
          if constexpr (decltype(KC)::value * P / (D ? D : 1) + P / (2 * (D ? D : 1)) == i) dma(KC);
        });
        f32x4& c = acc[hc * HC + t][hm * HM + u];
        c = mfma<F16>(fc[hc][t], fm[hm][u], c);
        __builtin_amdgcn_sched_barrier(0);
      });
    } else {
      mx_unroll<D>([&](auto KC) __attribute__((always_inline)) { dma(KC); });
    }
    if constexpr (BUSY && OP == DW && hc == 0) {
      if (with_db) {
#pragma unroll
        for (int u = 0; u < HM; u++) accb[hm * HM + u] = mfma<F16>(ones, fm[hm][u], accb[hm * HM + u]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> zero{};
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, HM> hm{};
  constexpr std::integral_constant<int, HC> hc{};
  uint32_t slot = 0;  // where the stage that is multiplied stands
  auto step = [&](auto busy, auto JC) __attribute__((always_inline)) {  // step J of a stage
    constexpr int J = decltype(JC)::value, f = J, JN = 1 - J;
    constexpr std::integral_constant<int, f> mf{};
    constexpr std::integral_constant<int, 1 - f> mo{};
    // DMAs into the slot that the last stage has left: the second half of the one asked for there, or the first half of a new one
    auto count = [](auto PC) {
      constexpr int P = decltype(PC)::value;
      return std::integral_constant<int, P < 0 ? 0 : DI * (P + 1) / 4 - DI * P / 4>{};
    };
    auto dmas = [&](auto PC) __attribute__((always_inline)) {  // fourth P of a stage's
      return [&](auto KC) __attribute__((always_inline)) {
        issue(std::integral_constant<int, DI * decltype(PC)::value / 4 + decltype(KC)::value>{});
      };
    };
    constexpr std::integral_constant<int, J == 0 ? 2 : -1> p1{};
    constexpr std::integral_constant<int, J == 0 ? 3 : -1> p2{};
    constexpr std::integral_constant<int, J == 0 ? -1 : 0> p3{};
    constexpr std::integral_constant<int, J == 0 ? -1 : 1> p4{};
    quarter(busy, zero, mf, hm, [&](int u) __attribute__((always_inline)) { read_m(fm[1 - f][u], J, (1 - f) * HM + u); }, count(p1),
            dmas(p1));
    quarter(busy, zero, mo, hc, [&](int t) __attribute__((always_inline)) { read_c(fc[1][t], J, HC + t); }, count(p2), dmas(p2));
    if constexpr (J == 1) {  // the next stage has landed, and this one is in registers
      wait_vm<(NS - 2) * DI>();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      bare_barrier();
      fill_m = lds0 + slot + wave * (MI * 1024);
      fill_c = lds0 + slot + kC + wave * (CI * 1024);
      const uint32_t on = slot == (NS - 1) * kSlot ? -slot : kSlot;
      slot += on;
#pragma unroll
      for (uint32_t& x : ma) x += on;
#pragma unroll
      for (uint32_t& x : ca) x += on;
      ask();
    }
    quarter(busy, one, mo, hc, [&](int t) __attribute__((always_inline)) { read_c(fc[0][t], JN, t); }, count(p3), dmas(p3));
    quarter(busy, one, mf, hm, [&](int u) __attribute__((always_inline)) { read_m(fm[1 - f][u], JN, (1 - f) * HM + u); }, count(p4),
            dmas(p4));
  };
#pragma unroll
  for (int t = 0; t < NS - 1; t++) {
    ask();
    mx_unroll<DI>([&](auto KC) __attribute__((always_inline)) { issue(KC); });
    fill_m += kSlot;
    fill_c += kSlot;
  }
  ask();
  mx_unroll<DI / 2>([&](auto KC) __attribute__((always_inline)) { issue(KC); });
  wait_vm<(NS - 2) * DI + DI / 2>();  // (of the last stage only the first half is asked for)
  bare_barrier();

  TilePlace at;
  while (tiles.next(at)) {
    const Part p = part_of(at);
    auto loop = [&](auto busy) __attribute__((always_inline)) {
      for (int s = 0; s < p.stages; s++) {
        step(busy, zero);
        step(busy, one);
      }
    };
    if (wm * (16 * TM) >= p.rows || wc * (16 * TC) >= p.cols) {  // nothing of the result is this wavefront's: its share of the DMAs alone
      loop(std::false_type{});
      continue;
    }
    with_db = OP == DW && a.db && at.tc == 0 && wc == 0;
    int bl = lane;
    asm volatile("" : "+v"(bl));
    // the sums begin with the bias
#pragma unroll
    for (int run = 0; run < TC / RUN; run++) {
      float bias[4 * RUN] = {};
      const int c = wc * (16 * TC) + run * (16 * RUN) + (bl >> 4) * (4 * RUN);
      if constexpr (OP == FORWARD) {
        if (a.bias && at.part == 0) mx_params<4 * RUN>(c < p.cols ? a.bias : nullptr, a.bias_dt, (i64)at.g * a.O + p.c0 + c, 0.f, bias);
      }
#pragma unroll
      for (int j = 0; j < RUN; j++)
#pragma unroll
        for (int u = 0; u < TM; u++) acc[run * RUN + j][u] = f32x4{bias[j * 4], bias[j * 4 + 1], bias[j * 4 + 2], bias[j * 4 + 3]};
    }
#pragma unroll
    for (int u = 0; u < (OP == DW ? TM : 1); u++) accb[u] = f32x4{};
    if (p.stages) {
#pragma unroll
      for (int u = 0; u < HM; u++) read_m(fm[0][u], 0, u);
#pragma unroll
      for (int t = 0; t < HC; t++) read_c(fc[0][t], 0, t);
    }
    loop(std::true_type{});

    int el = lane;  // what follows is computed here, not kept in registers over the loop
    asm volatile("" : "+v"(el));
    if (ADAPT && at.part == 0)
      add_adapters<F16>(a, acc, at.first + p.m0 + wm * (16 * TM), p.rows - wm * (16 * TM), p.c0, p.cols, el,
                        [&](int t, int r) __attribute__((always_inline)) { return channel(wc * (16 * TC) + t * 16 + r); },
                        stored_inner<F16>(a, at.first + p.m0 + wm * (16 * TM), p.rows - wm * (16 * TM), el));

    // Two runs' pieces change places between lanes 8 apart, so that a store writes whole 128-byte lines of 8 rows (a run alone is 64 bytes of
    // 16). Where rows are whole lines they go past the caches, which keep the operands ([8192, 1024] by [8192, 1024] 133 -> 116 us); parts of
    // lines are put together there (dw of [1416, 1032] in 16 bits: 32 us, 46 past the caches).
    const i64 obase = at.part * a.elems + (OP == DW ? ((i64)at.g * a.O + p.m0) * a.K : (at.first + p.m0) * ncols);
    constexpr int OS = OUT == OUT_F32 ? 4 : 2;
    const int er = el & 15, eg = el >> 4;
    const bool upper = er >= 8, lines = ((uintptr_t)a.out | (uintptr_t)(ncols * OS)) % 128 == 0;
#pragma unroll
    for (int run = 0; run < TC / RUN; run += 2) {
      const int c = wc * (16 * TC) + (run + upper) * (16 * RUN) + eg * (4 * RUN);
#pragma unroll
      for (int u = 0; u < TM; u++) {
        mx_u32x4 piece[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          if constexpr (OUT == OUT_F32) {
            piece[k] = __builtin_bit_cast(mx_u32x4, acc[run + k][u]);
          } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = acc[(run + k) * 2 + j / 4][u][j % 4];
            piece[k] = mx_pack8<F16>(v);
          }
        }
        mx_u32x4 low, high;  // of rows r16 % 8 and 8 further
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t away = upper ? piece[0][j] : piece[1][j];
          const uint32_t got = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)away, 0x128, 0xf, 0xf, true);  // from 8 lanes on
          low[j] = upper ? got : piece[0][j];
          high[j] = upper ? piece[1][j] : got;
        }
        const int m = wm * (16 * TM) + u * 16 + (er & 7);
        if (c >= p.cols) continue;
        char* to = (char*)a.out + (obase + (i64)m * ncols + p.c0 + c) * OS;
        char* const on = to + (i64)8 * ncols * OS;
        if (lines) {
          if (m < p.rows) __builtin_nontemporal_store(low, (mx_u32x4*)to);
          if (m + 8 < p.rows) __builtin_nontemporal_store(high, (mx_u32x4*)on);
        } else {
          if (m < p.rows) *(mx_u32x4*)to = low;
          if (m + 8 < p.rows) *(mx_u32x4*)on = high;
        }
      }
    }
    if constexpr (OP == DW) {
      if (with_db && eg == 0) {
#pragma unroll
        for (int u = 0; u < TM; u++) {
          const int m = wm * (16 * TM) + u * 16 + er;
          if (m >= p.rows) continue;
          const i64 to = ((i64)at.part * a.G + at.g) * a.O + p.m0 + m;
          if constexpr (OUT == OUT_F32) ((float*)a.db)[to] = accb[u][0];
          else ((uint16_t*)a.db)[to] = (uint16_t)mx_pack2<F16>(accb[u][0], 0.f);
        }
      }
    }
  }
  wait_vm<0>();  // nothing lands in LDS after this
  bare_barrier();
}
template <int OP, bool F16, int OUT, bool ADAPT>
__global__ void __launch_bounds__(512, 2) k_group_tile(GroupArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kTileLds];
  multiply_tiles<OP, F16, OUT, 8, 4, 2, 4, ADAPT, WHOLE>(a, lds);
  multiply_tiles<OP, F16, OUT, 4, 4, 4, 2, ADAPT, HALVES>(a, lds);
  multiply_tiles<OP, F16, OUT, 4, 2, 2, 4, ADAPT, QUARTERS>(a, lds);
}

// Adds the parts of the depth, in order, eight values a thread: the result's first `elems`, then the bias' gradient. Rows of no group stay.
// A kernel of its own, some 7 us behind the first with its reading of what that has just written: the order of the sums is fixed, as one
// of atomics is not.
template <bool F16, bool F32OUT>
__global__ void __launch_bounds__(64) k_group_sum(const float* parts, const float* db_parts, const int32_t* ends, void* out, void* db, i64 elems,
                                                   i64 db_elems, int split, int ncols, int G, i64 N) {
  i64 i = ((i64)blockIdx.x * 64 + threadIdx.x) * 8, each = elems;
  const float* from = parts;
  void* to = out;
  if (i >= elems) {
    i -= elems;
    each = db_elems;
    from = db_parts;
    to = db;
    if (i >= db_elems) return;
  } else if (ends && i / ncols >= min((i64)max(ends[G - 1], 0), N)) {
    return;
  }
  float v[8] = {};
  constexpr int AT = 8;  // parts loaded together
  for (int s = 0; s < split; s += AT) {
    f32x4 q[AT][2];
#pragma unroll
    for (int k = 0; k < AT; k++)
#pragma unroll
      for (int h = 0; h < 2; h++) q[k][h] = s + k < split ? *(const f32x4*)(from + (s + k) * each + i + h * 4) : f32x4{};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < AT; k++)
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += q[k][j / 4][j % 4];
  }
  if constexpr (F32OUT) {
    *(f32x4*)((float*)to + i) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)((float*)to + i + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    *(mx_u32x4*)((uint16_t*)to + i) = mx_pack8<F16>(v);
  }
}

template <int OP, bool F16, int OUT, bool ADAPT = false>
void launch_tile(GroupArgs a) {
  constexpr int BC = 256, BM = 256;
  a.width = BC;
  a.tiles_c = cdiv(OP == FORWARD ? a.O : a.K, BC);
  a.band = 4;
  if (OP == DW) {
    a.tiles_m = cdiv(a.O, BM);
    const i64 each = (i64)a.tiles_m * a.tiles_c;
    a.per = a.split == 1 && each >= 64 ? (int)((each + 7) / 8) : 0;  // (the list of eighths has no parts of the depth)
  }
  const int blocks = mx_device_cus() / 8 * 8;  // one workgroup fits a CU; what has no tile ends at once
  k_group_tile<OP, F16, OUT, ADAPT><<<blocks, 512, 0, stream()>>>(a);
  CK(hipGetLastError());
}
// Few rows: the weights' bytes count, and that many of them are on their way at once. A workgroup has 16 OT channels by up to 16 NT rows of a
// group; each of its 8 wavefronts takes a contiguous eighth of the depth, both operands straight into registers, and the sums meet in
// LDS in a fixed order. With adapters, 4 wavefronts more add them meanwhile; FUSED, they also make the first product.
// Measured: 384 rows by 64 groups of [1416, 2048] fp16 70 us (5.3 TB/s, a large copy's rate: bound by HBM); 2 rows by 16 groups of
// [1024, 1024] 4.9 us and 1 row by [4096, 4096] with an adapter of 16 ranks 11.4 us in the kernel, one trip to memory after another (the
// slots or ends, a, b). The form of 64 rows with adapters is short of registers: 12 wavefronts have 168 each, and it keeps 222 in scratch
// memory (no other of these forms keeps any).
template <bool F16, int OT, int NT, bool ADAPT, bool FUSED>
__global__ void __launch_bounds__(ADAPT ? 768 : 512) k_group_rows(GroupArgs a) {
  constexpr int NW = 8, NA = ADAPT ? 4 : 0, RUN = OT;
  static_assert(OT == 1 || OT == 2, "4 or 8 channels a lane");
  __shared__ f32x4 part[NW + NA][OT * NT][64];
  __shared__ __attribute__((aligned(16))) InnerSums inner[FUSED ? NA : 1];
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  TilePlace at;
  if (Tiles<FORWARD, 16 * NT, ADAPT, ALL> tiles(a, lane); !tiles.next(at)) return;
  const i64 n0 = at.first + at.tm * (16 * NT);
  const int rows = min(16 * NT, at.count - at.tm * (16 * NT)), c0 = at.tc * (16 * OT), cols = min(16 * OT, a.O - c0);
  auto chan = [](int t, int r) __attribute__((always_inline)) { return r / 4 * (4 * RUN) + t * 4 + r % 4; };
  f32x4 acc[OT][NT];
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int u = 0; u < NT; u++) acc[t][u] = f32x4{};
  if (!ADAPT || wave < NW) {
    // every load is a buffer load whose offset is past the end where there is nothing (a row or a channel past the last, depths past K)
    const auto rw = buffer((const char*)a.c + ((i64)at.g * a.O + c0) * a.K * 2, (uint32_t)(cols * a.K * 2));
    const auto rx = buffer((const char*)a.m + n0 * a.K * 2, (uint32_t)(rows * a.K * 2));
    // (the channels' operand as in Lines: row r of a tile is channel chan(t, r))
    const int even = r16 & 14, S = (a.K + 63) / 64, per = (S + NW - 1) / NW, s0 = wave * per, s1 = min(s0 + per, S), depth = line_depth(lane);
    const uint32_t off = depth * 2;
    uint32_t wo[OT][2], xo[NT][2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
#pragma unroll
      for (int t = 0; t < OT; t++) wo[t][k] = chan(t, even + k) < cols ? (uint32_t)(chan(t, even + k) * a.K * 2) + off : kOOR;
#pragma unroll
      for (int u = 0; u < NT; u++) xo[u][k] = u * 16 + even + k < rows ? (uint32_t)((u * 16 + even + k) * a.K * 2) + off : kOOR;
    }
    struct Step {
      Lines w[OT], x[NT];
    };
    auto load = [&](Step& q, int s) __attribute__((always_inline)) {
      const bool in = s * 64 + depth < a.K;
#pragma unroll
      for (int t = 0; t < OT; t++) {
        q.w[t].even = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? wo[t][0] : kOOR, s * 128, 0);
        q.w[t].odd = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? wo[t][1] : kOOR, s * 128, 0);
      }
#pragma unroll
      for (int u = 0; u < NT; u++) {
        q.x[u].even = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? xo[u][0] : kOOR, s * 128, 0);
        q.x[u].odd = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? xo[u][1] : kOOR, s * 128, 0);
      }
    };
    auto multiply = [&](const Step& q) __attribute__((always_inline)) {
      mx_u32x4 w[OT][2], x[2];
#pragma unroll
      for (int t = 0; t < OT; t++) operands(q.w[t], lane, w[t][0], w[t][1]);
#pragma unroll
      for (int u = 0; u < NT; u++) {
        operands(q.x[u], lane, x[0], x[1]);
#pragma unroll
        for (int t = 0; t < OT; t++)
#pragma unroll
          for (int j = 0; j < 2; j++) acc[t][u] = mfma<F16>(w[t][j], x[j], acc[t][u]);
      }
    };
    constexpr int U = 4;  // steps on their way together
    int s = s0;
    for (; s + U <= s1; s += U) {
      Step q[U];
#pragma unroll
      for (int k = 0; k < U; k++) load(q[k], s + k);
      __builtin_amdgcn_sched_barrier(0);  // the loads stay together
#pragma unroll
      for (int k = 0; k < U; k++) multiply(q[k]);
    }
    if (s < s1) {
      Step q[U];
#pragma unroll
      for (int k = 0; k < U; k++)
        if (s + k < s1) load(q[k], s + k);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < U; k++)
        if (s + k < s1) multiply(q[k]);
    }
  } else if constexpr (FUSED) {
    inner_products<F16, NA>(a, lane, wave - NW, inner[wave - NW]);
  } else {
    add_adapters<F16>(a, acc, n0, rows, c0, cols, lane, chan, stored_inner<F16>(a, n0, rows, lane), wave - NW, NA);
  }
  if constexpr (FUSED) {
    __syncthreads();
    if (wave >= NW) add_adapters<F16>(a, acc, n0, rows, c0, cols, lane, chan, summed_inner<F16, NA>(a, inner, lane), wave - NW, NA);
  }
#pragma unroll
  for (int t = 0; t < OT; t++)
#pragma unroll
    for (int u = 0; u < NT; u++) part[wave][t * NT + u][lane] = acc[t][u];
  __syncthreads();
  for (int u = wave; u < NT; u += NW + NA) {
    float v[4 * OT], bias[4 * OT];
#pragma unroll
    for (int t = 0; t < OT; t++) {
      f32x4 c = part[0][t * NT + u][lane];
#pragma unroll
      for (int w = 1; w < NW + NA; w++) c += part[w][t * NT + u][lane];
#pragma unroll
      for (int i = 0; i < 4; i++) v[t * 4 + i] = c[i];
    }
    const int m = u * 16 + r16, c = g * (4 * RUN);
    if (m >= rows || c >= cols) continue;
    mx_params<4 * OT>(a.bias, a.bias_dt, (i64)at.g * a.O + c0 + c, 0.f, bias);
#pragma unroll
    for (int j = 0; j < 4 * OT; j++) v[j] += bias[j];
    uint16_t* to = (uint16_t*)a.out + (n0 + m) * a.O + c0 + c;
    if constexpr (OT == 2) *(mx_u32x4*)to = mx_pack8<F16>(*(float(*)[8])v);
    else *(mx_u32x2*)to = mx_u32x2{mx_pack2<F16>(v[0], v[1]), mx_pack2<F16>(v[2], v[3])};
  }
}
template <bool F16, int OT, int NT, bool ADAPT, bool FUSED = false>
void launch_rows(GroupArgs a) {
  a.split = 1;
  a.tiles_c = cdiv(a.O, 16 * OT);
  a.band = 8;
  const i64 blocks = ((a.N / (16 * NT) + std::min<i64>(a.G, a.N)) * a.tiles_c + 7) / 8 * 8;  // (no more groups than rows have any)
  k_group_rows<F16, OT, NT, ADAPT, FUSED><<<(unsigned)blocks, ADAPT ? 768 : 512, 0, stream()>>>(a);
  CK(hipGetLastError());
}

// Whether a forward product's rows go straight into registers: up to 16 a group on average, or as many as make no more workgroups (of 32
// channels by 32 or 64 rows) than there are CUs. us by rows / in tiles, bf16, [rows, K] by groups of [O, K]: [640, 1024] 32 of 1024
// 21.8 / 21.1 (1280 rows 26.0 / 21.5), [60, 4096] one of 4096 17.4 / 21.2, [100, 4096] 17.9 / 25.3, [200, 4096] 32.1 / 21.6, [100, 1024] one of
// 1024 7.8 / 14.4, [500, 4096] one of 512 17.9 / 18.3. With adapters in any order, 16 ranks, and in four runs, 64 ranks: [32, 4096] one of
// 4096 19 / 38 and 24 / 36, [64, 4096] 39 / 50 and 46 / 38, [100, 4096] 44 / 51 and 51 / 40; [64, 1024] one of 1024 20 / 27 and 19 / 21, [500, 1024]
// 23 / 35 and 23 / 25.
constexpr i64 kCus = 256;  // (a workspace's size follows from it, also where no device is)
int row_tiles(i64 N, i64 G) { return N <= 16 * G ? 1 : N <= 32 * G ? 2 : 4; }  // of 16 rows
bool goes_by_rows(i64 N, i64 G, i64 O) {
  if (N <= 16 * G) return (N / 16 + std::min(G, N)) * cdiv(O, 16) < (1ll << 32) / 768;  // (a launch holds 2^32 threads)
  return N <= 512 * G && (N / (16 * row_tiles(N, G)) + G) * cdiv(O, 32) <= kCus;
}
// Parts of the depth for a product that is a few quartered tiles only, so that they fill the CUs: a stage of 64 of a quarter takes some 0.5 us,
// the second kernel 7 us and more. us whole / in parts of 4, 8 and 16 stages at least: forward [500, 4096] by [512, 4096] 34 / 21 / 18 / 20,
// [300, 2048] by [256, 2048] 21 / 14 / 16 / 19; dw of [512, 512] from 16000 rows 140 / 25 / 25 / 26, 2000 rows 26 / 16 / 17 / 20; with 16
// stages in all ([500, 1024] by [512, 1024]) 14.8 / 15.3.
constexpr int kSplitStages = 32;
int split_of(int op, i64 N, i64 G, i64 K, i64 O) {
  const i64 across = op == DW ? G * cdiv(O, 128) : N / 128 + (G + 1) / 2, quarters = std::max<i64>(across, 1) * cdiv(op == FORWARD ? O : K, 128);
  const i64 stages = op == DW ? cdiv(N, 64 * G) : cdiv(op == FORWARD ? K : O, 64);
  if (quarters > kCus / 2 || stages < kSplitStages) return 1;
  return (int)std::min(kCus / quarters, stages / 8);
}

template <bool ADAPT>
bool few_rows(const GroupArgs& a, DT dt) {
  if (!goes_by_rows(a.N, a.G, a.O)) return false;
  const int tiles = row_tiles(a.N, a.G);
  auto by = [&](auto F) {
    constexpr bool f = decltype(F)::value;
    if constexpr (ADAPT) {
      if (!a.ad.h) return launch_rows<f, 1, 1, true, true>(a);
    }
    // 4 channels a lane for up to 16384 over the groups that have rows, 8 for more. us with 4 / with 8, bf16: one row by [16384, 4096] 27.6 / 29.8, 8 rows by 16
    // groups of [1024, 1024] 8.3 / 8.3, 16 by 16 8.8 / 8.4; beyond, 32 rows by 32 groups of [1024, 1024] 14.2 / 11.7, 64 by 64 of [1416, 1024] 36 / 27
    if (tiles == 1) {
      if (a.O * (a.N < a.G ? a.N : a.G) <= 16 * 1024) launch_rows<f, 1, 1, ADAPT>(a);
      else launch_rows<f, 2, 1, ADAPT>(a);
    } else if (tiles == 2) {
      launch_rows<f, 2, 2, ADAPT>(a);
    } else {
      launch_rows<f, 2, 4, ADAPT>(a);
    }
  };
  dt == F16 ? by(std::true_type{}) : by(std::false_type{});
  return true;
}

i64 out_elems(int op, i64 N, i64 G, i64 K, i64 O) { return op == DW ? G * O * K : N * (op == FORWARD ? O : K); }
// What a tiled product takes of a workspace: the fp32 sums of each part of the depth
i64 split_bytes(int op, i64 N, i64 G, i64 K, i64 O) {
  if (N == 0 || (op == FORWARD && goes_by_rows(N, G, O))) return 0;
  const i64 s = split_of(op, N, G, K, O);
  return s > 1 ? s * 4 * (out_elems(op, N, G, K, O) + (op == DW ? G * O : 0)) : 0;
}
template <int OP, bool ADAPT = false>
void launch(GroupArgs a, DT dt, bool f32, void* workspace) {
  const i64 elems = out_elems(OP, a.N, a.G, a.K, a.O), db_elems = OP == DW && a.db ? (i64)a.G * a.O : 0;
  auto by = [&](auto F, auto T) { launch_tile<OP, decltype(F)::value, decltype(T)::value, ADAPT>(a); };
  constexpr std::integral_constant<int, OUT_16> o16{};
  constexpr std::integral_constant<int, OUT_F32> o32{};
  a.split = 1;
  if (workspace) {
    void *out = a.out, *db = a.db;
    a.split = split_of(OP, a.N, a.G, a.K, a.O);
    a.elems = elems;
    a.out = workspace;
    a.db = db ? (float*)workspace + a.split * elems : nullptr;
    dt == F16 ? by(std::true_type{}, o32) : by(std::false_type{}, o32);
    const unsigned blocks = (unsigned)((elems + db_elems + 511) / 512);
    auto sum = [&](auto F, auto T) {
      k_group_sum<decltype(F)::value, decltype(T)::value><<<blocks, 64, 0, stream()>>>(
          (const float*)a.out, (const float*)a.db, OP == DW || ADAPT ? nullptr : a.ends, out, db, elems, db_elems, a.split,
          OP == FORWARD ? a.O : a.K, a.G, a.N);
    };
    if (f32) sum(std::false_type{}, std::true_type{});
    else if (dt == F16) sum(std::true_type{}, std::false_type{});
    else sum(std::false_type{}, std::false_type{});
    CK(hipGetLastError());
    return;
  }
  if constexpr (OP == DW) {
    if (f32) return dt == F16 ? by(std::true_type{}, o32) : by(std::false_type{}, o32);
  }
  dt == F16 ? by(std::true_type{}, o16) : by(std::false_type{}, o16);
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
// The workspace of a call with the given tensors, its result (and the bias' gradient) last
struct GroupRoom {
  MxWorkspace ws;
  GroupRoom(void* workspace, i64 bytes, i64 need, std::initializer_list<const Tensor*> all) : ws(check(workspace, need, all), bytes, need) {}
  static void* check(void* workspace, i64 need, std::initializer_list<const Tensor*> all) {
    if (workspace)
      for (const Tensor* t : all)
        if (t) mx_apart(t->p, t->bytes(), workspace, (size_t)need, "the workspace");
    return need ? workspace : nullptr;
  }
};
}  // namespace

i64 adapter_product_bytes(i64 N, i64 K, i64 O) { return split_bytes(FORWARD, N, 1, K, O); }
void adapter_product(const GroupArgs& a, DT dt, void* workspace) {
  if (!few_rows<true>(a, dt)) launch<FORWARD, true>(a, dt, false, workspace);
}

i64 group_linear_workspace(int product, i64 N, i64 G, i64 K, i64 O) { return split_bytes(product, N, G, K, O); }

void group_linear(const Tensor& x, const Tensor& w, const Tensor& ends, const Tensor* bias, Tensor& y, void* workspace, i64 workspace_bytes) {
  i64 G, O, K;
  check_16(x, "x");
  const i64 N = rows_in(x, "x");
  check_weights(w, "w", G, O, K);
  REQ(w.dt == x.dt, "w must be of x's type");
  check_rows(x, "x", x.dt, N, K);
  check_rows(y, "out", x.dt, N, O);
  check_ends(ends, G);
  if (bias)
    REQ(bias->numel() == G * O && bias->p && (bias->dt == F32 || bias->dt == F16 || bias->dt == BF16), "bias must have %lld elements",
        (long long)(G * O));
  for (const Tensor* t : {&x, &w, &ends, bias}) apart(y, t, "out");
  if (N == 0) return;
  GroupRoom room(workspace, workspace_bytes, group_linear_workspace(FORWARD, N, G, K, O), {&x, &w, &ends, bias, &y});
  GroupArgs a{x.p, w.p, bias ? bias->p : nullptr, ends.ptr<int32_t>(), y.p, nullptr, N, (int)G, (int)K, (int)O, bias ? bias->dt : F32};
  if (!few_rows<false>(a, x.dt)) launch<FORWARD>(a, x.dt, false, room.ws.p);
}

void group_linear_dx(const Tensor& dy, const Tensor& w, const Tensor& ends, Tensor& dx, void* workspace, i64 workspace_bytes) {
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
  GroupRoom room(workspace, workspace_bytes, group_linear_workspace(DX, N, G, K, O), {&dy, &w, &ends, &dx});
  GroupArgs a{dy.p, w.p, nullptr, ends.ptr<int32_t>(), dx.p, nullptr, N, (int)G, (int)K, (int)O, F32};
  launch<DX>(a, dy.dt, false, room.ws.p);
}

void group_linear_dw(const Tensor& dy, const Tensor& x, const Tensor& ends, Tensor& dw, Tensor* db, void* workspace, i64 workspace_bytes) {
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
    REQ(db->dt == dw.dt && db->numel() == G * O && db->p && (uintptr_t)db->p % 16 == 0,
        "the bias' gradient must have %lld elements of out's type, 16-byte aligned", (long long)(G * O));
    for (const Tensor* t : std::initializer_list<const Tensor*>{&dy, &x, &ends, &dw}) apart(*db, t, "the bias' gradient");
  }
  GroupRoom room(workspace, workspace_bytes, group_linear_workspace(DW, N, G, K, O), {&dy, &x, &ends, &dw, db});
  GroupArgs a{dy.p, x.p, nullptr, ends.ptr<int32_t>(), dw.p, db ? db->p : nullptr, N, (int)G, (int)K, (int)O, F32};
  launch<DW>(a, dy.dt, dw.dt == F32, room.ws.p);
}
