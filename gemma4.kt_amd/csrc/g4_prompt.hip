// g4_prompt.hip -- attention of several tokens per sequence over a paged key-value
// cache: prompts, their chunks, drafted tokens.
//
// Every row is a token of a sequence and a query head; it sees what g4_paged.hip says,
// causally.  A query tile is up to BM rows of one sequence that share a kv head: its
// consecutive tokens times the heads of that kv head.  Keys and values come in tiles of
// KT tokens through LDS (two buffers, loaded straight to LDS by four of the waves while
// the other is worked on) and are used by all waves; a wave has 16 rows.
//
// Both products are on the matrix cores, transposed, so that a lane stays with one row
// (column lane % 16 of every product):
//   S^T = K Q^T   A = keys from LDS, B = the query's parts, which stay in registers
//   O^T = V^T P^T A = values from LDS, read transposed, B = the weights: a lane's scores
//                 are the weights it needs, since the keys of a product may come in any
//                 order as long as A and B agree
// For BF16 the queries and the weights are three bf16 parts each, exact; for F16 two
// f16 parts (22 bits, and 2^-39 of a query's largest element) of values scaled by a power of
// two, since a third part would add half to the matrix work; an F32 cache takes the fp32
// products.  The running maximum and sum are fp32.  The matrix cores round every sum
// down, so each tile's O^T is summed on its own, added in fp32, and every second tile
// is computed with -P and subtracted: those errors then cancel instead of adding up.
//
// The (kv head, query tile, key tile) units are cut into equal stretches, one per
// persistent workgroup, whatever the lengths, windows and causal triangles are
// (k_prompt_plan counts them; few query tiles are cut so that no stretch has parts of
// two).  A query tile whose key tiles are spread over several stretches leaves (maximum,
// sum, O) of each in a slot, and k_paged_prompt_join adds them.  A row whose sums are not finite (an infinite or NaN key or value among those it meets,
// maybe hidden from it) is computed again by k_paged_prompt_join, from the formula: a
// prompt of nothing but NaN takes 25 times as long as any other.
//
// Operands are read from LDS a few products ahead of their use (a read takes 64 clocks alone,
// more with eight waves reading).
//
// What bounds it, and what it measured (times of all three kernels; the products count
// once, though BF16 takes each three times and F16 twice; a library product of 8192^3 in
// the same type reaches 1086 and 1029 TFLOP/s on the card):
//   8192 tokens, causal, 16/8 heads of 256, BF16    1280 to 1340 us (the clock falls with the
//     matrix instructions, card by card): 410 to 430 TFLOP/s, 1.2 to 1.3 PFLOP/s of matrix
//     instructions, 60% of their cycles.  The transposed reads of values are 16% of the time
//     (441 us for 4096 tokens, 371 with a tile's first operands used throughout)
//   four chunks of 301 to 1100 rows behind up to 12001 tokens, window 4096, 16/4 heads of 128,
//     F16    182 us: 399 TFLOP/s; 4.9 vector instructions to a matrix instruction (the
//     weights of a row are the same work for a head of 128 as for one of 256).  Reads from
//     LDS are 6% of it (188 us on one card, 177 without any)
//   8 sequences of 5 drafted tokens behind 1000 to 16384, 16/8 heads of 256, BF16    92 us,
//     4.3 TB/s: one wave of eight has rows, and computes as long as a tile's 64 KB take
//   1001 tokens in a window of 512, 8/2 heads of 256, F16    44 us: five key tiles a
//     stretch, so as much its start and end, and the two small kernels
#include "g4_paged.hpp"

namespace g4 {

// A query tile: rows row .. row + toks - 1 of the call, the first at position `base`, of a
// sequence with `len` tokens; `count` key tiles, `first` (with those the others are padded
// to) before its own.
struct PromptTile {
  int32_t row;
  int32_t toks;
  int32_t base;
  int32_t seq;
  int32_t len;
  int32_t count;
  int64_t first;
};

struct PromptPlan {
  int32_t *n_tiles;   // query tiles of a kv head part
  int64_t *total;     // their key tiles, those of a stretch, and what a query tile's are padded to
  int32_t *start;     // [wgs][2] the query tile and the unit (kv head part) that a stretch begins in
  PromptTile *tiles;  // [cap]
  uint16_t *odd;      // [cap][units][bm / 16] rows whose sums are not finite, of tiles in one stretch
  float *part;        // [2 * wgs][bm][hs]
  float *ml;          // [2 * wgs][bm][2]
  int32_t cap;
  int32_t wgs;
  int32_t bm;
  int32_t kt;
  int32_t gh;         // query heads of a tile
  int32_t parts;      // head parts of a kv head
  int32_t tt;         // tokens of a query tile
};

// Length and number of its sequence.
G4_DEV int entry_length(const PagedArgs &a, int e, int &seq) {
  seq = a.seqs[e];
  if ((unsigned)seq >= (unsigned)a.kv.max_seqs) {
    seq = 0;
    return 0;
  }
  return min(max(a.kv.lengths[seq], 0), a.kv.max_pages << a.kv.shift);
}

// The key tiles that positions p0 .. p1 see together: the first `st`, then those from a0.
struct KeyTiles {
  int count;
  int st;
  int a0;
};

G4_DEV KeyTiles key_tiles(int p0, int p1, int window, int sinks, int kt) {
  KeyTiles k;
  const int from = window > 0 ? max(0, max(p0, 0) - window + 1) : 0;
  k.st = (min(sinks, from) + kt - 1) / kt;
  k.a0 = max(from / kt, k.st);
  k.count = p1 < 0 ? 0 : k.st + p1 / kt + 1 - k.a0;
  return k;
}

// Key tiles of a stretch.
G4_DEV int64_t prompt_stretch(int64_t total, int wgs) {
  const int64_t per = quotient(total + wgs - 1, wgs);
  return per < 1 ? 1 : per;
}

// The last of n ascending numbers (the first is 0) that is not above x.
template <typename F>
G4_DEV int last_not_above(F at, int n, int64_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at(mid) <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// One workgroup: the query tiles of every sequence in order, with their key tiles, and
// the tile that each stretch begins in.  5.5 us, all of it latency: two loads that depend on
// each other, two or three scans, a search in LDS.
__global__ __launch_bounds__(1024) void k_prompt_plan(PagedArgs a, PromptPlan pl) {
  __shared__ int tiles[1025], wsum[16], rows[1024], ends[1024], seqs[1024], lens[1024];
  __shared__ int counts[1024];
  __shared__ int64_t wsum64[16], firsts[1024];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int status = *a.kv.status;  // looked at once the rest is here too
  int mine = 0;
  bool bad = false;
  if (tid < a.n) {
    const int from = a.row_begin[tid], to = a.row_begin[tid + 1];
    bad = from < 0 || to < from || to > a.n_rows;  // rising, or there were more tiles than the table holds
    rows[tid] = from, ends[tid] = to;
    lens[tid] = entry_length(a, tid, seqs[tid]);
    mine = bad ? 0 : (to - from + pl.tt - 1) / pl.tt;
  }
  if (status != KV_OK) return;
  if (__syncthreads_or(bad)) {
    if (tid == 0) *a.kv.status = KV_BAD_DATA;
    return;
  }
  int x = wave_scan(mine);
  if (lane == 63) wsum[wid] = x;
  __syncthreads();
  for (int w = 0; w < wid; ++w) x += wsum[w];
  tiles[tid + 1] = x;
  if (tid == 0) tiles[0] = 0;
  __syncthreads();
  const int n_tiles = tiles[a.n], units = a.kv.n_kv * pl.parts;  // at most cap tiles
  int64_t before = 0;
  for (int t0 = 0; t0 < n_tiles; t0 += 1024) {
    const int t = t0 + tid;
    PromptTile it = {};
    if (t < n_tiles) {
      int lo = 0, hi = a.n - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tiles[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      const int from = rows[lo], to = ends[lo], tok = (t - tiles[lo]) * pl.tt;
      it.len = lens[lo], it.seq = seqs[lo];
      it.row = from + tok;
      it.toks = min(pl.tt, to - it.row);
      it.base = it.len - (to - from) + tok;
      it.count = key_tiles(it.base, it.base + it.toks - 1, a.window, a.sinks, pl.kt).count;
    }
    int64_t s = it.count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(s, d, 64);
      if (lane >= d) s += y;
    }
    if (lane == 63) wsum64[wid] = s;
    __syncthreads();
    int64_t all = 0, mybase = before;
    for (int w = 0; w < 16; ++w) {
      if (w < wid) mybase += wsum64[w];
      all += wsum64[w];
    }
    if (t < n_tiles) {
      it.first = mybase + s - it.count;
      pl.tiles[t] = it;
      if (t0 == 0) firsts[t] = it.first, counts[t] = it.count;
    }
    before += all;
    __syncthreads();
  }
  int64_t per = prompt_stretch(before * units, pl.wgs);
  int pad = 1;
  if (per > 1 && n_tiles <= 1024 && n_tiles * units <= pl.wgs) {
    // Stretches that end where query tiles do, if that makes them no longer than a second
    // segment would (its queries, first key tile and result take as long as three key tiles):
    // the shortest of four lengths with which every piece has a workgroup.  1001 tokens in a
    // window of 512, 8/2 heads of 256, F16: 42 to 44 us, 49 with equal stretches; 8 sequences of
    // 5 drafted tokens 92 and 101.
    auto wave_total = [](int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); };
    bool aligned = false;
    for (int i = 0; i < 4 && !aligned; ++i) {
      const uint32_t p = (int)min(per, (int64_t)1 << 26) + i;
      int pieces = 0;
      for (int r = lane; r < n_tiles; r += 64) pieces += min((counts[r] + p - 1) / p, 1u << 20);
      aligned = wave_total(pieces) <= pl.wgs / units;
      if (aligned) pad = p;
    }
    if (aligned) {
      per = pad;
      const int mine = tid < n_tiles ? (int)((uint32_t)(counts[tid] + pad - 1) / (uint32_t)pad) : 0;
      const int s = wave_scan(mine);
      if (lane == 63) wsum[wid] = s;
      __syncthreads();
      int base = s - mine;
      before = 0;
      for (int w = 0; w < 16; ++w) {
        if (w < wid) base += wsum[w];
        before += wsum[w];
      }
      before *= pad;
      if (tid < n_tiles) pl.tiles[tid].first = firsts[tid] = (int64_t)base * pad;
      __syncthreads();
    }
  }
  const int64_t all = before * units;
  if (tid == 0) *pl.n_tiles = n_tiles, pl.total[0] = before, pl.total[1] = per, pl.total[2] = pad;
  if (before == 0) return;
  if (n_tiles > 1024) {
    __threadfence_block();  // the tiles, for the search
    __syncthreads();
  }
  for (int w = tid; w < pl.wgs; w += 1024) {
    if (w * per >= all) break;
    const int64_t hu = quotient(w * per, before), rel = w * per - hu * before;
    pl.start[2 * w + 1] = (int)hu;
    pl.start[2 * w] = n_tiles > 1024 ? last_not_above([&](int i) { return pl.tiles[i].first; }, n_tiles, rel)
                                     : last_not_above([&](int i) { return firsts[i]; }, n_tiles, rel);
  }
}

// 16 bytes a lane from src (the same in all lanes) + off to LDS at `to` + 16 * lane.
G4_DEV void load_to_lds(const char *src, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(src)
               : "memory", "m0");
}

// The loads to LDS and the LDS operations of the wave are done; then all waves meet.
G4_DEV void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Operands read ahead of the product that takes them: with four (BF16) or six (F16) 4096 tokens
// of 16/4 heads of 128 take 257 and 221 us, with three 249 and 219, and BF16 spills fewer registers.
// F32 takes four products to an operand's 16 elements: six ahead 203 us for 2048 tokens, three 209.
constexpr int prompt_ahead(int type) { return type == T_F32 ? 6 : 3; }

// Waves of a workgroup: as many as fit a CU with the registers that a row's query, sums and
// weights take (up to 168 a lane for heads up to 128, 256 up to 256, 512 beyond).  For heads up
// to 128 a third wave on a SIMD has work where two wait for LDS and exponentials: 4096 tokens of
// 16/4 heads take 222 us with 12 waves and 247 with 8 for 128 elements in F16, 157 and 188 for
// 64, 258 and 267 for 128 in BF16 (which spills 3 registers), and in F32 649 and 671 for 128
// (which spills 37), 493 and 536 for 96, 346 and 375 for 64; 16 waves
// (128 registers) take as long for 64 elements and spill 35 for 128.  Where F32 has few rows to a
// sequence 8 waves are ahead for 128: 94 us against 117 for eight times 5 rows behind 4000.
constexpr int prompt_waves(int hs) { return hs > 256 ? 4 : hs <= 128 ? 12 : 8; }
constexpr int prompt_kt(int type, int hs) {
  const int es = type == T_F32 ? 4 : 2, kt = 32768 / (hs * es);
  return kt > 64 ? 64 : kt >= 64 ? 64 : kt >= 32 ? 32 : 16;
}

// The swizzles.  A row of LDS is CH = HS * ES / 16 words of 16 bytes, word c of row r
// standing at c ^ k_swz(r) or c ^ v_swz(r).  16 keys' words at one c (an A operand of
// S^T), and 8 rows' pairs of words (a transposed read of values), then lie on different
// banks.  CH is an odd number times 2^z: only its low z bits may be changed.
template <int CH>
struct Swz {
  static constexpr int Z = CH % 16 == 0 ? 4 : CH % 8 == 0 ? 3 : CH % 4 == 0 ? 2 : 0;
  static_assert(Z > 0, "words of a row");
  G4_DEV static int k(int row) { return (row & 15) >> (4 - Z); }
  // pairs of words (16-bit values) or fours (fp32 values, rows 4 apart)
  G4_DEV static int v16(int row) { return 2 * (((row & 15) >> (4 - Z)) & ((1 << (Z - 1)) - 1)); }
  G4_DEV static int v32(int row) { return Z >= 4 ? 4 * ((row & 15) >> 2) : Z == 3 ? 4 * ((row & 7) >> 2) : 0; }
};

template <int TYPE, int HS>
__global__ __launch_bounds__(64 * prompt_waves(HS), prompt_waves(HS) / 4) void k_paged_prompt(PagedArgs a,
                                                                                             PromptPlan pl) {
  using M = Mfma<TYPE>;
  constexpr bool F32 = TYPE == T_F32;
  constexpr int NW = prompt_waves(HS), BM = 16 * NW, KT = prompt_kt(TYPE, HS), ES = F32 ? 4 : 2;
  constexpr int NP = TYPE == T_BF16 ? 3 : TYPE == T_F16 ? 2 : 1;  // parts of a query or weight
  constexpr int STEPS = HS / M::STEP, NT = KT / 16, ND = HS / 16;
  constexpr int CH = HS * ES / 16, ROW = HS * ES, GROUP = 16 * ROW, HALF = KT * ROW;
  constexpr int GW = 4 / NT, IPW = CH / 4 / GW;  // waves that load a 16-token group, 1 KB loads of each
  static_assert(NT * GW == 4 && IPW * GW * 64 == 16 * CH, "loads of a tile");
  using Z = Swz<CH>;
  __shared__ __align__(1024) char lds[4 * HALF];  // [buffer][keys, values][KT][ROW]
  __shared__ int32_t okf[2][NT];                  // the groups' pages are there

  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), hs = kv.hs;
  if (*kv.status != KV_OK) return;
  const int group = a.n_heads / kv.n_kv, units = kv.n_kv * pl.parts, n_tiles = *pl.n_tiles;
  const int64_t per_unit = pl.total[0], per = pl.total[1], total = per_unit * units;
  const int pad = (int)pl.total[2];

  // Workgroups b, b + 8, ... run on one XCD: they take neighbouring stretches, so that
  // the key tiles of a kv head are read into few L2s.
  const int stretch = pl.wgs % 8 == 0 ? (blockIdx.x & 7) * (pl.wgs >> 3) + (blockIdx.x >> 3) : blockIdx.x;
  const int64_t begin = stretch * per, end = min(total, begin + per);

  const int col = lane & 15, g4 = lane >> 4;  // row of the tile's 16; quarter of a step, or of a key tile's 16
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;

  const int64_t layer_rows = (int64_t)a.layer * kv.n_pages * kv.n_kv << kv.shift;

  if (begin >= end) return;
  int tile = __builtin_amdgcn_readfirstlane(pl.start[2 * stretch]), hu = __builtin_amdgcn_readfirstlane(pl.start[2 * stretch + 1]);
  for (int64_t u = begin; u < end; ++tile) {
    if (tile == n_tiles) tile = 0, ++hu;
    const PromptTile it = pl.tiles[tile];
    const int cnt = __builtin_amdgcn_readfirstlane(it.count);
    if (cnt == 0) continue;
    const int j0 = __builtin_amdgcn_readfirstlane((int)(u - hu * per_unit - it.first));
    const int j1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)cnt, j0 + (end - u)));
    const int kvh = __builtin_amdgcn_readfirstlane(hu / pl.parts);
    const int h0 = (hu - kvh * pl.parts) * pl.gh, heads = min(pl.gh, group - h0);
    const int seq = __builtin_amdgcn_readfirstlane(it.seq), len = __builtin_amdgcn_readfirstlane(it.len);
    const int base = __builtin_amdgcn_readfirstlane(it.base), toks = __builtin_amdgcn_readfirstlane(it.toks);
    const int row0 = __builtin_amdgcn_readfirstlane(it.row);
    const KeyTiles kts = key_tiles(base, base + toks - 1, a.window, a.sinks, KT);
    const int32_t *table = kv.table + (int64_t)seq * kv.max_pages;

    // ---- this lane's row
    const int r = wid * 16 + col, tk = r / heads, hd = r - tk * heads;
    const bool row_ok = tk < toks;
    const int pos = row_ok ? base + tk : -1;
    const int seen_from = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int first_tk = wid * 16 / heads, last_tk = min((wid * 16 + 15) / heads, toks - 1);
    const bool wave_on = first_tk < toks && base + last_tk >= 0;  // uniform
    const int wave_lo = base + first_tk, wave_hi = base + last_tk;
    const int wave_from0 = a.window > 0 ? max(0, max(wave_lo, 0) - a.window + 1) : 0;
    const int wave_from = a.window > 0 ? max(0, wave_hi - a.window + 1) : 0;
    const int64_t q_row = ((int64_t)(row0 + tk) * a.n_heads + kvh * group + h0 + hd) * hs;

    // ---- the query's parts, as B operands
    u32x4 qb[NP][STEPS];
    float back;
    {
      const float f = a.scale * LOG2E;
      constexpr int W = F32 ? 4 : 8;
      float x[STEPS][W], top = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int d = s * M::STEP + g4 * W;
        const bool in = row_ok && d < hs;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const float4 v = in ? *(const float4 *)(a.q + q_row + d + i) : make_float4(0, 0, 0, 0);
          x[s][i] = v.x * f, x[s][i + 1] = v.y * f, x[s][i + 2] = v.z * f, x[s][i + 3] = v.w * f;
        }
#pragma unroll
        for (int i = 0; i < W; ++i) top = fmaxf(top, __builtin_fabsf(x[s][i]));
      }
      top = fmaxf(top, __uint_as_float(partner_u32<16>(__float_as_uint(top), lane)));
      top = fmaxf(top, __uint_as_float(partner_u32<32>(__float_as_uint(top), lane)));
      float scale_to;
      split_scale<TYPE>(top, scale_to, back);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
#pragma unroll
        for (int i = 0; i < W; ++i) x[s][i] *= scale_to;
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (F32) qb[p][s][i] = __float_as_uint(x[s][i]);
            else qb[p][s][i] = take_part<TYPE>(x[s][2 * i], x[s][2 * i + 1]);
          }
      }
    }

    f32x4 o[ND];  // the sums so far times the last tile's sign
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -__builtin_inff(), l = 0.f;
    float sign = 1.f;

    // ---- loads of key tiles, by the last four waves: each a group's keys and values, or
    // a part of them
    const int loader = wid - (NW - 4), gi = loader / GW, part = loader % GW;
    auto tile_token = [&](int j) { return (j < kts.st ? j : j - kts.st + kts.a0) * KT; };
    // the table's entry for the wave's group in tile j, read ahead (nothing looks at it
    // until the tile's loads are issued: that would wait for the loads before it)
    auto page_at = [&](int j) {
      const int t = tile_token(j) + gi * 16;
      return table[j < j1 && t < len ? t >> kv.shift : 0];
    };
    int next_page = 0;
    auto issue = [&](int j) {
      const int t = tile_token(j) + gi * 16, buf = (j - j0) & 1;
      int page = __builtin_amdgcn_readfirstlane(next_page);
      if (t >= len || !page_ok(page, kv)) page = -1;
      const int64_t row0 = uniform(
          (layer_rows + (((int64_t)max(page, 0) * kv.n_kv + kvh) << kv.shift) + (t & (kv.page - 1))) * (int64_t)(hs * ES));
      const uint32_t to = buf * 2 * HALF + gi * GROUP + part * IPW * 1024;
      if (part == 0 && lane == 0) okf[buf][gi] = page >= 0;
      // The lane's 16 bytes of load i: word c of a row of the group.  Formed for each tile:
      // kept over the loop these places would take the registers of the sums.
      const int ln = (int)opaque((uint32_t)lane);
      auto from = [&](int i, bool values) {
        const int at = (part * IPW + i) * 64 + ln, row = at / CH, c = at % CH;
        const int swz = !values ? Z::k(row) : F32 ? Z::v32(row) : Z::v16(row);
        return (uint32_t)(row * hs * ES + min((c ^ swz) * 16, hs * ES - 16));
      };
      // Whole rows of a power of two of words: the loads differ from the first one by their
      // rows and a change of the word's low bits.
      constexpr bool POW2 = (CH & (CH - 1)) == 0 && CH <= 64;
      const bool fast = POW2 && hs == HS;
      auto load = [&](const char *src, uint32_t first, uint32_t at, int i, bool values) {
        constexpr int R = 64 / CH > 0 ? 64 / CH : 1;  // rows of a load
        const int row = (part * IPW + i) * R;  // the same in all lanes
        const int swz = !values ? Z::k(row) : F32 ? Z::v32(row) : Z::v16(row);
        load_to_lds(src + row * ROW, first ^ (uint32_t)(swz << 4), at + i * 1024);
      };
      const int lrow = ln / CH, lc = ln % CH;
      if (page >= 0 && fast) {
        const uint32_t first = lrow * ROW + ((lc ^ Z::k(lrow)) << 4);
#pragma unroll
        for (int i = 0; i < IPW; ++i) load(kv.k + row0, first, lds0 + to, i, false);
      } else if (page >= 0) {
#pragma unroll
        for (int i = 0; i < IPW; ++i) load_to_lds(kv.k + row0, from(i, false), lds0 + to + i * 1024);
      }
      if (page >= 0 && t + 16 <= len) {
        if (fast) {
          const uint32_t first = lrow * ROW + ((lc ^ (F32 ? Z::v32(lrow) : Z::v16(lrow))) << 4);
#pragma unroll
          for (int i = 0; i < IPW; ++i) load(kv.v + row0, first, lds0 + HALF + to, i, true);
        } else {
#pragma unroll
          for (int i = 0; i < IPW; ++i) load_to_lds(kv.v + row0, from(i, true), lds0 + HALF + to + i * 1024);
        }
      } else {
        // rows that hold no token: zeros, since a weight of zero does not silence a NaN
#pragma unroll
        for (int i = 0; i < IPW; ++i) {
          const int row = ((part * IPW + i) * 64 + ln) / CH;
          u32x4 v = *(const u32x4 *)(kv.v + row0 + from(i, true));
          const bool in = page >= 0 && t + row < len;
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = in ? v[x] : 0u;
          *(u32x4 *)(lds + HALF + to + i * 1024 + lane * 16) = v;
        }
      }
      next_page = page_at(j + 1);
    };

    f32x4 s[NT];                                     // scores: s[n][i] of key 16 n + 4 g4 + i, then weights
    u32x4 pb[F32 ? 1 : NP][F32 ? 1 : (NT + 1) / 2];  // the weights' parts
    float shrunk = 0.f;                              // what the sums so far shrink by
    uint32_t there = 0;                              // groups of the scored tile whose pages are there
    bool scored = false, weighted = false;           // s holds a tile's scores; its weights wait for the values

    auto score = [&](int j) {
      const int t0 = tile_token(j), buf = (j - j0) & 1;
      scored = wave_on && t0 <= wave_hi && (t0 + KT > wave_from0 || t0 < a.sinks);  // else nothing is seen
      if (!scored) return;
      there = 0;
#pragma unroll
      for (int n = 0; n < NT; ++n) there |= (uint32_t)__builtin_amdgcn_readfirstlane(okf[buf][n]) << n;
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
      // the steps' places in a row: four patterns of its low bits.  They are formed ahead,
      // since an address formed between products waits for the one that had its register.
      typedef __attribute__((address_space(3))) const u32x4 *words;
      uint32_t pat[4];
      const int at_col = (int)opaque((uint32_t)col);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pat[i] = lds0 + buf * 2 * HALF + at_col * ROW + (((4 * i) ^ g4 ^ Z::k(at_col)) << 4);
        asm volatile("" : "+v"(pat[i]));
      }
      constexpr int N = STEPS * NT, A = prompt_ahead(TYPE);
      u32x4 k[A + 1];
      auto read = [&](int i) {
        const int st = i / NT;
        k[i % (A + 1)] = *(words)(uintptr_t)(pat[st & 3] + (i % NT * 16 * ROW + (st >> 2) * 256));
      };
#pragma unroll
      for (int i = 0; i < A; ++i) read(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + A < N) read(i + A);
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) s[i % NT] = M::step(k[i % (A + 1)], qb[p][i / NT], s[i % NT]);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // the read behind the first product
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    auto weigh = [&](int j) {
      weighted = scored;
      if (!scored) return;
      scored = false;
      const int t0 = tile_token(j);
      const bool full = there == (1u << NT) - 1 && t0 + KT - 1 <= wave_lo && (t0 >= wave_from || t0 + KT - 1 < a.sinks);
      if (!full) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = t0 + n * 16 + 4 * g4 + i;
            const bool seen = (there >> n & 1) && t <= pos && (t >= seen_from || t < a.sinks);
            s[n][i] = seen ? s[n][i] : -__builtin_inff();
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][i]);
      top = fmaxf(top, __uint_as_float(partner_u32<16>(__float_as_uint(top), lane)));
      top = fmaxf(top, __uint_as_float(partner_u32<32>(__float_as_uint(top), lane)));
      top = fmaxf(m, top * back);
      // weights of F16 stand 2^14 higher, so that the second part of a small one is not subnormal
      const float up = TYPE == T_F16 ? 14.f : 0.f;
      const float zero = top == -__builtin_inff() ? 0.f : top - up;
      shrunk = __builtin_amdgcn_exp2f(m - (zero + up));
      m = top;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][i], back, -zero));  // the product is exact
          sum += w;
          s[n][i] = F32 ? w * sign : w;
        }
      l = __builtin_fmaf(l, shrunk, sum);
      if constexpr (!F32) {
        const uint32_t flip = sign < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int n = 0; n < NT / 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = 2 * n + (i >> 1), x = 2 * (i & 1);
            float w0 = s[k][x], w1 = s[k][x + 1];
            if constexpr (TYPE == T_F16) {
              // the first part truncated, the remainder exact, the second to nearest
              const auto hi = __builtin_amdgcn_cvt_pkrtz(w0, w1);
              typedef float f32x2 __attribute__((ext_vector_type(2)));
              typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
              const f16x2 lo = __builtin_convertvector(
                  (f32x2{__builtin_fmaf((float)hi[0], -1.f, w0), __builtin_fmaf((float)hi[1], -1.f, w1)}), f16x2);
              pb[0][n][i] = __builtin_bit_cast(uint32_t, hi) ^ flip;
              pb[1][n][i] = __builtin_bit_cast(uint32_t, lo) ^ flip;
            } else {
#pragma unroll
              for (int p = 0; p < NP; ++p) pb[p][n][i] = take_part<TYPE>(w0, w1) ^ flip;
            }
          }
      }
    };

    // O^T = shrunk O^T + V^T P^T, o holding the sums times the last tile's sign
    auto add_values = [&](int j) {
      if (!weighted) return;
      weighted = false;
      const int buf = (j - j0) & 1;
      if constexpr (F32) {
        const char *vt_lds = lds + buf * 2 * HALF + HALF;
        const int vx = Z::v32(4 * g4);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          f32x4 t = {0.f, 0.f, 0.f, 0.f};
          const int word = ((4 * d) ^ vx) + (col >> 2);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float v = *(const float *)(vt_lds + (n * 16 + 4 * g4 + i) * ROW + word * 16 + 4 * (col & 3));
              t = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s[n][i], t, 0, 0, 0);
            }
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] = __builtin_fmaf(o[d][i], -shrunk, t[i]);
        }
      } else {
        const int at_col = (int)opaque((uint32_t)col), row = 4 * g4 + (at_col >> 2), vx = ((at_col & 3) >> 1) ^ Z::v16(row);
        const uint32_t v_at = lds0 + buf * 2 * HALF + HALF + row * ROW + 8 * (at_col & 1);
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 *tr;
        union Operand {
          s16x4 h[2];
          u32x4 w;
        };
        // 16 elements of the head after the other, over 32 keys a product
        constexpr int N = ND * NT / 2, A = prompt_ahead(TYPE);
        Operand v[A + 1];
        uint32_t pat[8];  // as for the keys
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pat[i] = v_at + (((2 * i) ^ vx) << 4);
          asm volatile("" : "+v"(pat[i]));
        }
        auto read = [&](int i) {
          const int d = i / (NT / 2), n = i % (NT / 2);
          const uint32_t at = pat[d & 7] + (d >> 3) * 256 + n * 2 * GROUP;
          v[i % (A + 1)].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(uintptr_t)at);
          v[i % (A + 1)].h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(uintptr_t)(at + GROUP));
        };
        f32x4 t[2];  // a sum is added while the next one is formed
#pragma unroll
        for (int i = 0; i < A; ++i) read(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int d = i / (NT / 2), n = i % (NT / 2);
          if (i + A < N) read(i + A);
          if (n == 0) t[d & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) t[d & 1] = M::step(v[i % (A + 1)].w, pb[p][n], t[d & 1]);
          if (n == NT / 2 - 1 && d > 0)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[d - 1][x] = __builtin_fmaf(o[d - 1][x], -shrunk, t[(d - 1) & 1][x]);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) o[ND - 1][x] = __builtin_fmaf(o[ND - 1][x], -shrunk, t[(ND - 1) & 1][x]);
      }
      sign = -sign;
    };

    // The loads of a tile's successor take their waves a while to issue.  The other waves
    // of their SIMDs begin with the tile at once and so stay ahead: one has the matrix
    // cores while another forms weights.
    if (loader >= 0) next_page = page_at(j0);
    tile_barrier();  // the last segment's tiles are done with
    if (loader >= 0) issue(j0);
    for (int j = j0; j < j1; ++j) {
      tile_barrier();  // tile j is here, and everyone is done with tile j - 1
      if (loader >= 0 && j + 1 < j1) issue(j + 1);
      score(j);
      weigh(j);
      add_values(j);
    }

    // ---- the segment's result
    l += __uint_as_float(partner_u32<16>(__float_as_uint(l), lane));
    l += __uint_as_float(partner_u32<32>(__float_as_uint(l), lane));
    const bool whole = j0 == 0 && j1 == cnt;
    if (wave_on || first_tk < toks) {
      const float fix = -sign;  // the last tile's sign
      if (whole) {
        const float inv = l == 0.f ? 0.f : fix / l;
        bool odd = !(l < __builtin_inff());
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const int at = d * 16 + 4 * g4;
          const float4 v = l == 0.f ? make_float4(0, 0, 0, 0)
                                    : make_float4(o[d][0] * inv, o[d][1] * inv, o[d][2] * inv, o[d][3] * inv);
          if (row_ok && at < hs) {
            *(float4 *)(a.out + q_row + at) = v;
            odd |= !(__builtin_fabsf(v.x) < __builtin_inff()) || !(__builtin_fabsf(v.y) < __builtin_inff()) ||
                   !(__builtin_fabsf(v.z) < __builtin_inff()) || !(__builtin_fabsf(v.w) < __builtin_inff());
          }
        }
        const uint64_t b = __ballot(odd && row_ok);
        if (lane == 0)
          pl.odd[((int64_t)tile * units + hu) * NW + wid] = (uint16_t)(b | b >> 16 | b >> 32 | b >> 48);
      } else {
        const int64_t slot = 2 * (int64_t)stretch + (u != begin);
        float *part = pl.part + (slot * BM + r) * hs;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const int at = d * 16 + 4 * g4;
          if (row_ok && at < hs) *(float4 *)(part + at) = make_float4(o[d][0] * fix, o[d][1] * fix, o[d][2] * fix, o[d][3] * fix);
        }
        if (g4 == 0 && row_ok) pl.ml[(slot * BM + r) * 2] = m, pl.ml[(slot * BM + r) * 2 + 1] = l;
      }
    }
    u += (j1 == cnt ? padded(cnt, pad) : j1) - j0;
  }
}

// Row `at` of the call's (row, head) pairs from the formula, by a workgroup of four waves: LS lanes share a cached row,
// eight elements a lane, so a wave takes RS rows at a time, U of them in flight.  Each
// group of LS lanes keeps a running maximum, sum and accumulator of the rows it has
// met; they are joined at the end.
template <int TYPE, int HS>
G4_DEV void plain_row(const PagedArgs &a, int64_t at, int kvh, int seq, int pos, float *sm, float *sl, float *so) {
  constexpr int LS = HS / 8, RS = 64 / LS, U = 4;
  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, ql = lane % LS, rl = lane / LS;
  const Seen see = seen_by(pos, a.window, a.sinks);
  const bool live = 8 * ql < kv.hs;
  const int32_t *table = kv.table + (int64_t)seq * kv.max_pages;
  const int64_t head_rows = ((int64_t)a.layer * kv.n_pages * kv.n_kv + kvh) << kv.shift;
  float q[8], acc[8], m = -__builtin_inff(), l = 0.f;
  const float f = a.scale * LOG2E;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = live ? a.q[at * kv.hs + 8 * ql + i] : 0.f;
    acc[i] = 0.f;
  }
  for (int j0 = wid * RS * U; j0 < see.count; j0 += 4 * RS * U) {
    Raw8<TYPE> kr[U], vr[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * RS + rl;
      const int t = j < see.ns ? j : j + see.skip;
      const int page = j < see.count ? table[t >> kv.shift] : -1;
      ok[u] = page_ok(page, kv);
      kr[u].zero(), vr[u].zero();
      if (ok[u] && live) {
        const int64_t row = (head_rows + (((int64_t)page * kv.n_kv) << kv.shift) + (t & (kv.page - 1))) * kv.hs + 8 * ql;
        kr[u].load(kv.k, row);
        vr[u].load(kv.v, row);
      }
    }
    float s[U], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[8], d = 0.f;
      kr[u].floats(k);
#pragma unroll
      for (int i = 0; i < 8; ++i) d = __builtin_fmaf(q[i], k[i], d);
      d = lanes_sum<LS>(d, lane) * f;  // by all lanes of the wave
      s[u] = ok[u] ? d : -__builtin_inff();
      top = fmaxf(top, s[u]);
    }
    const float c = shrink(m, top);
    m = top;
    l *= c;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float e = shrink(s[u], top);
      float v[8];
      vr[u].floats(v);
      l += e;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(e, v[i], acc[i]);
    }
  }
  __syncthreads();
  if (ql == 0) sm[wid * RS + rl] = m, sl[wid * RS + rl] = l;
  __syncthreads();
  float top = -__builtin_inff(), sum = 0.f;
  for (int i = 0; i < 4 * RS; ++i) top = fmaxf(top, sm[i]);
  for (int i = 0; i < 4 * RS; ++i) sum = __builtin_fmaf(sl[i], shrink(sm[i], top), sum);
  const float c = shrink(m, top);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = acc[i] * c;
#pragma unroll
    for (int d = LS; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    if (rl == 0) so[wid * HS + 8 * ql + i] = v;
  }
  __syncthreads();
  for (int d = tid; d < kv.hs; d += 256) {
    const float o = ((so[d] + so[HS + d]) + so[2 * HS + d]) + so[3 * HS + d];
    a.out[at * kv.hs + d] = sum == 0.f ? 0.f : o / sum;
  }
}

// One workgroup per (query tile, kv head part, 16 rows): adds the slots of a tile whose
// key tiles were spread over several stretches, in order, computes rows again that are
// not finite, and writes the zeros of rows that see nothing.  A wave has four rows, and
// their slots' weights a lane each; four slots of four rows are on their way at a time.
// Bound by latency, and by its 104 registers (four workgroups to a CU): 7.5 us for 64 tiles
// of 10 rows, 10.5 us for 30 MB of slots.  Workgroups per boundary between stretches,
// which looked for rows to be done again afterwards, took 2 to 5 us longer.
template <int TYPE, int HS>
__global__ __launch_bounds__(256) void k_paged_prompt_join(PagedArgs a, PromptPlan pl) {
  __shared__ float sm[4 * 8], sl[4 * 8], so[4 * HS];
  __shared__ int32_t bad[16];
  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hs = kv.hs, words = hs / 4;
  const int units = kv.n_kv * pl.parts, tile = blockIdx.x / units, hu = blockIdx.x - tile * units;
  const int status = *kv.status, n_tiles = *pl.n_tiles;
  const PromptTile it = pl.tiles[tile];  // inside the table, if behind the last tile
  const int64_t per_unit = pl.total[0], per = pl.total[1];
  if (status != KV_OK || tile >= n_tiles) return;
  const int group = a.n_heads / kv.n_kv, kvh = hu / pl.parts, h0 = (hu - kvh * pl.parts) * pl.gh;
  const int heads = min(pl.gh, group - h0), r0 = blockIdx.y * 16, r1 = min(r0 + 16, it.toks * heads);
  if (r0 >= r1) return;
  auto out_at = [&](int r, int &tk) {  // the call's (row, head) of the tile's row r
    tk = r / heads;
    return (int64_t)(it.row + tk) * a.n_heads + kvh * group + h0 + (r - tk * heads);
  };
  int tk;
  if (it.count == 0) {
    for (int i = tid; i < (r1 - r0) * words; i += 256)
      *(float4 *)(a.out + out_at(r0 + i / words, tk) * hs + 4 * (i % words)) = make_float4(0, 0, 0, 0);
    return;
  }
  const int64_t ua = hu * per_unit + it.first;
  const int w0 = (int)quotient(ua, per), w1 = (int)quotient(ua + it.count - 1, per);
  if (w0 == w1) {
    const uint32_t odd = pl.odd[(int64_t)blockIdx.x * (pl.bm / 16) + blockIdx.y];
    if (odd == 0) return;
    if (tid < 16) bad[tid] = odd >> tid & 1;
    __syncthreads();
  } else {
    const int n = w1 - w0 + 1, rw = r0 + 4 * wid;  // slots, and the first of the wave's four rows
    const int64_t s0 = 2 * (int64_t)w0 + (ua != w0 * per);
    auto slot = [&](int i) { return (i == 0 ? s0 : 2 * (int64_t)(w0 + i)) * pl.bm; };
    auto row = [&](int j) { return min(rw + j, r1 - 1); };
    if (tid < 16) bad[tid] = 0;
    __syncthreads();
    for (int d0 = 0; d0 < hs; d0 += 256) {
      const int d = d0 + 4 * lane;
      const float *part = pl.part + (d < hs ? d : 0);
      float4 o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = make_float4(0, 0, 0, 0);
      float top = -__builtin_inff(), sum = 0.f;  // of row lane / 16
      for (int i0 = 0; i0 < n; i0 += 16) {
        const int mine = i0 + (lane & 15);
        const float2 ml = *(const float2 *)(pl.ml + (slot(min(mine, n - 1)) + row(lane >> 4)) * 2);
        float x = 0.f;
        for (int k0 = 0; k0 < 16; k0 += 4) {
          if (i0 + k0 >= n) break;
          float4 v[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (i0 + k0 + k < n) {
              const int64_t at = slot(i0 + k0 + k);
#pragma unroll
              for (int j = 0; j < 4; ++j) v[k][j] = *(const float4 *)(part + (at + row(j)) * hs);
            }
          }
          if (k0 == 0) {
            const float m = mine < n ? ml.x : -__builtin_inff();
            const float t = fmaxf(top, lanes16_max(m, lane)), c = shrink(top, t);
            x = shrink(m, t);
            top = t;
            sum = __builtin_fmaf(sum, c, mine < n ? x * ml.y : 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float cj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(c), 16 * j));
              o[j] = make_float4(o[j].x * cj, o[j].y * cj, o[j].z * cj, o[j].w * cj);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (i0 + k0 + k < n) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16 * j + k0 + k));
                o[j].x = __builtin_fmaf(v[k][j].x, w, o[j].x), o[j].y = __builtin_fmaf(v[k][j].y, w, o[j].y);
                o[j].z = __builtin_fmaf(v[k][j].z, w, o[j].z), o[j].w = __builtin_fmaf(v[k][j].w, w, o[j].w);
              }
            }
          }
        }
      }
      sum = lanes_sum<16>(sum, lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sum), 16 * j));
        if (rw + j >= r1 || d >= hs) continue;
        const bool none = s == 0.f;
        const float4 y = make_float4(none ? 0.f : o[j].x / s, none ? 0.f : o[j].y / s, none ? 0.f : o[j].z / s,
                                     none ? 0.f : o[j].w / s);
        *(float4 *)(a.out + out_at(rw + j, tk) * hs + d) = y;
        if (!(__builtin_fabsf(y.x) < __builtin_inff()) || !(__builtin_fabsf(y.y) < __builtin_inff()) ||
            !(__builtin_fabsf(y.z) < __builtin_inff()) || !(__builtin_fabsf(y.w) < __builtin_inff()))
          bad[rw + j - r0] = 1;
      }
    }
    __syncthreads();
  }
  for (int r = r0; r < r1; ++r) {
    if (!bad[r - r0]) continue;
    const int64_t at = out_at(r, tk);
    plain_row<TYPE, HS>(a, at, kvh, it.seq, it.base + tk, sm, sl, so);
  }
}

static int prompt_class(int hs) { return hs <= 64 ? 64 : hs <= 96 ? 96 : hs <= 128 ? 128 : hs <= 192 ? 192 : hs <= 256 ? 256 : 512; }

static size_t prompt_layout(const PagedArgs &a, const DevInfo &dev, char *base, PromptPlan *p) {
  const int hs = prompt_class(a.kv.hs), group = a.n_heads / a.kv.n_kv;
  p->bm = 16 * prompt_waves(hs);
  p->kt = prompt_kt(a.kv.type, hs);
  p->gh = group < p->bm ? group : p->bm;
  p->parts = (group + p->gh - 1) / p->gh;
  p->tt = p->bm / p->gh;
  p->wgs = dev.cu_count;
  p->cap = a.n_rows / p->tt + a.n;
  size_t off = 0;
  auto add = [&](size_t bytes) {
    char *at = base + off;
    off += (bytes + 255) & ~size_t(255);
    return at;
  };
  const size_t cap = (size_t)p->cap, units = (size_t)a.kv.n_kv * p->parts;
  p->n_tiles = (int32_t *)add(4);
  p->total = (int64_t *)add(24);
  p->start = (int32_t *)add(8 * (size_t)p->wgs);
  p->tiles = (PromptTile *)add(sizeof(PromptTile) * cap);
  p->odd = (uint16_t *)add(2 * cap * units * (p->bm / 16));
  p->part = (float *)add(sizeof(float) * 2 * (size_t)p->wgs * p->bm * a.kv.hs);
  p->ml = (float *)add(sizeof(float) * 4 * (size_t)p->wgs * p->bm);
  return off;
}

size_t prompt_scratch_bytes(const PagedArgs &a, const DevInfo &dev) {
  PromptPlan p;
  return prompt_layout(a, dev, nullptr, &p);
}

template <int TYPE, int HS>
static hipError_t launch_tiles(const PagedArgs &a, const PromptPlan &p, hipStream_t s) {
  hipLaunchKernelGGL((k_paged_prompt<TYPE, HS>), dim3(p.wgs), dim3(64 * prompt_waves(HS)), 0, s, a, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  constexpr int JHS = HS == 96 ? 128 : HS == 192 ? 256 : HS;
  hipLaunchKernelGGL((k_paged_prompt_join<TYPE, JHS>), dim3(p.cap * a.kv.n_kv * p.parts, p.bm / 16), dim3(256), 0, s, a, p);
  return hipGetLastError();
}

template <int TYPE>
static hipError_t launch_tiles(const PagedArgs &a, const PromptPlan &p, hipStream_t s) {
  switch (prompt_class(a.kv.hs)) {
    case 64: return launch_tiles<TYPE, 64>(a, p, s);
    case 96: return launch_tiles<TYPE, 96>(a, p, s);
    case 128: return launch_tiles<TYPE, 128>(a, p, s);
    case 192: return launch_tiles<TYPE, 192>(a, p, s);
    case 256: return launch_tiles<TYPE, 256>(a, p, s);
    default: return launch_tiles<TYPE, 512>(a, p, s);
  }
}

hipError_t launch_prompt(const PagedArgs &a, const DevInfo &dev, char *scratch, hipStream_t s) {
  PromptPlan p;
  prompt_layout(a, dev, scratch, &p);
  hipLaunchKernelGGL(k_prompt_plan, dim3(1), dim3(1024), 0, s, a, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.kv.type == T_F32) return launch_tiles<T_F32>(a, p, s);
  if (a.kv.type == T_F16) return launch_tiles<T_F16>(a, p, s);
  return launch_tiles<T_BF16>(a, p, s);
}

}  // namespace g4
