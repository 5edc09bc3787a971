// g4_paged.hip -- decode attention over a paged key-value cache.
//
// Row r of a call is the last token of a sequence; query head h reads kv head
// h / group.  It sees the tokens t <= pos of its sequence with t > pos - window
// (window > 0) or t < sinks, and of those the ones whose page is there:
//   out = sum_t p_t V[t] / sum_t p_t,  p_t = exp(scale q . K[t] - max),
// and zeros where it sees nothing.  One pass over K and V with a running maximum and
// sum; products, statistics and sums are fp32 whatever the cache holds.
#include "g4_paged.hpp"

namespace g4 {

// ---------------------------------------------------------- one token, split ----
//
// Decode attention for a list of sequences of any lengths.  The tokens that a row sees
// are taken in groups of 16 aligned ones, each inside one page; a (row, kv head, up to
// GT of its query heads) has as many units of work as groups.  The units of all of them,
// in order, are cut into equal stretches, one per workgroup, whatever the lengths are:
// they are device data, which each workgroup sums up itself.  Where there are fewer heads than
// workgroups, stretches end where heads do, if they get little longer by it: a stretch
// across two heads costs a second start and end.  Where a stretch holds all
// of a head's groups the result is final; otherwise (maximum, sum, weighted values) goes
// to the stretch's first or second slot and k_paged_join adds the slots of a head.  One
// workgroup per (row, kv head, pair of query heads) left the chip to the longest row: it
// took 936 us for the 64 rows below and 580 us for the one of 8192 tokens.
//
// A wave takes NG groups at a time.  Scores come from the matrix cores: A = the query
// heads, B = 16 keys as they lie in memory.  A head is four rows of A: for a 16-bit
// cache the query's three 16-bit parts, which add up to it (BF16 exactly, F16 to 2^-39 of
// its largest element), for F32 the query
// itself; the products are then exact (F32: rounded once), and a lane's sum over its
// four rows of C is the score of (head lane / 16, key lane % 16).  The queries carry
// scale * log2(e) (split_scale keeps their parts in range).  Values are weighted by the
// vector unit in fp32, eight elements of a row per lane, with the weights handed over
// through the wave's own LDS.  While a tile is worked on, the next one's keys and values
// are on their way: a wave's registers hold both, and LDS only the queries.
//
// What bounds it is the cache's bytes, read once (FETCH_SIZE is 1.00 to 1.09 of K and V),
// where rows are long, and the chain of loads at a stretch's start (lengths, page table,
// keys: about 2000 clocks each) where a stretch is a few groups.  Measured, with its join:
//   4 rows of 20001 to 65536 tokens, 8/2 heads of 256, F32    123 us, 5.3 TB/s
//   64 rows of 200 to 16384 tokens, 32/4 heads of 128, F16    136 us, 3.6 TB/s: with eight
//     heads to a kv head the 64 products of a value lane take as long as its loads
//   1 row of 8192 tokens, 16/8 heads of 256, BF16             21 us, 3.2 TB/s
//   24 rows in a window of 1024, 8/1 heads of 512, BF16       27 us, 1.9 TB/s: two groups a wave
// (a copy's reads alone reach 5.86 TB/s).  Tiles of twice the groups where one workgroup
// fills a CU (512 registers a lane) took 40% longer on the last: the values pass through
// accumulation registers.

// A row's visible tokens as groups: the first gs, then those from g0.
struct Groups {
  int count;
  int gs;
  int g0;
  int from;  // t is seen if t <= pos and (t >= from or t < ns)
  int ns;
};

G4_DEV Groups groups_of(int pos, int window, int sinks) {
  Groups g;
  g.from = window > 0 ? max(0, pos - window + 1) : 0;
  g.ns = min(sinks, g.from);
  g.gs = (g.ns + 15) >> 4;
  g.g0 = max(g.from >> 4, g.gs);
  g.count = pos < 0 ? 0 : g.gs + (pos >> 4) + 1 - g.g0;
  return g;
}

// Workgroups that a CU holds: one where the registers of a tile's keys and values and of
// the sums leave no room for two (with two, 512 elements of 16 bits and 8 heads spill 79
// registers a lane).  For eight heads of fewer than 64 elements two spill 11 registers in F16 and
// 17 in BF16, of 65 to 127 in F16 4: 64 rows of 200 to 16384 tokens, 32/4 heads of 56, take 91 and
// 92 us, of 64 88, of 120 128 and of 128 126.
constexpr int split_per_cu(int type, int hs, int gt) {
  const int row_bytes = hs * (type == T_F32 ? 4 : 2);
  return (row_bytes > 512 ? row_bytes / 8 : 64) + 8 * gt > 150 ? 1 : 2;
}

// Where the stretches and their slots lie.
struct SplitPlan {
  int64_t *first;  // [n + 1] units before each row; then the units of a stretch, and what heads are padded to
  int32_t *count;  // [n] groups of each row
  float *part;     // [2 * wgs][GT][hs]
  float *ml;       // [2 * wgs][GT][2]
  int32_t wgs;
  int32_t parts;   // head parts of a kv head
  int32_t gt;
};

// Units of a stretch: an equal share, but at least a group for each of a workgroup's four
// waves, where heads have that many.
G4_DEV int64_t stretch_of(int64_t total, int wgs, int heads) {
  const int64_t per = quotient(total + wgs - 1, wgs), mean = quotient(total + heads - 1, heads);
  const int64_t least = mean < 1 ? 1 : mean > 4 ? 4 : mean;
  return per < least ? least : per;
}

// Groups that a segment's start and end are worth: 15000 clocks of a CU's 10 bytes.
constexpr int segment_worth(int type, int hs) {
  const int groups = 150000 / (32 * hs * (type == T_F32 ? 4 : 2));
  return groups < 4 ? 4 : groups;
}

// A score whose products or sums the matrix cores could not form (an infinite key times
// a part that is zero, a sum beyond fp32): the dot product as it is written.
template <int TYPE>
G4_DEV float plain_score(const float *q, const char *k, int hs, float f) {
  float d = 0.f;
#pragma unroll 1
  for (int i = 0; i < hs; i += 8) {
    Raw8<TYPE> r;
    float x[8];
    r.load(k, i);
    r.floats(x);
    for (int j = 0; j < 8; ++j) d = __builtin_fmaf(q[i + j], x[j], d);
  }
  return d * f;
}

template <int TYPE, int HS, int GT, bool FULL>
__global__ __launch_bounds__(256, split_per_cu(TYPE, HS, GT)) void k_paged_split(PagedArgs a, SplitPlan pl) {
  using M = Mfma<TYPE>;
  constexpr int ES = TYPE == T_F32 ? 4 : 2, RW = TYPE == T_F32 ? 2 : 1;
  constexpr int NG0 = 64 * 128 / (HS * 16 * ES), NG = NG0 < 1 ? 1 : NG0;  // groups of a tile: 8 KB of keys
  constexpr int STEPS = HS / M::STEP, SETS = (GT + 3) / 4;
  constexpr int LS = HS / 8, RS = 64 / LS, VS = 16 / RS;  // values: lanes of a row, rows and steps of a group
  constexpr int QOP = SETS * STEPS * 64 * 16, SO = 4 * GT * HS * 4;
  __shared__ __align__(16) char shared[QOP > SO ? QOP : SO];
  __shared__ float pw[4][NG * 16][GT];
  __shared__ float sm[4][GT], sl[4][GT], stat[GT][2], back[SETS * 4];
  __shared__ int64_t wsum[4];
  extern __shared__ __align__(16) char dyn[];  // first [n + 1], count [n], length [n], sequence [n]
  int64_t per;
  int pad = 1;
  bool aligned = false;
  u32x4(*qop)[64] = (u32x4(*)[64])shared;
  float(*so)[GT][HS] = (float(*)[GT][HS])shared;
  int64_t *first = (int64_t *)dyn;
  int32_t *count = (int32_t *)(first + a.n + 1), *length = count + a.n, *sequence = length + a.n;

  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), hs = FULL ? HS : kv.hs;
  const int status = *kv.status;  // looked at once the lengths are here too
  const int group = a.n_heads / kv.n_kv, units = kv.n_kv * pl.parts;

  // ---- the units before each row: four rows a thread
  {
    int64_t mine = 0;
    int c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 4 * tid + j;
      c[j] = 0;
      if (e < a.n) {
        const int seq = a.seqs[e];
        int len = 0;
        if ((unsigned)seq < (unsigned)kv.max_seqs) len = min(max(kv.lengths[seq], 0), kv.max_pages << kv.shift);
        c[j] = groups_of(len - 1, a.window, a.sinks).count;
        count[e] = c[j];
        length[e] = len;
        sequence[e] = (unsigned)seq < (unsigned)kv.max_seqs ? seq : 0;
        mine += (int64_t)c[j] * units;
      }
    }
    if (a.n * units <= (int)gridDim.x) {
      // Stretches that end where heads do, if that makes them no longer than a second segment
      // would: the shortest of three lengths with which every head's pieces have a workgroup each.
      // (Sums in 32 bits: of counts cut to 2^21 groups, for the lengths to try only.)
      // 24 rows in a window of 1024, 8/1 heads of 512, BF16: 27.2 us, 34.4 with equal stretches;
      // 30 of up to 3000 in a window of 512, 8/2 of 128, F16: 17.4 and 21.5; one row whose heads
      // fill equal stretches anyway takes as long.
      __syncthreads();
      auto wave_total = [](int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); };
      int all = 0;
      for (int r = lane; r < a.n; r += 64) all += min(count[r], 1 << 21);
      const int least = (int)stretch_of((int64_t)wave_total(all) * units, gridDim.x, a.n * units);
      for (int i = 0; i < 3 && !aligned; ++i) {
        const uint32_t p = least + i * (segment_worth(TYPE, HS) / 2);
        int pieces = 0;
        for (int r = lane; r < a.n; r += 64) pieces += min((count[r] + p - 1) / p, 1u << 20);
        aligned = wave_total(pieces) <= (int)gridDim.x / units;
        if (aligned) pad = p;
      }
    }
    // first: sums of 64 bits, or of the heads' pieces, of which there are few
    int64_t x, step[4];
    if (aligned) {
      int few = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) few += c[j] = (int)((uint32_t)(c[j] + pad - 1) / (uint32_t)pad);
      const int s = wave_scan(few);
      if (lane == 63) wsum[wid] = s;
      x = s - few;
#pragma unroll
      for (int j = 0; j < 4; ++j) step[j] = c[j];
    } else {
      x = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
      }
      if (lane == 63) wsum[wid] = x;
      x -= mine;
#pragma unroll
      for (int j = 0; j < 4; ++j) step[j] = (int64_t)c[j] * units;
    }
    __syncthreads();
    for (int w = 0; w < wid; ++w) x += wsum[w];
    const int64_t each = aligned ? (int64_t)pad * units : 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 4 * tid + j;
      if (e < a.n) first[e] = x * each;
      x += step[j];
      if (e + 1 == a.n) first[a.n] = x * each;
    }
    __syncthreads();
  }
  if (status != KV_OK) return;
  if (blockIdx.x == 0) {
    for (int e = tid; e <= a.n; e += 256) {
      pl.first[e] = first[e];
      if (e < a.n) pl.count[e] = count[e];
    }
  }
  for (int e = blockIdx.x; e < a.n; e += gridDim.x)  // rows that see nothing
    if (count[e] == 0)
      for (int i = tid; i < a.n_heads * hs; i += 256) a.out[(int64_t)e * a.n_heads * hs + i] = 0.f;

  per = aligned ? pad : stretch_of(first[a.n], gridDim.x, a.n * units);
  if (blockIdx.x == 0 && tid == 0) pl.first[a.n + 1] = per, pl.first[a.n + 2] = pad;
  const int64_t begin = blockIdx.x * per, end = min(first[a.n], begin + per);
  const float f = a.scale * LOG2E;
  const int key = lane & 15, kq = lane >> 4;  // of a score; of a key's dims
  const int ql = lane % LS, rl = lane / LS;   // of a value row

  int e = 0;
  for (int64_t u = begin; u < end;) {
    {
      int lo = e, hi = a.n - 1;  // the row of unit u: the last whose first unit is <= u
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= u) lo = mid;
        else hi = mid - 1;
      }
      e = lo;
    }
    const int cnt = count[e], room = padded(cnt, pad);
    const int64_t rel = u - first[e];
    const int hu = __builtin_amdgcn_readfirstlane((int)quotient(rel, room));
    const int gi0 = __builtin_amdgcn_readfirstlane((int)(rel - (int64_t)hu * room));
    const int gi1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)cnt, gi0 + (end - u)));
    const int kvh = hu / pl.parts, h0 = (hu - kvh * pl.parts) * GT, heads = min(GT, group - h0);
    const int seq = __builtin_amdgcn_readfirstlane(sequence[e]);
    const int pos = __builtin_amdgcn_readfirstlane(length[e]) - 1;
    const Groups g = groups_of(pos, a.window, a.sinks);
    const float *q0 = a.q + ((int64_t)e * a.n_heads + kvh * group + h0) * hs;

    // ---- this wave's groups
    const int share = (gi1 - gi0 + 3) >> 2;
    const int wa = min(gi1, gi0 + wid * share), wb = min(gi1, wa + share);
    const int32_t *table = kv.table + (int64_t)seq * kv.max_pages;
    const int64_t layer_rows = (int64_t)a.layer * kv.n_pages * kv.n_kv << kv.shift;
    auto token_group = [&](int i) { return i < g.gs ? i : i - g.gs + g.g0; };
    auto load_pages = [&](int i0) {  // lane i: the page of group i0 + i, -1 behind the last
      const int i = i0 + lane;
      return i < wb ? table[token_group(i) << 4 >> kv.shift] : -1;
    };
    auto page_of = [&](int pids, int i) {  // -1 where there is none
      const int page = __builtin_amdgcn_readlane(pids, i);
      return page_ok(page, kv) ? page : -1;
    };
    const int pids0 = load_pages(wa);

    // ---- the queries: wave w takes heads w and w + 4, lane c dims 8c .. 8c + 7
    float x[SETS][8];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const bool in = 4 * s + wid < heads && 8 * lane < hs;
      const float4 *at = (const float4 *)(q0 + (in ? (int64_t)(4 * s + wid) * hs + 8 * lane : 0));
      const float4 y = at[0], z = at[1];
      x[s][0] = y.x, x[s][1] = y.y, x[s][2] = y.z, x[s][3] = y.w, x[s][4] = z.x, x[s][5] = z.y, x[s][6] = z.z, x[s][7] = z.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] = in ? x[s][i] : 0.f;
    }

    float acc[GT][8], m[SETS], l[SETS];
#pragma unroll
    for (int h = 0; h < GT; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[h][i] = 0.f;
#pragma unroll
    for (int s = 0; s < SETS; ++s) m[s] = -__builtin_inff(), l[s] = 0.f;

    u32x4 kr[NG][STEPS], vr[NG][VS][RW];
    // the bytes of a group's first row of this head (page 0 stands in for a missing one: it is read, not used)
    auto row_at = [&](int page, int tg) {
      return (layer_rows + (((int64_t)max(page, 0) * kv.n_kv + kvh) << kv.shift) + ((tg << 4) & (kv.page - 1))) *
             (int64_t)(hs * ES);
    };
    // Lanes whose elements lie behind the head read its last ones again: the query is zero
    // there, and what they make of the values is not used.
    // Buffer loads: a group's rows of the head from a scalar base, 32 bits of offset a lane,
    // bounded by the hardware.
    const int kd = kq * (M::STEP / 4), k_last = hs - M::STEP / 4;
    const uint32_t k_off = (uint32_t)(key * hs + (FULL ? kd : 0)) * ES;
    const uint32_t v_off = (uint32_t)(rl * hs + min(8 * ql, hs - 8)) * ES;
    auto load_k = [&](int n, int64_t row) {
      const auto at = __builtin_amdgcn_make_buffer_rsrc(kv.k + uniform(row), 0, 16 * hs * ES, 0x00027000);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint32_t off = FULL ? k_off + s * M::STEP * ES : k_off + min(s * M::STEP + kd, k_last) * ES;
        kr[n][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(at, off, 0, 0));
      }
    };
    auto load_v = [&](int n, int64_t row) {
      const auto at = __builtin_amdgcn_make_buffer_rsrc(kv.v + uniform(row), 0, 16 * hs * ES, 0x00027000);
#pragma unroll
      for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int r = 0; r < RW; ++r)
          vr[n][s][r] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(at, v_off + 16 * r, s * RS * hs * ES, 0));
    };

    int pids = pids0, pids_next = load_pages(wa + 64);
    int page[NG], nextp[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      page[n] = page_of(pids, n);
      const int64_t at = row_at(page[n], token_group(wa + n));
      if (wa < wb) load_k(n, at);
      if (wa < wb) load_v(n, at);
    }
    // ---- the queries as A operands, while the first tile is on its way
    __syncthreads();  // the last segment's sums have been read
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      const int h = 4 * s + wid;
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[s][i] *= f;
        top = fmaxf(top, __builtin_fabsf(x[s][i]));
      }
      top = lanes16_max(top, lane);
      top = fmaxf(top, __uint_as_float(partner_u32<16>(__float_as_uint(top), lane)));
      top = fmaxf(top, __uint_as_float(partner_u32<32>(__float_as_uint(top), lane)));
      float to, bk;
      split_scale<TYPE>(top, to, bk);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[s][i] *= to;
      if (lane == 0) back[h] = bk;
      if (8 * lane < HS) {
        const int row = 4 * wid;
        if constexpr (TYPE == T_F32) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int d = 8 * lane + 4 * half, at = s * STEPS + d / 16, l0 = (d % 16) / 4 * 16 + row;
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[s][4 * half + i]);
            qop[at][l0] = w;
#pragma unroll
            for (int r = 1; r < 4; ++r) qop[at][l0 + r] = u32x4{0, 0, 0, 0};
          }
        } else {
          const int at = s * STEPS + lane / 4, l0 = (lane & 3) * 16 + row;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            u32x4 w = {0, 0, 0, 0};
            if (r < 3)
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = take_part<TYPE>(x[s][2 * i], x[s][2 * i + 1]);
            qop[at][l0 + r] = w;
          }
        }
      }
    }
    __syncthreads();
    float bk[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) bk[s] = back[s * 4 + kq];

    for (int i0 = wa; i0 < wb; i0 += NG) {
      const int nx = i0 + NG - wa;  // the next tile
      if ((nx & 63) == 0) {
        pids = pids_next;
        pids_next = load_pages(wa + nx + 64);
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) nextp[n] = page_of(pids, (nx + n) & 63);

      // ---- scores
      f32x4 c[SETS][NG];
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int n = 0; n < NG; ++n) c[s][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < STEPS; ++t)
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          const u32x4 qa = qop[s * STEPS + t][lane];
#pragma unroll
          for (int n = 0; n < NG; ++n) c[s][n] = M::step(qa, kr[n][t], c[s][n]);
        }
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int n = 0; n < NG; ++n) asm volatile("" : "+v"(c[s][n]));
      __builtin_amdgcn_sched_barrier(0);  // the loads below take the registers of the keys above
      if (i0 + NG < wb)
#pragma unroll
        for (int n = 0; n < NG; ++n) load_k(n, row_at(nextp[n], token_group(i0 + NG + n)));

      __builtin_amdgcn_sched_barrier(0);

      float sc[SETS][NG];
      bool odd = false;
      bool full[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const int t0 = token_group(i0 + n) << 4;
        full[n] = page[n] >= 0 && t0 + 15 <= pos && (t0 >= g.from || t0 + 15 < g.ns);
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          const float v = ((c[s][n][2] + c[s][n][1]) + c[s][n][0]) * bk[s];
          const int t = t0 + key;
          const bool seen = full[n] || (page[n] >= 0 && t <= pos && (t >= g.from || t < g.ns));
          odd |= seen && !(__builtin_fabsf(v) < __builtin_inff());
          sc[s][n] = seen ? v : -__builtin_inff();
        }
      }
      if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int s = 0; s < SETS; ++s) {
            const int h = s * 4 + kq, t = (token_group(i0 + n) << 4) + key;
            const bool seen = full[n] || (page[n] >= 0 && t <= pos && (t >= g.from || t < g.ns));
            if (seen && h < heads && !(__builtin_fabsf(sc[s][n]) < __builtin_inff()))
              sc[s][n] = plain_score<TYPE>(q0 + (int64_t)h * hs,
                                           kv.k + row_at(page[n], token_group(i0 + n)) + (int64_t)key * hs * ES, hs, f);
          }
      }

      // ---- weights
      float al[SETS];
      bool moved = false;
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        float top = sc[s][0];
#pragma unroll
        for (int n = 1; n < NG; ++n) top = fmaxf(top, sc[s][n]);
        top = fmaxf(m[s], lanes16_max(top, lane));
        al[s] = shrink(m[s], top);
        moved |= m[s] != top;
        m[s] = top;
        l[s] *= al[s];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float w = shrink(sc[s][n], top);
          l[s] += w;
          if (s * 4 + kq < GT) pw[wid][n * 16 + key][s * 4 + kq] = w;
        }
      }
      if (__any(moved)) {
#pragma unroll
        for (int h = 0; h < GT; ++h) {
          const float x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(al[h >> 2]), 16 * (h & 3)));
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[h][i] *= x;
        }
      }

      // ---- values
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        if (!full[n]) {
          const int t0 = token_group(i0 + n) << 4;
#pragma unroll
          for (int s = 0; s < VS; ++s) {
            const int t = t0 + s * RS + rl;
            const bool seen = page[n] >= 0 && t <= pos && (t >= g.from || t < g.ns);
#pragma unroll
            for (int r = 0; r < RW; ++r)
#pragma unroll
              for (int i = 0; i < 4; ++i) vr[n][s][r][i] = seen ? vr[n][s][r][i] : 0u;
          }
        }
#pragma unroll
        for (int s = 0; s < VS; ++s) {
          Raw8<TYPE> raw;
          float v[8];
#pragma unroll
          for (int r = 0; r < RW; ++r) raw.w[r] = vr[n][s][r];
          raw.floats(v);
#pragma unroll
          for (int h = 0; h < GT; ++h) {
            const float w = pw[wid][n * 16 + s * RS + rl][h];
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[h][i] = __builtin_fmaf(w, v[i], acc[h][i]);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < GT; ++h) formed(acc[h]);
      __builtin_amdgcn_sched_barrier(0);
      if (i0 + NG < wb)
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          load_v(n, row_at(nextp[n], token_group(i0 + NG + n)));
          page[n] = nextp[n];
        }
    }

    // ---- the four waves joined
#pragma unroll
    for (int s = 0; s < SETS; ++s) l[s] = lanes_sum<16>(l[s], lane);
    if (key == 0)
#pragma unroll
      for (int s = 0; s < SETS; ++s)
        if (s * 4 + kq < GT) sm[wid][s * 4 + kq] = m[s], sl[wid][s * 4 + kq] = l[s];
    __syncthreads();  // and everyone is done with the queries, whose memory the sums take
    {
      const int h = lane % GT;  // lane h: head h
      const float m0 = sm[0][h], m1 = sm[1][h], m2 = sm[2][h], m3 = sm[3][h];
      const float top = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
      const float mine = shrink(wid < 2 ? (wid == 0 ? m0 : m1) : (wid == 2 ? m2 : m3), top);
      if (wid == 0 && lane < GT) {
        stat[h][0] = top;
        stat[h][1] = ((sl[0][h] * shrink(m0, top) + sl[1][h] * shrink(m1, top)) + sl[2][h] * shrink(m2, top)) +
                     sl[3][h] * shrink(m3, top);
      }
#pragma unroll
      for (int g = 0; g < GT; ++g) {
        const float c = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), g));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v = acc[g][i] * c;
          if constexpr (LS <= 8) v = add_partner<8>(v, lane);
          if constexpr (LS <= 16) v = add_partner<16>(v, lane);
          if constexpr (LS <= 32) v = add_partner<32>(v, lane);
          acc[g][i] = v;
        }
        formed(acc[g]);
      }
    }
    if (rl == 0)
#pragma unroll
      for (int h = 0; h < GT; ++h)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *(float4 *)&so[wid][h][8 * ql + i] = make_float4(acc[h][i], acc[h][i + 1], acc[h][i + 2], acc[h][i + 3]);
    __syncthreads();
    const bool whole = gi0 == 0 && gi1 == cnt;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (u != begin);
    float *const out = whole ? a.out + ((int64_t)e * a.n_heads + kvh * group + h0) * hs : pl.part + slot * GT * hs;
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      if (h >= heads) break;
      const float sum = stat[h][1];
      const float by = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      for (int d = 4 * tid; d < hs; d += 1024) {
        const float4 o0 = *(const float4 *)&so[0][h][d], o1 = *(const float4 *)&so[1][h][d];
        const float4 o2 = *(const float4 *)&so[2][h][d], o3 = *(const float4 *)&so[3][h][d];
        float4 o = make_float4(((o0.x + o1.x) + o2.x) + o3.x, ((o0.y + o1.y) + o2.y) + o3.y, ((o0.z + o1.z) + o2.z) + o3.z,
                               ((o0.w + o1.w) + o2.w) + o3.w);
        if (whole && sum == 0.f) o = make_float4(0, 0, 0, 0);
        *(float4 *)(out + (int64_t)h * hs + d) = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
      }
    }
    if (!whole && tid < heads) {
      pl.ml[(slot * GT + tid) * 2] = stat[tid][0];
      pl.ml[(slot * GT + tid) * 2 + 1] = stat[tid][1];
    }
    u += (gi1 == cnt ? room : gi1) - gi0;
  }
}

// The slots of a head: workgroup (row * n_heads + head, 4 ls elements).  64 slots at a time,
// each wave forms all their weights, a lane each; the slots' values go around the waves,
// 64 / ls slots to a load, and the waves' sums are added in wave order.  Bound by latency
// (status, plan, slots, one after the other): 5 us for one row's 64 slots a head, 9 us for
// 2048 heads of one to three.
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a, SplitPlan pl, int ls) {
  __shared__ float4 ws[4][64];
  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int e = blockIdx.x / a.n_heads, h = blockIdx.x - e * a.n_heads;
  const int status = *kv.status, cnt = pl.count[e];
  const int64_t before = pl.first[e], per = pl.first[a.n + 1];
  const int pad = (int)pl.first[a.n + 2];
  if (status != KV_OK || cnt == 0) return;
  const int group = a.n_heads / kv.n_kv, kvh = h / group, hg = h - kvh * group;
  const int64_t ua = before + (int64_t)(kvh * pl.parts + hg / pl.gt) * padded(cnt, pad);
  const int w0 = (int)quotient(ua, per), w1 = (int)quotient(ua + cnt - 1, per);
  if (w0 == w1) return;
  const int n = w1 - w0 + 1, g = hg % pl.gt;
  const int64_t s0 = 2 * (int64_t)w0 + (ua != w0 * per);  // the first slot; the others are first slots of their stretch
  auto slot = [&](int i) { return (i == 0 ? s0 : 2 * (int64_t)(w0 + i)) * pl.gt + g; };
  const int rows = 64 / ls, sub = lane / ls, d = 4 * (blockIdx.y * ls + lane % ls);
  const float *part = pl.part + (d < kv.hs ? d : 0);
  float4 o = make_float4(0, 0, 0, 0);
  float sum = 0.f, top = -__builtin_inff();
  constexpr int U = 8;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const float2 ml = *(const float2 *)(pl.ml + slot(min(i0 + lane, n - 1)) * 2);
    float c = 1.f, x = 0.f;
    for (int k0 = 0; k0 < 64; k0 += 4 * U * rows) {
      if (i0 + k0 >= n) break;
      float4 v[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        v[k] = make_float4(0, 0, 0, 0);
        const int i = i0 + k0 + (4 * k + wid) * rows;
        if (i < n && i < i0 + 64) v[k] = *(const float4 *)(part + slot(min(i + sub, n - 1)) * kv.hs);
      }
      if (k0 == 0) {
        const float m = i0 + lane < n ? ml.x : -__builtin_inff();
        float t = lanes16_max(m, lane);
        t = fmaxf(t, __uint_as_float(partner_u32<16>(__float_as_uint(t), lane)));
        t = fmaxf(t, __uint_as_float(partner_u32<32>(__float_as_uint(t), lane)));
        t = fmaxf(t, top);
        c = shrink(top, t), x = shrink(m, t);
        top = t;
        sum = __builtin_fmaf(sum, c, x * ml.y);
        o = make_float4(o.x * c, o.y * c, o.z * c, o.w * c);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int at = k0 + (4 * k + wid) * rows;
        if (at >= 64 || i0 + at >= n) break;
        const float w = __shfl(x, at + sub);  // 0 behind the last slot
        o.x = __builtin_fmaf(v[k].x, w, o.x), o.y = __builtin_fmaf(v[k].y, w, o.y);
        o.z = __builtin_fmaf(v[k].z, w, o.z), o.w = __builtin_fmaf(v[k].w, w, o.w);
      }
    }
  }
  for (int s = ls; s < 64; s <<= 1)
    o.x += __shfl_xor(o.x, s), o.y += __shfl_xor(o.y, s), o.z += __shfl_xor(o.z, s), o.w += __shfl_xor(o.w, s);
  ws[wid][lane] = o;
  sum = lanes_sum<64>(sum, lane);
  __syncthreads();
  if (wid == 0 && sub == 0 && d < kv.hs) {
    for (int w = 1; w < 4; ++w) {
      const float4 v = ws[w][lane];
      o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    }
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    o = make_float4(o.x * by, o.y * by, o.z * by, o.w * by);
    *(float4 *)(a.out + ((int64_t)e * a.n_heads + h) * kv.hs + d) = sum == 0.f ? make_float4(0, 0, 0, 0) : o;
  }
}

static int split_heads(const PagedArgs &a) {  // query heads that share a pass over their kv head
  const int group = a.n_heads / a.kv.n_kv;
  return group <= 2 ? 2 : group <= 4 ? 4 : 8;
}

static size_t split_layout(const PagedArgs &a, const DevInfo &dev, char *base, SplitPlan *p) {
  p->gt = split_heads(a);
  p->parts = (a.n_heads / a.kv.n_kv + p->gt - 1) / p->gt;
  const int hs = a.kv.hs <= 64 ? 64 : a.kv.hs <= 128 ? 128 : a.kv.hs <= 256 ? 256 : 512;
  p->wgs = split_per_cu(a.kv.type, hs, p->gt) * dev.cu_count;
  size_t off = 0;
  auto add = [&](size_t bytes) {
    char *at = base + off;
    off += (bytes + 255) & ~size_t(255);
    return at;
  };
  p->first = (int64_t *)add(8 * (size_t)(a.n + 3));
  p->count = (int32_t *)add(4 * (size_t)a.n);
  p->part = (float *)add(sizeof(float) * 2 * (size_t)p->wgs * p->gt * a.kv.hs);
  p->ml = (float *)add(sizeof(float) * 4 * (size_t)p->wgs * p->gt);
  return off;
}

template <int TYPE, int HS, int GT>
static void launch_split(const PagedArgs &a, const SplitPlan &p, hipStream_t s) {
  const size_t lds = 8 * (size_t)(a.n + 1) + 12 * (size_t)a.n;
  if (a.kv.hs == HS) hipLaunchKernelGGL((k_paged_split<TYPE, HS, GT, true>), dim3(p.wgs), dim3(256), lds, s, a, p);
  else hipLaunchKernelGGL((k_paged_split<TYPE, HS, GT, false>), dim3(p.wgs), dim3(256), lds, s, a, p);
}

template <int TYPE, int HS>
static void launch_split(const PagedArgs &a, const SplitPlan &p, hipStream_t s) {
  if (p.gt == 2) launch_split<TYPE, HS, 2>(a, p, s);
  else if (p.gt == 4) launch_split<TYPE, HS, 4>(a, p, s);
  else launch_split<TYPE, HS, 8>(a, p, s);
}

template <int TYPE>
static void launch_split(const PagedArgs &a, const SplitPlan &p, hipStream_t s) {
  if (a.kv.hs <= 64) launch_split<TYPE, 64>(a, p, s);
  else if (a.kv.hs <= 128) launch_split<TYPE, 128>(a, p, s);
  else if (a.kv.hs <= 256) launch_split<TYPE, 256>(a, p, s);
  else launch_split<TYPE, 512>(a, p, s);
}

size_t paged_scratch_bytes(const PagedArgs &a, const DevInfo &dev) {
  SplitPlan p;
  return split_layout(a, dev, nullptr, &p);
}

hipError_t launch_paged(const PagedArgs &a, const DevInfo &dev, char *scratch, hipStream_t s) {
  SplitPlan p;
  split_layout(a, dev, scratch, &p);
  if (a.kv.type == T_F32) launch_split<T_F32>(a, p, s);
  else if (a.kv.type == T_F16) launch_split<T_F16>(a, p, s);
  else launch_split<T_BF16>(a, p, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  int ls = 64;
  while (ls > 1 && ls * 2 >= a.kv.hs) ls >>= 1;
  // Heads of many slots are read by more workgroups, or a few CUs would have all of it to
  // read: 16 heads of 64 slots take 4.8 us, with 256 elements a workgroup 6.8; 2048 heads of
  // one to three slots 9.0 us that way, and 10.6 with 64 elements.
  if (p.wgs > 16 * a.n * a.kv.n_kv * p.parts) ls = ls < 16 ? ls : 16;
  hipLaunchKernelGGL(k_paged_join, dim3(a.n * a.n_heads, (a.kv.hs + 4 * ls - 1) / (4 * ls)), dim3(256), 0, s, a, p, ls);
  return hipGetLastError();
}

}  // namespace g4
