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
// they are device data, which each workgroup sums up itself.  Where a stretch holds all
// of a head's groups the result is final; otherwise (maximum, sum, weighted values) goes
// to the stretch's first or second slot and k_paged_join adds the slots of a head.
//
// A wave takes NG groups at a time.  Scores come from the matrix cores: A = the query
// heads, B = 16 keys as they lie in memory.  A head is four rows of A: for a 16-bit
// cache the query's three 16-bit parts, which add up to it exactly, for F32 the query
// itself; the products are then exact (F32: rounded once), and a lane's sum over its
// four rows of C is the score of (head lane / 16, key lane % 16).  The queries carry
// scale * log2(e) (split_scale keeps their parts in range).  Values are weighted by the vector unit in fp32, eight
// elements of a row per lane, with the weights handed over through the wave's own LDS.
// While a tile is worked on, the next one's keys and values are on their way.

constexpr int SPLIT_MIN = 8;  // least groups of a stretch

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
// registers a lane).
constexpr int split_per_cu(int type, int hs, int gt) {
  const int row_bytes = hs * (type == T_F32 ? 4 : 2);
  return (row_bytes > 512 ? row_bytes / 8 : 64) + 8 * gt > 150 ? 1 : 2;
}

// Where the stretches and their slots lie.
struct SplitPlan {
  int64_t *first;  // [n + 1] units before each row
  int32_t *count;  // [n] groups of each row
  float *part;     // [2 * wgs][GT][hs]
  float *ml;       // [2 * wgs][GT][2]
  int32_t wgs;
  int32_t parts;   // head parts of a kv head
  int32_t gt;
};

G4_DEV int64_t stretch_of(int64_t total, int wgs) {
  const int64_t per = (total + wgs - 1) / wgs;
  return per < SPLIT_MIN ? SPLIT_MIN : per;
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

template <int TYPE, int HS, int GT>
__global__ __launch_bounds__(256, split_per_cu(TYPE, HS, GT)) void k_paged_split(PagedArgs a, SplitPlan pl) {
  using M = Mfma<TYPE>;
  constexpr int ES = TYPE == T_F32 ? 4 : 2, RW = TYPE == T_F32 ? 2 : 1;
  constexpr int NG0 = 64 * 128 / (HS * 16 * ES), NG = NG0 < 1 ? 1 : NG0;  // groups of a tile: 8 KB of keys
  constexpr int STEPS = HS / M::STEP, SETS = (GT + 3) / 4;
  constexpr int LS = HS / 8, RS = 64 / LS, VS = 16 / RS;  // values: lanes of a row, rows and steps of a group
  constexpr int QOP = SETS * STEPS * 64 * 16, SO = 4 * GT * HS * 4;
  __shared__ __align__(16) char shared[QOP > SO ? QOP : SO];
  __shared__ float pw[4][NG * 16][GT];
  __shared__ float sm[4][GT], sl[4][GT], back[SETS * 4];
  __shared__ int64_t wsum[4];
  extern __shared__ __align__(16) char dyn[];  // first [n + 1], count [n], length [n]
  u32x4(*qop)[64] = (u32x4(*)[64])shared;
  float(*so)[GT][HS] = (float(*)[GT][HS])shared;
  int64_t *first = (int64_t *)dyn;
  int32_t *count = (int32_t *)(first + a.n + 1), *length = count + a.n;

  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), hs = kv.hs;
  if (*kv.status != KV_OK) return;
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
        mine += (int64_t)c[j] * units;
      }
    }
    int64_t x = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    if (lane == 63) wsum[wid] = x;
    __syncthreads();
    x -= mine;
    for (int w = 0; w < wid; ++w) x += wsum[w];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 4 * tid + j;
      if (e < a.n) first[e] = x;
      x += (int64_t)c[j] * units;
      if (e + 1 == a.n) first[a.n] = x;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0) {
    for (int e = tid; e <= a.n; e += 256) {
      pl.first[e] = first[e];
      if (e < a.n) pl.count[e] = count[e];
    }
  }
  for (int e = blockIdx.x; e < a.n; e += gridDim.x)  // rows that see nothing
    if (count[e] == 0)
      for (int i = tid; i < a.n_heads * hs; i += 256) a.out[(int64_t)e * a.n_heads * hs + i] = 0.f;

  const int64_t per = stretch_of(first[a.n], gridDim.x);
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
    const int cnt = count[e];
    const int64_t rel = u - first[e];
    const int hu = __builtin_amdgcn_readfirstlane((int)(rel / cnt));
    const int gi0 = __builtin_amdgcn_readfirstlane((int)(rel - (int64_t)hu * cnt));
    const int gi1 = __builtin_amdgcn_readfirstlane((int)min((int64_t)cnt, gi0 + (end - u)));
    const int kvh = hu / pl.parts, h0 = (hu - kvh * pl.parts) * GT, heads = min(GT, group - h0);
    const int seq = __builtin_amdgcn_readfirstlane(a.seqs[e]);
    const int pos = __builtin_amdgcn_readfirstlane(length[e]) - 1;
    const Groups g = groups_of(pos, a.window, a.sinks);
    const float *q0 = a.q + ((int64_t)e * a.n_heads + kvh * group + h0) * hs;

    // ---- the queries as A operands: wave w takes heads w and w + 4, lane c dims 8c .. 8c + 7
    __syncthreads();
#pragma unroll
    for (int h = wid; h < SETS * 4; h += 4) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
      if (h < heads && 8 * lane < hs) {
        const float4 y = ((const float4 *)(q0 + (int64_t)h * hs))[2 * lane];
        const float4 z = ((const float4 *)(q0 + (int64_t)h * hs))[2 * lane + 1];
        x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w, x[4] = z.x, x[5] = z.y, x[6] = z.z, x[7] = z.w;
      }
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= f;
        top = fmaxf(top, __builtin_fabsf(x[i]));
      }
      top = lanes16_max(top, lane);
      top = fmaxf(top, __uint_as_float(partner_u32<16>(__float_as_uint(top), lane)));
      top = fmaxf(top, __uint_as_float(partner_u32<32>(__float_as_uint(top), lane)));
      float to, bk;
      split_scale<TYPE>(top, to, bk);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= to;
      if (lane == 0) back[h] = bk;
      if (8 * lane < HS) {
        const int row = 4 * (h & 3);
        if constexpr (TYPE == T_F32) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int d = 8 * lane + 4 * half, at = (h >> 2) * STEPS + d / 16, l0 = (d % 16) / 4 * 16 + row;
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[4 * half + i]);
            qop[at][l0] = w;
#pragma unroll
            for (int r = 1; r < 4; ++r) qop[at][l0 + r] = u32x4{0, 0, 0, 0};
          }
        } else {
          const int at = (h >> 2) * STEPS + lane / 4, l0 = (lane & 3) * 16 + row;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            u32x4 w = {0, 0, 0, 0};
            if (r < 3)
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = take_part<TYPE>(x[2 * i], x[2 * i + 1]);
            qop[at][l0 + r] = w;
          }
        }
      }
    }
    __syncthreads();
    float bk[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) bk[s] = back[s * 4 + kq];

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
    const int kd = kq * (M::STEP / 4), k_last = hs - M::STEP / 4;
    const uint32_t k_row = (uint32_t)(key * hs * ES), v_off = (uint32_t)(rl * hs + min(8 * ql, hs - 8)) * ES;
    auto load_k = [&](int n, int64_t row) {
      const char *at = kv.k + uniform(row);
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        kr[n][s] = *(const u32x4 *)(at + (uint32_t)(k_row + min(s * M::STEP + kd, k_last) * ES));
    };
    auto load_v = [&](int n, int64_t row) {
      const char *at = kv.v + uniform(row);
#pragma unroll
      for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int r = 0; r < RW; ++r) vr[n][s][r] = *(const u32x4 *)(at + (uint32_t)(v_off + s * RS * hs * ES) + 16 * r);
    };

    int pids = load_pages(wa), pids_next = load_pages(wa + 64);
    int page[NG], nextp[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      page[n] = page_of(pids, n);
      const int64_t at = row_at(page[n], token_group(wa + n));
      if (wa < wb) load_k(n, at);
      if (wa < wb) load_v(n, at);
    }
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
    for (int h = 0; h < GT; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int d = LS; d < 64; d <<= 1) acc[h][i] += __shfl_xor(acc[h][i], d, 64);
#pragma unroll
    for (int s = 0; s < SETS; ++s) l[s] = lanes_sum<16>(l[s], lane);
    __syncthreads();  // everyone is done with the queries, whose memory this is
    if (rl == 0)
#pragma unroll
      for (int h = 0; h < GT; ++h)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *(float4 *)&so[wid][h][8 * ql + i] = make_float4(acc[h][i], acc[h][i + 1], acc[h][i + 2], acc[h][i + 3]);
    if (key == 0)
#pragma unroll
      for (int s = 0; s < SETS; ++s)
        if (s * 4 + kq < GT) sm[wid][s * 4 + kq] = m[s], sl[wid][s * 4 + kq] = l[s];
    __syncthreads();
    const bool whole = gi0 == 0 && gi1 == cnt;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (u != begin);
    for (int i = tid; i < heads * hs; i += 256) {
      const int h = i / hs, d = i - h * hs;
      const float top = fmaxf(fmaxf(sm[0][h], sm[1][h]), fmaxf(sm[2][h], sm[3][h]));
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float x = shrink(sm[w][h], top);
        o = __builtin_fmaf(so[w][h][d], x, o);
        sum = __builtin_fmaf(sl[w][h], x, sum);
      }
      if (whole) {
        a.out[((int64_t)e * a.n_heads + kvh * group + h0 + h) * hs + d] = sum == 0.f ? 0.f : o / sum;
      } else {
        pl.part[(slot * GT + h) * hs + d] = o;
        if (d == 0) pl.ml[(slot * GT + h) * 2] = top, pl.ml[(slot * GT + h) * 2 + 1] = sum;
      }
    }
    u += gi1 - gi0;
  }
}

// The slots of a head: workgroup (row * n_heads + head, 64 elements), wave w takes slots
// w, w + 4, ... in order, and the four sums are added in wave order.
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a, SplitPlan pl) {
  __shared__ float ws[4][64], top4[4], sum4[4];
  const KvArgs &kv = a.kv;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int e = blockIdx.x / a.n_heads, h = blockIdx.x - e * a.n_heads;
  if (*kv.status != KV_OK) return;
  const int cnt = pl.count[e];
  if (cnt == 0) return;
  const int group = a.n_heads / kv.n_kv, kvh = h / group, hg = h - kvh * group;
  const int64_t per = stretch_of(pl.first[a.n], pl.wgs);
  const int64_t ua = pl.first[e] + (int64_t)(kvh * pl.parts + hg / pl.gt) * cnt;
  const int w0 = (int)(ua / per), w1 = (int)((ua + cnt - 1) / per);
  if (w0 == w1) return;
  const int n = w1 - w0 + 1, g = hg % pl.gt;
  const int64_t s0 = 2 * (int64_t)w0 + (ua != w0 * per);  // the first slot; the others are first slots of their stretch
  auto slot = [&](int i) { return (i == 0 ? s0 : 2 * (int64_t)(w0 + i)) * pl.gt + g; };
  float top = -__builtin_inff();
  for (int i = tid; i < n; i += 256) top = fmaxf(top, pl.ml[slot(i) * 2]);
  top = lanes16_max(top, lane);
  top = fmaxf(top, __uint_as_float(partner_u32<16>(__float_as_uint(top), lane)));
  top = fmaxf(top, __uint_as_float(partner_u32<32>(__float_as_uint(top), lane)));
  if (lane == 0) top4[wid] = top;
  __syncthreads();
  top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
  const int d = blockIdx.y * 64 + lane;
  const bool live = d < kv.hs;
  float o = 0.f, sum = 0.f;
#pragma unroll 8
  for (int i = wid; i < n; i += 4) {
    const int64_t s = slot(i);
    const float x = shrink(pl.ml[s * 2], top);
    sum = __builtin_fmaf(pl.ml[s * 2 + 1], x, sum);
    o = __builtin_fmaf(live ? pl.part[s * kv.hs + d] : 0.f, x, o);
  }
  ws[wid][lane] = o;
  if (lane == 0) sum4[wid] = sum;
  __syncthreads();
  if (wid == 0 && live) {
    const float all = ((sum4[0] + sum4[1]) + sum4[2]) + sum4[3];
    o = ((ws[0][lane] + ws[1][lane]) + ws[2][lane]) + ws[3][lane];
    a.out[((int64_t)e * a.n_heads + h) * kv.hs + d] = all == 0.f ? 0.f : o / all;
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
  p->first = (int64_t *)add(8 * (size_t)(a.n + 1));
  p->count = (int32_t *)add(4 * (size_t)a.n);
  p->part = (float *)add(sizeof(float) * 2 * (size_t)p->wgs * p->gt * a.kv.hs);
  p->ml = (float *)add(sizeof(float) * 4 * (size_t)p->wgs * p->gt);
  return off;
}

template <int TYPE, int HS>
static void launch_split(const PagedArgs &a, const SplitPlan &p, hipStream_t s) {
  const size_t lds = 8 * (size_t)(a.n + 1) + 8 * (size_t)a.n;
  if (p.gt == 2) hipLaunchKernelGGL((k_paged_split<TYPE, HS, 2>), dim3(p.wgs), dim3(256), lds, s, a, p);
  else if (p.gt == 4) hipLaunchKernelGGL((k_paged_split<TYPE, HS, 4>), dim3(p.wgs), dim3(256), lds, s, a, p);
  else hipLaunchKernelGGL((k_paged_split<TYPE, HS, 8>), dim3(p.wgs), dim3(256), lds, s, a, p);
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
  hipLaunchKernelGGL(k_paged_join, dim3(a.n * a.n_heads, (a.kv.hs + 63) / 64), dim3(256), 0, s, a, p);
  return hipGetLastError();
}

}  // namespace g4
