// g4_paged.hip -- attention over a paged key-value cache.
//
// Row r of a call is token `pos` of a sequence; query head h reads kv head h / group.
// It sees the tokens t <= pos of its sequence with t > pos - window (window > 0) or
// t < sinks, and of those the ones whose page is there:
//   out = sum_t p_t V[t] / sum_t p_t,  p_t = exp(scale q . K[t] - max),
// and zeros where it sees nothing.  One pass over K and V with a running maximum and
// sum; products, statistics and sums are fp32 whatever the cache holds.
#include "g4_device.hpp"
#include "g4_internal.hpp"

namespace g4 {

constexpr float LOG2E = 1.4426950408889634f;

// What a row sees: visible index j < ns is token j, later ones are token j + skip.
struct Seen {
  int count;
  int ns;
  int skip;
};

G4_DEV Seen seen_by(int pos, int window, int sinks) {
  Seen s;
  const int from = window > 0 ? max(0, pos - window + 1) : 0;
  s.ns = min(sinks, from);
  s.skip = from - s.ns;
  s.count = pos + 1 - s.skip;
  return s;
}

G4_DEV bool page_ok(int page, const KvArgs &kv) { return (unsigned)page < (unsigned)kv.n_pages; }

// Entry of row r in the list and its position; false where the row belongs to no
// sequence (it is left as it is).  A position that its sequence does not have is -1.
G4_DEV bool row_place(const PagedArgs &a, int r, int &seq, int &pos) {
  int e = r, rows = 1, at = 0;
  if (a.row_begin) {
    if (r < a.row_begin[0] || r >= a.row_begin[a.n]) return false;
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.row_begin[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    e = lo;
    rows = a.row_begin[e + 1] - a.row_begin[e];
    at = r - a.row_begin[e];
  }
  seq = a.seqs[e];
  int len = 0;
  if ((unsigned)seq < (unsigned)a.kv.max_seqs) len = min(max(a.kv.lengths[seq], 0), a.kv.max_pages << a.kv.shift);
  else seq = 0;
  pos = len - rows + at;
  if (pos < 0 || pos >= len) pos = -1;
  return true;
}

// Eight elements of a cached row as they are loaded, and as fp32.
template <int TYPE>
struct Raw8 {
  u32x4 w[TYPE == T_F32 ? 2 : 1];
  G4_DEV void load(const char *base, int64_t elem) {
    const u32x4 *p = (const u32x4 *)(base + elem * (TYPE == T_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (TYPE == T_F32 ? 2 : 1); ++i) w[i] = p[i];
  }
  G4_DEV void zero() {
#pragma unroll
    for (int i = 0; i < (TYPE == T_F32 ? 2 : 1); ++i) w[i] = u32x4{0, 0, 0, 0};
  }
  G4_DEV void floats(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (TYPE == T_F32) f[i] = __uint_as_float(w[i >> 2][i & 3]);
      else if constexpr (TYPE == T_F16) f[i] = i & 1 ? f16hi(w[0][i >> 1]) : f16lo(w[0][i >> 1]);
      else f[i] = __uint_as_float(i & 1 ? w[0][i >> 1] & 0xFFFF0000u : w[0][i >> 1] << 16);
    }
  }
};

template <int N>
G4_DEV float lanes_sum(float s, int lane) {  // over each aligned group of N lanes, in every lane of it
  if constexpr (N > 1) s += __uint_as_float(partner_u32<1>(__float_as_uint(s), lane));
  if constexpr (N > 2) s += __uint_as_float(partner_u32<2>(__float_as_uint(s), lane));
  if constexpr (N > 4) s += __uint_as_float(partner_u32<4>(__float_as_uint(s), lane));
  if constexpr (N > 8) s += __uint_as_float(partner_u32<8>(__float_as_uint(s), lane));
  if constexpr (N > 16) s += __uint_as_float(partner_u32<16>(__float_as_uint(s), lane));
  if constexpr (N > 32) s += __uint_as_float(partner_u32<32>(__float_as_uint(s), lane));
  return s;
}

// 2^(a - b), b >= a, where both may be -infinity (nothing seen yet, or a hidden token)
G4_DEV float shrink(float a, float b) { return a == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(a - b); }

// One workgroup per (row, kv head, stretch of up to GT of its query heads).  LS = HS / 8
// lanes share a cached row, eight elements a lane, so a wave takes RS = 64 / LS rows at
// a time, U of them in flight.  Each group of LS lanes keeps a running maximum, sum and
// accumulator of the rows it has met; the groups of the four waves are joined at the
// end.  Head sizes between the powers of two leave the lanes behind the head idle.
template <int TYPE, int HS, int GT>
__global__ __launch_bounds__(256) void k_paged_row(PagedArgs a) {
  constexpr int LS = HS / 8, RS = 64 / LS, U = 4;
  __shared__ float sm[4 * RS][GT], sl[4 * RS][GT];
  __shared__ float so[4][GT][HS];
  const KvArgs &kv = a.kv;
  if (*kv.status != KV_OK) return;
  const int group = a.n_heads / kv.n_kv, parts = (group + GT - 1) / GT;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, ql = lane % LS, rl = lane / LS;
  const int kvh = blockIdx.y / parts, g0 = (blockIdx.y % parts) * GT;
  int seq, pos;
  if (!row_place(a, blockIdx.x, seq, pos)) return;
  const Seen see = seen_by(pos, a.window, a.sinks);
  const bool live = 8 * ql < kv.hs;
  const int32_t *table = kv.table + (int64_t)seq * kv.max_pages;
  const int64_t head_rows = ((int64_t)a.layer * kv.n_pages * kv.n_kv + kvh) << kv.shift;

  float q[GT][8], acc[GT][8], m[GT], l[GT];
  const float f = a.scale * LOG2E;
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    const int h = kvh * group + min(g0 + g, group - 1);
    const float4 *qp = (const float4 *)(a.q + ((int64_t)blockIdx.x * a.n_heads + h) * kv.hs) + 2 * ql;
    const float4 x = live ? qp[0] : make_float4(0, 0, 0, 0), y = live ? qp[1] : make_float4(0, 0, 0, 0);
    q[g][0] = x.x, q[g][1] = x.y, q[g][2] = x.z, q[g][3] = x.w, q[g][4] = y.x, q[g][5] = y.y, q[g][6] = y.z, q[g][7] = y.w;
    m[g] = -__builtin_inff(), l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[g][i] = 0.f;
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
        const int64_t at = (head_rows + (((int64_t)page * kv.n_kv) << kv.shift) + (t & (kv.page - 1))) * kv.hs + 8 * ql;
        kr[u].load(kv.k, at);
        vr[u].load(kv.v, at);
      }
    }
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float s[U], top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float k[8], d = 0.f;
        kr[u].floats(k);
#pragma unroll
        for (int i = 0; i < 8; ++i) d = __builtin_fmaf(q[g][i], k[i], d);
        d = lanes_sum<LS>(d, lane) * f;  // by all lanes of the wave
        s[u] = ok[u] ? d : -__builtin_inff();
        top = fmaxf(top, s[u]);
      }
      const float c = shrink(m[g], top);
      m[g] = top;
      l[g] *= c;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[g][i] *= c;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float e = shrink(s[u], top);
        float v[8];
        vr[u].floats(v);
        l[g] += e;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[g][i] = __builtin_fmaf(e, v[i], acc[g][i]);
      }
    }
  }

  // join: first the groups of a wave, then the waves
  if (ql == 0)
#pragma unroll
    for (int g = 0; g < GT; ++g) sm[wid * RS + rl][g] = m[g], sl[wid * RS + rl][g] = l[g];
  __syncthreads();
#pragma unroll
  for (int g = 0; g < GT; ++g) {
    float top = -__builtin_inff();
    for (int i = 0; i < 4 * RS; ++i) top = fmaxf(top, sm[i][g]);
    const float c = shrink(m[g], top);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = acc[g][i] * c;
#pragma unroll
      for (int d = LS; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
      if (rl == 0) so[wid][g][8 * ql + i] = v;
    }
  }
  __syncthreads();
  for (int i = tid; i < GT * HS; i += 256) {
    const int g = i / HS, d = i % HS;
    if (d >= kv.hs || g0 + g >= group) continue;
    float top = -__builtin_inff(), sum = 0.f;
    for (int j = 0; j < 4 * RS; ++j) top = fmaxf(top, sm[j][g]);
    for (int j = 0; j < 4 * RS; ++j) sum = __builtin_fmaf(sl[j][g], shrink(sm[j][g], top), sum);
    const float o = ((so[0][g][d] + so[1][g][d]) + so[2][g][d]) + so[3][g][d];
    a.out[((int64_t)blockIdx.x * a.n_heads + kvh * group + g0 + g) * kv.hs + d] = sum == 0.f ? 0.f : o / sum;
  }
}

template <int TYPE, int HS>
static void launch_row(const PagedArgs &a, hipStream_t s) {
  const int group = a.n_heads / a.kv.n_kv;
  if (group == 1)
    hipLaunchKernelGGL((k_paged_row<TYPE, HS, 1>), dim3(a.n_rows, a.kv.n_kv), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_paged_row<TYPE, HS, 2>), dim3(a.n_rows, a.kv.n_kv * ((group + 1) / 2)), dim3(256), 0, s, a);
}

template <int TYPE>
static void launch_size(const PagedArgs &a, hipStream_t s) {
  if (a.kv.hs <= 64) launch_row<TYPE, 64>(a, s);
  else if (a.kv.hs <= 128) launch_row<TYPE, 128>(a, s);
  else if (a.kv.hs <= 256) launch_row<TYPE, 256>(a, s);
  else launch_row<TYPE, 512>(a, s);
}

hipError_t launch_paged(const PagedArgs &a, const DevInfo &, char *, hipStream_t s) {
  if (a.kv.type == T_F32) launch_size<T_F32>(a, s);
  else if (a.kv.type == T_F16) launch_size<T_F16>(a, s);
  else launch_size<T_BF16>(a, s);
  return hipGetLastError();
}

}  // namespace g4
