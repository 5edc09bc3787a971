// g4_kv.hip -- a paged key-value cache: rotary positions and the write of new rows,
// and the pages' bookkeeping (extend, fork, compact, release), all of it device data,
// so that a captured decode step advances by itself when it is replayed.
//
// K and V are [layer][page][kv head][token of the page][head size]: a page holds a kv
// head's tokens next to each other, which is what attention reads.  A sequence's
// token p is in page table[p / page].  refs counts the sequences that hold a page, 0:
// free.  The pages that sequences share are full ones; a partly filled page has one
// owner, so an append never writes into another sequence.
//
// The bookkeeping calls are all or nothing: one workgroup (k_kv_extend, k_kv_plan,
// k_kv_release) checks every index of the call and counts the pages it needs before
// anything is written, and takes the lowest free pages in the order of the list, so
// results do not depend on timing.  A call that cannot be done sets *status, and
// while that is set no call on the cache does anything.
#include "g4_device.hpp"
#include "g4_internal.hpp"

namespace g4 {

constexpr int KV_T = 1024;  // threads of the bookkeeping workgroup, one per list entry

static_assert(KV_T >= KV_MAX_SEQS, "one thread per entry");

// Exclusive sums of N numbers over a workgroup of KV_T threads; total: everyone's.  `ws`:
// N ints per wave.  Ends with a barrier, so that ws can be used again.
template <int N>
G4_DEV void block_scan(int (&v)[N], int *ws, int (&total)[N]) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  int x[N], mine[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = wave_scan(v[i]);
    if (lane == 63) ws[N * wid + i] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {  // a lane for each wave
    const int t = wave_scan(lane < KV_T / 64 ? ws[N * lane + i] : 0);
    total[i] = __builtin_amdgcn_readlane(t, KV_T / 64 - 1);
    mine[i] = wid ? __shfl(t, wid - 1) : 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = mine[i] + x[i] - v[i];
}

G4_DEV int block_scan(int v, int *ws, int *total) {
  int a[1] = {v}, t[1];
  block_scan(a, ws, t);
  *total = t[0];
  return a[0];
}

G4_DEV int64_t block_sum_i64(int64_t v, int64_t *ws) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  if (lane == 0) ws[wid] = v;
  __syncthreads();
  int64_t all = 0;
  for (int w = 0; w < KV_T / 64; ++w) all += ws[w];
  __syncthreads();
  return all;
}

G4_DEV bool in_range(int v, int n) { return (unsigned)v < (unsigned)n; }

// A cached length as kernels use it: never past the table.
G4_DEV int safe_length(const KvArgs &kv, int seq) {
  return in_range(seq, kv.max_seqs) ? min(max(kv.lengths[seq], 0), kv.max_pages << kv.shift) : 0;
}

// The last i with begin[i] <= x, for begin[0] = lo of n + 1 rising entries (n >= 1).
G4_DEV int find_entry(const int *begin, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (begin[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Which of a thread's four pages from `base` on are free: bit j for page base + 4 thread + j.
G4_DEV int four_free(const KvArgs &kv, int64_t base) {
  typedef int32_t i32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
  const int64_t p0 = base + 4 * (int64_t)threadIdx.x;
  int f = 0;
  if (p0 + 4 <= kv.n_pages) {
    const i32x4a4 r = *(const i32x4a4 *)(kv.refs + p0);
#pragma unroll
    for (int j = 0; j < 4; ++j) f |= (r[j] == 0) << j;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f |= (p0 + j < kv.n_pages && kv.refs[p0 + j] == 0) << j;
  }
  return f;
}

// Calls give(rank, page) for the `total` lowest free pages, from a whole workgroup.
// Returns the number found, at most total.  f: four_free(kv, 0).
template <class F>
G4_DEV int lowest_free(const KvArgs &kv, int total, int *ws, int f, F give) {
  int found = 0;
  for (int64_t base = 0; base < kv.n_pages && found < total; base += 4 * KV_T) {
    if (base > 0) f = four_free(kv, base);
    const int p0 = (int)base + 4 * threadIdx.x;
    int all, rank = found + block_scan(__builtin_popcount(f), ws, &all);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f >> j & 1) {
        if (rank < total) give(rank, p0 + j);
        ++rank;
      }
    found += all;
  }
  return min(found, total);
}

// ------------------------------------------------------------ bookkeeping ----

__global__ __launch_bounds__(256) void k_kv_init(KvArgs kv) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t j = i; j < (int64_t)kv.max_seqs * kv.max_pages; j += step) kv.table[j] = -1;
  for (int64_t j = i; j < kv.n_pages; j += step) kv.refs[j] = 0;
  for (int64_t j = i; j < kv.max_seqs; j += step) kv.lengths[j] = 0;
  if (i == 0) *kv.status = KV_OK;
}

// lengths[seqs[i]] += counts[i], with the pages that takes.  The free pages are found
// by counting refs, 4096 at a time: latency, as in k_kv_plan (4.2 us for 32 sequences that grow
// by a token, 4.7 for 1024).
__global__ __launch_bounds__(KV_T) void k_kv_extend(KvArgs kv, int n, const int32_t *seqs, const int32_t *counts) {
  __shared__ int mark[KV_MAX_SEQS], first[KV_T + 1], row[KV_T], have[KV_T], ws[KV_T / 64];
  __shared__ int64_t ws64[KV_T / 64];
  const int tid = threadIdx.x;
  if (*kv.status != KV_OK) return;
  mark[tid] = 0;
  __syncthreads();
  int seq = 0, len = 0, count = 0, need = 0;
  bool bad = false;
  if (tid < n) {
    seq = seqs[tid];
    count = counts[tid];
    bad = !in_range(seq, kv.max_seqs);
    if (!bad) {
      bad = atomicAdd(&mark[seq], 1) > 0;
      len = kv.lengths[seq];
      const int64_t to = (int64_t)len + count;
      bad |= len < 0 || count < 0 || to > (int64_t)kv.max_pages << kv.shift;
    }
    if (!bad) {
      have[tid] = (len + kv.page - 1) >> kv.shift;
      need = ((len + count + kv.page - 1) >> kv.shift) - have[tid];
      row[tid] = seq;
    }
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) *kv.status = KV_BAD_DATA;
    return;
  }
  const int64_t total64 = block_sum_i64(need, ws64);
  int total;
  const int f = block_scan(need, ws, &total);
  first[tid] = f;
  __syncthreads();
  // the pages are counted before the first is given out
  if (total64 > 0) {
    const int free4 = four_free(kv, 0);
    const int found = total64 > kv.n_pages ? 0 : lowest_free(kv, total, ws, free4, [](int, int) {});
    if (found < total64) {
      if (tid == 0) *kv.status = KV_NO_PAGES;
      return;
    }
    lowest_free(kv, total, ws, free4, [&](int rank, int page) {
      const int e = find_entry(first, n, rank);
      kv.table[(int64_t)row[e] * kv.max_pages + have[e] + rank - first[e]] = page;
      kv.refs[page] = 1;
    });
  }
  if (tid < n) kv.lengths[seq] = len + count;
}

// Pages of the listed sequences given back: all of them (window < 0), or those that no
// later position of a sliding window with `sinks` first tokens sees.  A wave takes every 16th
// sequence, one dependent load after the other: 3.7 us for 32 sequences, 34 for 1024.
__global__ __launch_bounds__(KV_T) void k_kv_release(KvArgs kv, int n, const int32_t *seqs, int window, int sinks) {
  __shared__ int mark[KV_MAX_SEQS];
  const int tid = threadIdx.x, lane = tid & 63;
  if (*kv.status != KV_OK) return;
  mark[tid] = 0;
  __syncthreads();
  bool bad = false;
  if (tid < n) {
    const int seq = seqs[tid];
    bad = !in_range(seq, kv.max_seqs) || atomicAdd(&mark[seq], 1) > 0;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) *kv.status = KV_BAD_DATA;
    return;
  }
  for (int e = tid >> 6; e < n; e += KV_T / 64) {
    const int seq = seqs[e], len = safe_length(kv, seq);
    int from = 0, to = (len + kv.page - 1) >> kv.shift;
    if (window >= 0) {
      from = (int)(((int64_t)sinks + kv.page - 1) >> kv.shift);
      to = len > window ? (len - window + 1) >> kv.shift : 0;  // the last token of a freed page is <= len - window
      to = min(to, kv.max_pages);
    }
    for (int p = from + lane; p < to; p += 64) {
      int32_t *at = kv.table + (int64_t)seq * kv.max_pages + p;
      const int page = *at;
      if (in_range(page, kv.n_pages)) atomicAdd(&kv.refs[page], -1);
      *at = -1;
    }
    if (window < 0 && lane == 0) kv.lengths[seq] = 0;
  }
}

// ---- fork and compact: sequence dst[i] becomes the first prefix[i] tokens of src[i]
// and then its listed tokens.  Whole pages of the prefix are shared; what follows goes
// to fresh pages, free before the call, so that no copy reads a page another writes.
struct Plan {
  int32_t *ok;          // 1: the call can be done
  int32_t *bad;         // per workgroup of k_kv_resolve: a listed token is not there
  int32_t *shared;      // [n] pages taken over from src
  int32_t *prefix;      // [n] tokens that stay where they are
  int32_t *length;      // [n] the new length
  int32_t *fresh_begin; // [n + 1] into fresh
  int32_t *copy_begin;  // [n + 1] over the tokens to copy
  int32_t *src_page;    // [n] the page of src that the prefix ends in
  int32_t *fresh;       // pages
  int32_t *resolved;    // [n_keep] page * tokens of a page + place in it
  int32_t n_bad;
  int32_t fresh_cap;
};

constexpr int KV_RES = 256;  // listed tokens per workgroup of k_kv_resolve

static size_t plan_layout(const KvArgs &kv, const KvMove &m, char *base, Plan *p) {
  size_t off = 0;
  auto add = [&](int64_t n) {
    int32_t *at = (int32_t *)(base + off);
    off += ((size_t)n * 4 + 255) & ~size_t(255);
    return at;
  };
  p->n_bad = (m.n_keep + KV_RES - 1) / KV_RES;
  const int64_t cap = (int64_t)m.n_keep / kv.page + 2 * (int64_t)m.n + 1;
  p->fresh_cap = (int32_t)(cap < kv.n_pages ? cap : kv.n_pages);
  p->ok = add(1);
  p->bad = add(p->n_bad);
  p->shared = add(m.n);
  p->prefix = add(m.n);
  p->length = add(m.n);
  p->fresh_begin = add(m.n + 1);
  p->copy_begin = add(m.n + 1);
  p->src_page = add(m.n);
  p->fresh = add(p->fresh_cap);
  p->resolved = add(m.n_keep);
  return off;
}

size_t kv_move_scratch_bytes(const KvArgs &kv, const KvMove &m) {
  Plan p;
  return plan_layout(kv, m, nullptr, &p);
}

// Where each listed token is: two dependent loads each, 5 us for 18000 tokens, which one
// workgroup (k_kv_plan's) would take 18 rounds for.
__global__ __launch_bounds__(KV_RES) void k_kv_resolve(KvArgs kv, KvMove m, Plan p) {
  __shared__ int begin[KV_MAX_SEQS];
  if (*kv.status != KV_OK) return;
  for (int i = threadIdx.x; i < m.n; i += KV_RES) begin[i] = m.keep_begin[i];
  __syncthreads();
  const int t = blockIdx.x * KV_RES + threadIdx.x;
  bool bad = false;
  if (t < m.n_keep && t >= begin[0] && t < m.keep_begin[m.n]) {
    const int seq = m.src[find_entry(begin, m.n, t)], tok = m.keep[t];
    int at = -1;
    if (in_range(seq, kv.max_seqs) && in_range(tok, safe_length(kv, seq))) {
      const int page = kv.table[(int64_t)seq * kv.max_pages + (tok >> kv.shift)];
      if (in_range(page, kv.n_pages)) at = (page << kv.shift) + (tok & (kv.page - 1));
    }
    p.resolved[t] = at;
    bad = at < 0;
  }
  const int any = __syncthreads_or(bad);
  if (threadIdx.x == 0) p.bad[blockIdx.x] = any;
}

// Checks the call, counts what it needs and lists the fresh pages.  One workgroup: 5 us
// for 64 entries and 4000 pages, of which a launch is 2; its loads depend on each other
// (lists, lengths, table, refs).  Sums by lane permutes and two counts a barrier took it
// from 6.5 us.
__global__ __launch_bounds__(KV_T) void k_kv_plan(KvArgs kv, KvMove m, Plan p) {
  __shared__ int mark[KV_MAX_SEQS], taken[KV_MAX_SEQS], ws[2 * KV_T / 64];  // taken: full pages that an entry shares
  const int tid = threadIdx.x, status = *kv.status;
  const int free4 = four_free(kv, 0);  // on its way while the lists are read
  mark[tid] = taken[tid] = 0;
  bool bad = false;
  for (int i = tid; i < p.n_bad; i += KV_T) bad |= p.bad[i] != 0;
  __syncthreads();
  if (status != KV_OK) {
    if (tid == 0) *p.ok = 0;
    return;
  }
  int src = 0, prefix = 0, shared = 0, length = 0, need = 0, copies = 0, src_page = -1;
  bool stays = false;
  if (tid < m.n) {
    src = m.src[tid];
    const int dst = m.dst[tid];
    bool off = !in_range(src, kv.max_seqs) || !in_range(dst, kv.max_seqs);
    if (!off) {
      off = atomicAdd(&mark[dst], 1) > 0;
      const int len = kv.lengths[src];
      prefix = m.prefix ? m.prefix[tid] : m.keep_begin ? 0 : len;
      int listed = 0;
      if (m.keep_begin) {
        const int a = m.keep_begin[tid], b = m.keep_begin[tid + 1];
        off |= a < 0 || b < a || b > m.n_keep || (tid == 0 && a != 0);
        listed = b - a;
      }
      off |= prefix < 0 || prefix > len || (int64_t)len > (int64_t)kv.max_pages << kv.shift;
      off |= (int64_t)prefix + listed > (int64_t)kv.max_pages << kv.shift;
      if (!off) {
        length = prefix + listed;
        shared = prefix >> kv.shift;
        atomicMax(&taken[src], shared);
        if (prefix & (kv.page - 1)) {
          src_page = kv.table[(int64_t)src * kv.max_pages + shared];
          off = !in_range(src_page, kv.n_pages);
          stays = !off && src == dst && listed == 0 && kv.refs[src_page] == 1;
        }
      }
    }
    bad |= off;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) *kv.status = KV_BAD_DATA, *p.ok = 0;
    return;
  }
  if (tid < m.n) {
    // A sequence that stays where it is keeps its last page if no other holds it, before the
    // call or after it: a longer continuation takes the page over as a full one, and its
    // tokens behind this prefix with it.
    if (stays && taken[src] <= shared) ++shared;
    need = max(0, ((length + kv.page - 1) >> kv.shift) - shared);
    copies = max(0, length - (shared << kv.shift));
  }
  // The lists of kept tokens follow each other, so the copies are at most n_keep + n * page,
  // which the host has checked, and the pages fewer.
  int sums[2] = {need, copies}, all[2];
  block_scan(sums, ws, all);
  if (tid < m.n) {
    p.prefix[tid] = prefix;
    p.shared[tid] = shared;
    p.length[tid] = length;
    p.src_page[tid] = src_page;
    p.fresh_begin[tid] = sums[0];
    p.copy_begin[tid] = sums[1];
  }
  if (tid == 0) p.fresh_begin[m.n] = all[0], p.copy_begin[m.n] = all[1];
  int found = 0;
  if (all[0] <= p.fresh_cap)
    found = lowest_free(kv, all[0], ws, free4, [&](int rank, int page) { p.fresh[rank] = page; });
  if (tid == 0) {
    *p.ok = found == all[0];
    if (found != all[0]) *kv.status = KV_NO_PAGES;
  }
}

// The copies (workgroups below n_copy: `per` tokens of one layer each), and the new
// rows of the table, 16 columns a workgroup: every old row is read before one is
// written, since a sequence can be another's source.  Bound by memory: 64 forks of 16
// prompts copy 55 MB in 23.5 us (4.7 TB/s read and written; a large copy reaches 5.1),
// tokens kept out of 16 sequences 169 MB in 74 us (4.6 TB/s, rows of 256 bytes).
constexpr int KV_COLS = 16;

__global__ __launch_bounds__(256) void k_kv_move(KvArgs kv, KvMove m, Plan p, int n_copy, int per) {
  extern __shared__ int lds[];
  const int tid = threadIdx.x;
  if (*p.ok == 0) return;
  if ((int)blockIdx.x < n_copy) {
    const int total = p.copy_begin[m.n];
    const int groups = (total + per - 1) / per;
    for (int64_t w = blockIdx.x; w < (int64_t)groups * kv.n_layers; w += n_copy) {
      const int layer = (int)(w / groups), c0 = (int)(w % groups) * per, c1 = min(total, c0 + per);
      if (w == blockIdx.x) {
        for (int i = tid; i < m.n; i += 256) lds[i] = p.copy_begin[i];
        __syncthreads();
      }
      const int row = kv.hs * (kv.type == T_F32 ? 4 : 2) / 16;  // 16-byte words of a token of a head
      const int words = row * kv.n_kv;
      const int64_t base = (int64_t)layer * kv.n_pages * kv.n_kv * kv.page * row;
      for (int i = tid; i < (c1 - c0) * words; i += 256) {
        const int c = c0 + i / words, j = i % words, h = j / row, x = j % row;
        const int e = find_entry(lds, m.n, c);
        const int pos = (p.shared[e] << kv.shift) + c - lds[e];
        const int at = pos < p.prefix[e] ? (p.src_page[e] << kv.shift) + (pos & (kv.page - 1))
                                         : p.resolved[m.keep_begin[e] + pos - p.prefix[e]];
        const int to = p.fresh[p.fresh_begin[e] + (pos >> kv.shift) - p.shared[e]];
        const int64_t from = base + ((int64_t)(at >> kv.shift) * kv.n_kv + h) * kv.page * row +
                             (int64_t)(at & (kv.page - 1)) * row + x;
        const int64_t dest = base + ((int64_t)to * kv.n_kv + h) * kv.page * row + (int64_t)(pos & (kv.page - 1)) * row + x;
        ((u32x4 *)kv.k)[dest] = ((const u32x4 *)kv.k)[from];
        ((u32x4 *)kv.v)[dest] = ((const u32x4 *)kv.v)[from];
      }
    }
    return;
  }
  const int c0 = ((int)blockIdx.x - n_copy) * KV_COLS;
  for (int i = tid; i < m.n * KV_COLS; i += 256) {
    const int e = i / KV_COLS, col = c0 + i % KV_COLS;
    lds[i] = col < min(p.shared[e], kv.max_pages) ? kv.table[(int64_t)m.src[e] * kv.max_pages + col] : -1;
  }
  __syncthreads();
  for (int i = tid; i < m.n * KV_COLS; i += 256) {
    const int e = i / KV_COLS, col = c0 + i % KV_COLS;
    if (col >= kv.max_pages) continue;
    int32_t *at = kv.table + (int64_t)m.dst[e] * kv.max_pages + col;
    const int old = *at, fresh = p.fresh_begin[e] + col - p.shared[e];
    int page = -1;
    if (in_range(old, kv.n_pages)) atomicAdd(&kv.refs[old], -1);
    if (col < p.shared[e]) {
      if (in_range(lds[i], kv.n_pages)) page = lds[i];
    } else if (fresh < p.fresh_begin[e + 1]) {
      page = p.fresh[fresh];
    }
    if (page >= 0) atomicAdd(&kv.refs[page], 1);
    *at = page;
    if (col == 0) kv.lengths[m.dst[e]] = p.length[e];
  }
}

hipError_t launch_kv_init(const KvArgs &kv, hipStream_t s) {
  int64_t n = (int64_t)kv.max_seqs * kv.max_pages;
  if (n < kv.n_pages) n = kv.n_pages;
  const int64_t blocks = (n + 255) / 256;
  hipLaunchKernelGGL(k_kv_init, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, s, kv);
  return hipGetLastError();
}

hipError_t launch_kv_extend(const KvArgs &kv, int32_t n, const int32_t *seqs, const int32_t *counts, hipStream_t s) {
  hipLaunchKernelGGL(k_kv_extend, dim3(1), dim3(KV_T), 0, s, kv, n, seqs, counts);
  return hipGetLastError();
}

hipError_t launch_kv_release(const KvArgs &kv, int32_t n, const int32_t *seqs, int32_t window, int32_t sinks,
                             hipStream_t s) {
  hipLaunchKernelGGL(k_kv_release, dim3(1), dim3(KV_T), 0, s, kv, n, seqs, window, sinks);
  return hipGetLastError();
}

hipError_t launch_kv_move(const KvArgs &kv, const KvMove &m, char *scratch, hipStream_t s) {
  Plan p;
  plan_layout(kv, m, scratch, &p);
  if (m.n_keep > 0) {
    hipLaunchKernelGGL(k_kv_resolve, dim3(p.n_bad), dim3(KV_RES), 0, s, kv, m, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(KV_T), 0, s, kv, m, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int row = kv.n_kv * kv.hs * (kv.type == T_F32 ? 4 : 2) / 16;
  const int per = row >= 1024 ? 1 : 1024 / row;  // about four words of K and of V for each thread
  const int64_t tokens = (int64_t)m.n_keep + (int64_t)m.n * kv.page;
  const int64_t work = (tokens + per - 1) / per * kv.n_layers;
  const int n_copy = (int)(work < 65536 ? work : 65536);
  const int cols = (kv.max_pages + KV_COLS - 1) / KV_COLS;
  hipLaunchKernelGGL(k_kv_move, dim3(n_copy + cols), dim3(256), (size_t)m.n * KV_COLS * 4, s, kv, m, p, n_copy, per);
  return hipGetLastError();
}

// --------------------------------------------------------- rotary positions ----

// cos and sin of position * freq, times gain.  The angle is taken in turns in double
// precision and reduced there: at position 10^6 its error stays below 2^-25 turns,
// where fp32 would be off by 0.1 radian.
G4_DEV void turn_of(double pos, double freq, float gain, float &c, float &s) {
  const double t = pos * freq * 0.15915494309189533577;  // 1 / (2 pi)
  const float r = (float)(t - __builtin_rint(t));
  float sn, cs;
  sincospif(2.f * r, &sn, &cs);
  c = cs * gain, s = sn * gain;
}

template <int N>
G4_DEV void load_floats(const float *p, float (&v)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 t = ((const float4 *)p)[i];
      v[4 * i] = t.x, v[4 * i + 1] = t.y, v[4 * i + 2] = t.z, v[4 * i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}

// fp32 to the cache's type, to nearest (F16 overflows to infinity)
template <int TYPE>
G4_DEV uint32_t to_half(float f) {
  if constexpr (TYPE == T_F16) return (uint32_t)__half_as_ushort(__float2half_rn(f));
  else return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f);
}

template <int TYPE, int N>
G4_DEV void store_as(char *base, int64_t elem, const float (&v)[N]) {
  if constexpr (TYPE == T_F32) {
    float *p = (float *)base + elem;
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        ((float4 *)p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = v[i];
    }
  } else {
    uint16_t *p = (uint16_t *)base + elem;
    if constexpr (N >= 4) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        uint2 w;
        w.x = to_half<TYPE>(v[4 * i]) | to_half<TYPE>(v[4 * i + 1]) << 16;
        w.y = to_half<TYPE>(v[4 * i + 2]) | to_half<TYPE>(v[4 * i + 3]) << 16;
        ((uint2 *)p)[i] = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = (uint16_t)to_half<TYPE>(v[i]);
    }
  }
}

// The two runs of N elements that unit u of a head covers: N pairs of the rotated part,
// or 2N elements behind it.  Both runs lie next to each other where the pairs do.
template <int N>
G4_DEV void unit_at(const RopeArgs &r, int u, int &a, int &b, bool &turn) {
  turn = u * N < r.rot / 2;
  a = turn && !r.pairs ? u * N : 2 * N * u;
  b = turn && !r.pairs ? u * N + r.rot / 2 : a + N;
}

template <int N>
G4_DEV void rotate(bool turn, bool pairs, const float (&c)[N], const float (&s)[N], float (&x)[N], float (&y)[N]) {
  if (!turn) return;
  if (!pairs) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float a = x[i], b = y[i];
      x[i] = a * c[i] - b * s[i];
      y[i] = b * c[i] + a * s[i];
    }
  } else {  // pair i is elements 2i and 2i + 1 of x, y
    float v[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x[i], v[N + i] = y[i];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float a = v[2 * i], b = v[2 * i + 1];
      v[2 * i] = a * c[i] - b * s[i];
      v[2 * i + 1] = b * c[i] + a * s[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i], y[i] = v[N + i];
  }
}

// A write is all or nothing.  Its rows are looked at through LDS lists of its entries:
struct WriteList {
  int mark[KV_MAX_SEQS];       // times that a sequence is named
  int first[KV_MAX_SEQS + 1];  // first row of an entry
  int len[KV_MAX_SEQS];
  int seq[KV_MAX_SEQS];
};

G4_DEV int page_of(const KvArgs &kv, int seq, int len, int pos) {  // -1: out of range
  return in_range(pos, len) ? kv.table[(int64_t)seq * kv.max_pages + (pos >> kv.shift)] : -1;
}

// A page that can be written: it is there, and no other sequence holds it.
G4_DEV bool own_page(const KvArgs &kv, int page) { return in_range(page, kv.n_pages) && kv.refs[page] == 1; }

// The entries read into the list by T threads.  True: the thread met one that does not rise.
template <int T>
G4_DEV bool read_write_list(const KvArgs &kv, const KvWrite &w, WriteList &l) {
  bool bad = false;
  for (int i = threadIdx.x; i < kv.max_seqs; i += T) l.mark[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < w.n; i += T) {
    const int seq = w.seqs[i];
    int from = i, to = i + 1;
    if (w.row_begin) {
      from = w.row_begin[i], to = w.row_begin[i + 1];
      bad |= from < 0 || to < from || to > w.n_rows;
    }
    l.first[i] = from;
    if (i + 1 == w.n) l.first[w.n] = to;
    l.seq[i] = seq, l.len[i] = safe_length(kv, seq);
    if (in_range(seq, kv.max_seqs)) atomicAdd(&l.mark[seq], 1);
  }
  return bad;
}

// Then the pages: those of the first and last row of each entry, and those between, each of
// which holds a row whose number is a multiple of a page's tokens.  `meanwhile` is done
// while the thread's first pages are on their way.
template <int T, class F>
G4_DEV bool check_write_list(const KvArgs &kv, const KvWrite &w, const WriteList &l, F meanwhile) {
  bool bad = false;
  auto ends = [&](int i, int &a, int &b) {  // false: an entry without rows needs no page
    const int rows = i < w.n ? l.first[i + 1] - l.first[i] : 0;
    if (rows == 0) return false;
    a = page_of(kv, l.seq[i], l.len[i], l.len[i] - rows);
    b = rows > 1 ? page_of(kv, l.seq[i], l.len[i], l.len[i] - 1) : a;
    return true;
  };
  auto check = [&](int i, int a, int b) { bad |= !own_page(kv, a) || (b != a && !own_page(kv, b)) || l.mark[l.seq[i]] > 1; };
  int a, b;
  const bool some = ends(threadIdx.x, a, b);
  meanwhile();
  if (some) check(threadIdx.x, a, b);
  for (int i = threadIdx.x + T; i < w.n; i += T)
    if (ends(i, a, b)) check(i, a, b);
  if (w.row_begin)
    for (int64_t row = (int64_t)threadIdx.x << kv.shift; row < l.first[w.n]; row += (int64_t)T << kv.shift) {
      if (row < l.first[0]) continue;
      const int e = find_entry(l.first, w.n, (int)row);
      bad |= !own_page(kv, page_of(kv, l.seq[e], l.len[e], l.len[e] - l.first[e + 1] + (int)row));
    }
  return bad;
}

__global__ __launch_bounds__(KV_T) void k_kv_write_check(KvArgs kv, KvWrite w) {
  __shared__ WriteList l;
  if (*kv.status != KV_OK) return;
  bool bad = __syncthreads_or(read_write_list<KV_T>(kv, w, l));
  if (!bad) bad = __syncthreads_or(check_write_list<KV_T>(kv, w, l, [] {}));
  if (bad && threadIdx.x == 0) *kv.status = KV_BAD_DATA;
}

// A workgroup turns a stretch of the heads of one row (blockIdx.x; blockIdx.y of
// gridDim.y stretches): thread (slot, u) takes unit u of every slots-th head and so
// forms its cosines once.  Heads 0 .. n_heads - 1 are q, then n_kv of k, then n_kv of v.
// CHECK: every workgroup looks at the whole call before it writes.  All find the same, so a
// call that cannot be done writes nothing, whichever of them sets *status first; otherwise
// k_kv_write_check has looked.
// Bound by memory for prompts and by latency for single rows: 7900 rows of 32/4 heads of 128,
// F16: 55 us, 5.6 TB/s, and 5 us for k_kv_write_check; 32 rows of 16/8 heads of 256, BF16: 5.8 us,
// 1 us of it the look at the whole call.
template <int TYPE, int N, bool CHECK>
__global__ __launch_bounds__(256) void k_kv_write(KvArgs kv, RopeArgs r, KvWrite w) {
  __shared__ WriteList l;
  const int row = blockIdx.x, tid = threadIdx.x;
  const int status = *kv.status;
  const int units = kv.hs / (2 * N), slots = 256 / units, slot = tid / units, u = tid % units;
  const int heads = w.n_heads + 2 * kv.n_kv;
  const int per = (heads + gridDim.y - 1) / gridDim.y;
  const int h0 = blockIdx.y * per, h1 = slot < slots ? min(heads, h0 + per) : 0;
  int a, b;
  bool turn;
  unit_at<N>(r, u, a, b, turn);
  float x[N], y[N];
  auto load = [&](int h) {
    const float *from = h < w.n_heads ? w.q + ((int64_t)row * w.n_heads + h) * kv.hs
                        : h < w.n_heads + kv.n_kv
                            ? w.k + ((int64_t)row * kv.n_kv + h - w.n_heads) * kv.hs
                            : w.v + ((int64_t)row * kv.n_kv + h - w.n_heads - kv.n_kv) * kv.hs;
    load_floats<N>(from + a, x);
    load_floats<N>(from + b, y);
  };
  if (h0 + slot < h1) load(h0 + slot);  // on its way while the row's place is looked up
  if constexpr (CHECK) {
    // A wave may see what another workgroup of this launch has set: all waves decide together.
    if (__syncthreads_or(read_write_list<256>(kv, w, l) || status != KV_OK)) {
      if (tid == 0) atomicCAS(kv.status, KV_OK, KV_BAD_DATA);
      return;
    }
  } else {
    if (status != KV_OK) return;  // nobody sets it in this launch
    if (w.row_begin) {
      for (int i = tid; i <= w.n; i += 256) l.first[i] = w.row_begin[i];
      __syncthreads();
    }
  }
  int e = row, to_end = 1;  // the row's entry, and how far before its end the row stands
  bool mine = true;         // rows of no sequence are left as they are
  if (w.row_begin) {
    mine = row >= l.first[0] && row < l.first[w.n];
    e = find_entry(l.first, w.n, row);
    to_end = l.first[e + 1] - row;
  }
  const int seq = CHECK ? l.seq[e] : w.seqs[e], len = CHECK ? l.len[e] : safe_length(kv, seq);
  const int pos = len - to_end, page = mine ? page_of(kv, seq, len, pos) : -1;
  float c[N], s[N];
  auto turns = [&] {
    if (turn && h0 + slot < min(h1, w.n_heads + kv.n_kv))
#pragma unroll
      for (int i = 0; i < N; ++i) turn_of((double)pos, r.freqs[u * N + i], r.gain, c[i], s[i]);
  };
  if constexpr (CHECK) {
    if (__syncthreads_or(check_write_list<256>(kv, w, l, turns))) {
      if (tid == 0) atomicCAS(kv.status, KV_OK, KV_BAD_DATA);
      return;
    }
  } else {
    turns();
  }
  if (!in_range(page, kv.n_pages)) return;
  for (int h = h0 + slot; h < h1;) {
    const bool is_q = h < w.n_heads, is_k = !is_q && h < w.n_heads + kv.n_kv;
    rotate<N>(turn && (is_q || is_k), r.pairs, c, s, x, y);
    if (is_q) {
      float *to = w.q_out + ((int64_t)row * w.n_heads + h) * kv.hs;
      store_as<T_F32, N>((char *)to, a, x);
      store_as<T_F32, N>((char *)to, b, y);
    } else {
      const int kh = is_k ? h - w.n_heads : h - w.n_heads - kv.n_kv;
      const int64_t at_page = ((((int64_t)w.layer * kv.n_pages + page) * kv.n_kv + kh) * kv.page + (pos & (kv.page - 1))) *
                              (int64_t)kv.hs;
      store_as<TYPE, N>(is_k ? kv.k : kv.v, at_page + a, x);
      store_as<TYPE, N>(is_k ? kv.k : kv.v, at_page + b, y);
    }
    h += slots;
    if (h < h1) load(h);
  }
}

// Rows at given positions, as k_kv_write turns them; bound by memory: 7900 rows of 32 heads of
// 128 take 39.5 us (259 MB, some of which stay in the last-level cache), 32 of 16 of 256 3.4 us.
template <int N>
__global__ __launch_bounds__(256) void k_rope(RopeArgs r, const float *x, float *out, int n_heads, int hs,
                                              const int32_t *positions) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, units = hs / (2 * N);
  const double pos = (double)positions[row];
  const int per = (n_heads + gridDim.y - 1) / gridDim.y;
  const int h0 = blockIdx.y * per, h1 = min(n_heads, h0 + per);
  const int wide = min(units, 256), slots = 256 / wide, slot = tid / wide;
  if (slot >= slots) return;
  for (int u = tid % wide; u < units; u += wide) {
    int a, b;
    bool turn;
    unit_at<N>(r, u, a, b, turn);
    float c[N], s[N];
    if (turn)
#pragma unroll
      for (int i = 0; i < N; ++i) turn_of(pos, r.freqs[u * N + i], r.gain, c[i], s[i]);
    for (int h = h0 + slot; h < h1; h += slots) {
      const int64_t at = (row * n_heads + h) * hs;
      float p[N], q[N];
      load_floats<N>(x + at + a, p);
      load_floats<N>(x + at + b, q);
      rotate<N>(turn, r.pairs, c, s, p, q);
      store_as<T_F32, N>((char *)out, at + a, p);
      store_as<T_F32, N>((char *)out, at + b, q);
    }
  }
}

// Workgroups per row: few rows spread their heads over more of the chip.
static unsigned row_split(int32_t n_rows, int heads, int slots) {
  const int most = (heads + slots - 1) / slots;
  int y = 512 / (n_rows > 0 ? n_rows : 1);
  if (y < 1) y = 1;
  return (unsigned)(y < most ? y : most);
}

static bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

hipError_t launch_rope(const RopeArgs &r, const float *x, float *out, int32_t n_rows, int32_t n_heads, int32_t hs,
                       const int32_t *positions, hipStream_t s) {
  // runs of four floats where both ends of every run are 16-byte aligned
  if (r.rot % 8 == 0 && hs % 8 == 0 && aligned16(x) && aligned16(out)) {
    const int units = hs / 8, slots = units < 256 ? 256 / units : 1;
    hipLaunchKernelGGL(k_rope<4>, dim3(n_rows, row_split(n_rows, n_heads, slots)), dim3(256), 0, s, r, x, out, n_heads,
                       hs, positions);
  } else {
    const int units = hs / 2, slots = units < 256 ? 256 / units : 1;
    hipLaunchKernelGGL(k_rope<1>, dim3(n_rows, row_split(n_rows, n_heads, slots)), dim3(256), 0, s, r, x, out, n_heads,
                       hs, positions);
  }
  return hipGetLastError();
}

template <int TYPE, bool CHECK>
static void launch_write(const KvArgs &kv, const RopeArgs &r, const KvWrite &w, hipStream_t s) {
  const int heads = w.n_heads + 2 * kv.n_kv;
  if (r.rot % 8 == 0 && aligned16(w.q) && aligned16(w.q_out) && aligned16(w.k) && aligned16(w.v))
    hipLaunchKernelGGL((k_kv_write<TYPE, 4, CHECK>), dim3(w.n_rows, row_split(w.n_rows, heads, 256 / (kv.hs / 8))),
                       dim3(256), 0, s, kv, r, w);
  else
    hipLaunchKernelGGL((k_kv_write<TYPE, 1, CHECK>), dim3(w.n_rows, row_split(w.n_rows, heads, 256 / (kv.hs / 2))),
                       dim3(256), 0, s, kv, r, w);
}

template <int TYPE>
static void launch_write(const KvArgs &kv, const RopeArgs &r, const KvWrite &w, bool check, hipStream_t s) {
  if (check) launch_write<TYPE, true>(kv, r, w, s);
  else launch_write<TYPE, false>(kv, r, w, s);
}

hipError_t launch_kv_write(const KvArgs &kv, const RopeArgs &r, const KvWrite &w, hipStream_t s) {
  // Few rows are looked at by every workgroup, many by one before them: 32 rows take 5.8 and
  // 7.2 us, 512 10.7 and 11.5, 2000 of one sequence 17.7 and 18.7, 2560 of 64 22.1 and 22.4, 3000
  // of three 23.9 and 23.8, 8000 of one 66.9 and 57.6.
  const bool check = w.n_rows <= 2048;
  if (!check) {
    hipLaunchKernelGGL(k_kv_write_check, dim3(1), dim3(KV_T), 0, s, kv, w);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (kv.type == T_F32) launch_write<T_F32>(kv, r, w, check, s);
  else if (kv.type == T_F16) launch_write<T_F16>(kv, r, w, check, s);
  else launch_write<T_BF16>(kv, r, w, check, s);
  return hipGetLastError();
}

}  // namespace g4
