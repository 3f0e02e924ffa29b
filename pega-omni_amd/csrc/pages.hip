// Pages of a paged cache (gfx950, wave64): forked requests share them, ended ones
// give them back, a pool moves below a limit, and what has to move is copied.
//
// shares[p] counts the lines that hold page p beside the first: 0 for a page that one
// line holds, and for a free one. So the row tables' takes and returns (tables.hip)
// need not know of it as long as a request shares nothing.
//
// Every workgroup works out by itself what the whole call amounts to (whether it can
// be made at all, which pages it takes), from the few numbers that say so, and then
// does its share: no order between workgroups. Counts go up and down by integer
// atomics, and what is put in an order (the queue, the moves) is put there by page
// id or by the call's own order, so that the results have the same bits every time.
#include "common.h"
#include "kernels.h"

#include <algorithm>

namespace omni {

namespace {

constexpr int kBad = 1, kPages = 3, kLine = 4, kExhausted = 5, kUnheld = 6;

__device__ __forceinline__ bool bad_state(int head, int avail, int num_pages) {
  return head < 0 || head >= num_pages || avail < 0 || avail > num_pages;
}

// Entry head + k of the free queue, 0 <= k <= num_pages.
__device__ __forceinline__ uint32_t queue_at(int head, int k, int num_pages) {
  const uint32_t i = (uint32_t)head + (uint32_t)k;
  return i >= (uint32_t)num_pages ? i - (uint32_t)num_pages : i;
}

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// ------------------------------------------------------------------ fork, free

// A call's lines, looked over by one workgroup: which lines it writes (`marked`), the
// code, and sums over the entries, all of them and those before entry `me`.
template <int THREADS>
struct Looked {
  uint32_t marked[kMostLines / 32];
  int codes[THREADS / 64], part[THREADS / 64], before[THREADS / 64];
  int pages[THREADS / 64];
};

// One workgroup per fork: the whole pages of the parent's line into the child's, a
// holder more for each, and the queue's next page for the part-filled one, in the
// order of the forks. Latency bounds it: the call's numbers, a page list, the stores,
// one after the other (224 forks of up to 250 pages move 0.5 MB: 5.8 us; 8 forks 4.4).
constexpr int kForkThreads = 256;

// What a workgroup's own entry is, and (asked for before it is known whether the call
// can be made) its thread's first page.
struct Mine {
  int tokens, held;
  const int32_t* line;
  int id0;
};

__device__ __forceinline__ Mine mine_of(const PagesArgs& a, const int32_t* lines) {
  const int me = blockIdx.x;
  Mine m{-1, 0, a.table, -1};
  if (me >= a.n) return m;
  m.tokens = a.tokens[me];
  const int line = lines[me];
  if (m.tokens <= 0 || line < 0 || line >= a.num_lines) return m;
  m.held = page_index(a.pd, m.tokens - 1) + 1;
  m.line = a.table + (int64_t)line * a.table_ld;
  if ((int)threadIdx.x < m.held && m.held <= a.table_ld) m.id0 = m.line[threadIdx.x];
  return m;
}

__global__ __launch_bounds__(kForkThreads) void pages_fork(PagesArgs a) {
  const int tid = threadIdx.x, me = blockIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ Looked<kForkThreads> s;
  const Mine mine = mine_of(a, a.parents);
  for (int i = tid; i < (a.num_lines + 31) / 32; i += kForkThreads) s.marked[i] = 0;
  const int head = a.free_state[0], avail = a.free_state[1];
  __syncthreads();
  int codes = bad_state(head, avail, a.num_pages) ? 1 << kBad : 0;
  int part = 0, before = 0, pages = 0;
  for (int i = tid; i < a.n; i += kForkThreads) {
    const int tokens = a.tokens[i], p = a.parents[i], c = a.lines[i];
    if (tokens < 0) continue;
    if (p < 0 || p >= a.num_lines || c < 0 || c >= a.num_lines) {
      codes |= 1 << kBad;
      continue;
    }
    const int held = tokens > 0 ? page_index(a.pd, tokens - 1) + 1 : 0, full = page_index(a.pd, tokens);
    if (held > a.table_ld) codes |= 1 << kLine;
    if (atomicOr(&s.marked[c >> 5], 1u << (c & 31)) >> (c & 31) & 1) codes |= 1 << kBad;  // a child twice
    part += held - full;
    before += i < me ? held - full : 0;
    pages = (int)min((uint32_t)pages + (uint32_t)full, 0x7fffffffu);
  }
  __syncthreads();
  for (int i = tid; i < a.n; i += kForkThreads) {  // a child that is a parent too
    const int p = a.parents[i];
    if (a.tokens[i] >= 0 && p >= 0 && p < a.num_lines && (s.marked[p >> 5] >> (p & 31) & 1)) codes |= 1 << kBad;
  }
#pragma unroll
  for (int c = kBad; c <= kExhausted; ++c)
    if (__any(codes >> c & 1)) codes |= 1 << c;
  part = wave_sum(part), before = wave_sum(before);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) pages = (int)min((uint32_t)pages + (uint32_t)__shfl_xor(pages, d), 0x7fffffffu);
  if (lane == 0) s.codes[wave] = codes, s.part[wave] = part, s.before[wave] = before, s.pages[wave] = pages;
  __syncthreads();
  codes = part = before = pages = 0;
#pragma unroll
  for (int w = 0; w < kForkThreads / 64; ++w) {
    codes |= s.codes[w], part += s.part[w], before += s.before[w];
    pages = (int)min((uint32_t)pages + (uint32_t)s.pages[w], 0x7fffffffu);
  }
  if (part > avail) codes |= 1 << kExhausted;
  const int code = codes ? __ffs(codes) - 1 : 0;
  if (me == 0 && tid == 0) {
    a.status[0] = code;
    a.status[1] = code ? 0 : part;
    a.status[2] = code ? 0 : pages;
    a.status[3] = code ? head : (int)queue_at(head, part, a.num_pages);
    a.status[4] = code ? avail : avail - part;
  }
  if (me >= a.n) return;
  if (code || mine.tokens < 0) {
    if (tid == 0) a.src[me] = a.dst[me] = -1;
    return;
  }
  int32_t* to = a.table_out + (int64_t)a.lines[me] * a.table_ld;
  const int full = page_index(a.pd, mine.tokens);
  for (int j = tid; j < full; j += kForkThreads) {
    const int id = j == tid ? mine.id0 : mine.line[j];
    to[j] = id;
    if (id >= 0 && id < a.num_pages) atomicAdd(a.shares + id, 1);
  }
  if (tid == 0) {
    const bool has_part = mine.held > full;
    const int id = has_part ? a.free_pages[queue_at(head, before, a.num_pages)] : -1;
    if (has_part) to[full] = id;
    a.src[me] = has_part ? mine.line[full] : -1;
    a.dst[me] = id;
  }
}

// Whether lines can be given back: the code, the same in every thread.
template <int THREADS>
__device__ __forceinline__ int free_code(const PagesArgs& a, Looked<THREADS>& s, int head, int avail) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < (a.num_lines + 31) / 32; i += THREADS) s.marked[i] = 0;
  __syncthreads();
  int codes = bad_state(head, avail, a.num_pages) ? 1 << kBad : 0, pages = 0;
  for (int i = tid; i < a.n; i += THREADS) {
    const int tokens = a.tokens[i], c = a.lines[i];
    if (tokens < 0) continue;
    if (c < 0 || c >= a.num_lines) {
      codes |= 1 << kBad;
      continue;
    }
    const int held = tokens > 0 ? page_index(a.pd, tokens - 1) + 1 : 0;
    if (held > a.table_ld) codes |= 1 << kLine;
    if (atomicOr(&s.marked[c >> 5], 1u << (c & 31)) >> (c & 31) & 1) codes |= 1 << kBad;  // a line twice
    pages = (int)min((uint32_t)pages + (uint32_t)held, 0x7fffffffu);
  }
#pragma unroll
  for (int c = kBad; c <= kLine; ++c)
    if (__any(codes >> c & 1)) codes |= 1 << c;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) pages = (int)min((uint32_t)pages + (uint32_t)__shfl_xor(pages, d), 0x7fffffffu);
  if (lane == 0) s.codes[wave] = codes, s.pages[wave] = pages;
  __syncthreads();
  codes = pages = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    codes |= s.codes[w];
    pages = (int)min((uint32_t)pages + (uint32_t)s.pages[w], 0x7fffffffu);
  }
  const int code = codes ? __ffs(codes) - 1 : 0;
  if (blockIdx.x == 0 && tid == 0) a.status[0] = code, a.status[2] = code ? 0 : pages;
  return code;
}

// Ended lines, a workgroup each: every page of theirs loses a holder. A page that had
// none beside this one is at -1 afterwards, which gather() looks for.
__global__ __launch_bounds__(kForkThreads) void pages_drop(PagesArgs a) {
  __shared__ Looked<kForkThreads> s;
  const Mine mine = mine_of(a, a.lines);
  if (free_code(a, s, a.free_state[0], a.free_state[1])) return;
  for (int j = threadIdx.x; j < mine.held; j += kForkThreads) {
    const int id = j == (int)threadIdx.x ? mine.id0 : mine.line[j];
    if (id >= 0 && id < a.num_pages) atomicSub(a.shares + id, 1);
  }
}

// The pages without a holder, in ascending order, to the queue's end. One workgroup,
// a wave for each sixteenth of the pool: counted, then written, from bits in LDS. A page
// that is in the queue already was held by nobody: the queue is looked through for those
// before anything joins it. SAME: the launch that dropped them, so that the counts are
// read where its atomics work, past the caches.
// Bound by round trips, a batch's under way while the one before is looked at: for the
// counts, eight rounds of a wave's, and the queue, 8192 entries, of which a thread's first
// is asked for beforehand. A fork of a few lines and their end, us: pools of 4600 pages
// with 600 in the queue 14.6, 31,000 with 30,930 21, 524,288 with 511,788 197 (287 when
// the counts were read twice, one batch after the other, and the queue not at all). All of
// the array asked for at the start, which needs no head, and 16 at a time were slower: the
// instructions of sixteen waves, 0.1 us for two dozen, count as much as a round trip.
constexpr int kGatherThreads = 1024;

struct Returned {
  uint64_t bits[kMostPool / 64];  // pages without a holder, where the pool has so many at most
  int count[kGatherThreads / 64];
  int twice;
};

// A thread's entries of the queue from entry k0 on, the last one again past its end.
constexpr int kQueueAhead = 8;
struct Queued {
  int id[kQueueAhead];
};
__device__ __forceinline__ int queued_at(const PagesArgs& a, uint32_t k, int head, int avail) {
  return a.free_pages[queue_at(head, (int)min(k, (uint32_t)avail - 1), a.num_pages)];
}
__device__ __forceinline__ Queued queued_from(const PagesArgs& a, uint32_t k0, int head, int avail) {
  Queued q;
#pragma unroll
  for (int i = 0; i < kQueueAhead; ++i) q.id[i] = queued_at(a, k0 + i * kGatherThreads + threadIdx.x, head, avail);
  return q;
}
// Its first entry, to be asked for early; none where the state is bad.
__device__ __forceinline__ int queued_first(const PagesArgs& a, int head, int avail) {
  return avail > 0 && !bad_state(head, avail, a.num_pages) ? queued_at(a, threadIdx.x, head, avail) : -1;
}

template <bool SAME>
__device__ __forceinline__ void gather(const PagesArgs& a, int code, int head, int avail, int queued0) {
  constexpr int kWaves = kGatherThreads / 64, kAhead = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ Returned s;
  const bool kept = a.num_pages <= kMostPool;
  // Rounds of 64 pages; the first `rounds % kWaves` waves have one more.
  const int rounds = (a.num_pages + 63) / 64;
  const int r0 = wave * (rounds / kWaves) + min(wave, rounds % kWaves), r1 = r0 + rounds / kWaves + (wave < rounds % kWaves ? 1 : 0);
  const auto holders = [&](int p) {
    return SAME ? __hip_atomic_load(a.shares + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : a.shares[p];
  };
  // The holders of kAhead rounds' pages from r on.
  const auto ask = [&](int r, int* v) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = r + i < r1 && 64 * (r + i) + lane < a.num_pages ? holders(64 * (r + i) + lane) : 0;
  };
  uint64_t free[kAhead] = {};
  int count = 0;
  if (kept)
    for (int r = r0 + lane; r < r1; r += 64) s.bits[r] = 0;
  int v[kAhead], next[kAhead] = {};
  ask(r0, v);
  for (int r = r0; r < r1; r += kAhead) {
    if (r + kAhead < r1) ask(r + kAhead, next);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) free[i] = __ballot(v[i] < 0), v[i] = next[i];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (free[i] == 0) continue;  // uniform
      count += __popcll(free[i]);
      if (kept && lane == 0) s.bits[r + i] = free[i];
    }
  }
  if (code) {  // nothing was dropped
    if (tid == 0) a.status[1] = 0, a.status[3] = head, a.status[4] = avail;
    return;
  }
  if (lane == 0) s.count[wave] = count;
  if (tid == 0) s.twice = 0;
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at += s.count[w];
    total += s.count[w];
  }
  bool twice = false;
  const auto back = [&](int id) {
    return id >= 0 && id < a.num_pages && (kept ? (s.bits[id >> 6] >> (id & 63) & 1) != 0 : holders(id) < 0);
  };
  if (total > 0) twice = back(queued0);
  if (total > 0 && avail > kGatherThreads) {
    Queued q = queued_from(a, kGatherThreads, head, avail);
    for (uint32_t k0 = kGatherThreads; k0 < (uint32_t)avail; k0 += kQueueAhead * kGatherThreads) {
      const Queued next = queued_from(a, k0 + kQueueAhead * kGatherThreads, head, avail);
#pragma unroll
      for (int i = 0; i < kQueueAhead; ++i) twice |= back(q.id[i]);
      q = next;
    }
  }
  if (twice) s.twice = 1;
  __syncthreads();
  // Else pages were given back that nobody held: they are in the queue, or there are more than were in use.
  const bool fits = !s.twice && total <= a.num_pages - avail;
  if (tid == 0) {
    if (!fits) a.status[0] = kUnheld;
    a.status[1] = fits ? total : 0;
    a.status[3] = head;
    a.status[4] = fits ? avail + total : avail;
  }
  if (count == 0) return;
  for (int r = r0; r < r1; r += kAhead) {
    if (r1 - r0 > kAhead) {  // else they are the ones at hand
      if (kept) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) free[i] = r + i < r1 ? s.bits[r + i] : 0;
      } else {
        ask(r, v);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) free[i] = __ballot(v[i] < 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int p = 64 * (r + i) + lane;
      if (free[i] >> lane & 1) {
        a.shares[p] = 0;
        if (fits) a.free_pages[queue_at(head, avail + at + __popcll(free[i] & ((1ull << lane) - 1)), a.num_pages)] = p;
      }
      at += __popcll(free[i]);
    }
  }
}

__global__ __launch_bounds__(kGatherThreads) void pages_gather(PagesArgs a) {
  const int head = a.free_state[0], avail = a.free_state[1];
  gather<false>(a, a.status[0], head, avail, queued_first(a, head, avail));
}

// Both for a few short lines, a wave each, in one workgroup and launch: 8 lines of 12
// pages 3.0 + 2.4 us apart.
__global__ __launch_bounds__(kGatherThreads) void pages_end(PagesArgs a) {
  __shared__ Looked<kGatherThreads> s;
  const int head = a.free_state[0], avail = a.free_state[1];
  const int queued0 = queued_first(a, head, avail);
  const int code = free_code(a, s, head, avail);
  if (!code) {
    for (int i = threadIdx.x >> 6; i < a.n; i += kGatherThreads / 64) {
      const int tokens = a.tokens[i], held = tokens > 0 ? page_index(a.pd, tokens - 1) + 1 : 0;
      const int32_t* line = a.table + (held > 0 ? (int64_t)a.lines[i] * a.table_ld : 0);
      for (int j = threadIdx.x & 63; j < held; j += 64) {
        const int id = line[j];
        if (id >= 0 && id < a.num_pages) atomicSub(a.shares + id, 1);
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the counts are down before the barrier (a device fence took 3 us more)
  }
  __syncthreads();
  gather<true>(a, code, head, avail, queued0);
}

// ------------------------------------------------------------------ compact

// The free pages as bits, 32 a word, and how many are free below each word.
struct FreeBits {
  uint32_t bits[kMostPool / 32];
  int below[kMostPool / 32 + 1];
  int sums[16];
  int code;
};

// Free pages with an id below p.
__device__ __forceinline__ int free_below(const FreeBits& s, int p) {
  return (p & 31) ? s.below[p >> 5] + __popc(s.bits[p >> 5] & ((1u << (p & 31)) - 1)) : s.below[p >> 5];
}

// The k-th free page (k from 0; there is one).
__device__ __forceinline__ int nth_free(const FreeBits& s, int k, int words) {
  int lo = 0, hi = words - 1;
  while (lo < hi) {  // the last word with at most k free pages before it
    const int mid = (lo + hi + 1) >> 1;
    if (s.below[mid] <= k)
      lo = mid;
    else
      hi = mid - 1;
  }
  k -= s.below[lo];
  const uint32_t b = s.bits[lo];
  int at = 0;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {  // the lower half holds the k-th bit, or it is that many bits on in the upper
    const int c = __popc(b >> at & ((1u << d) - 1));
    if (k >= c) k -= c, at += d;
  }
  return 32 * lo + at;
}

// The k-th page in use from `limit` on moves to the k-th free page below it. Every
// workgroup reads the free queue into bits of its own, and then maps its share of the
// table, the holders and the queue: one launch, bound by its chain (state, queue, bits,
// sums, search): a pool of 31,000 pages 9.6 us, one of 900 4.9. With the sums by 256
// pages in place of 32, the large one took 15.
constexpr int kCompactThreads = 1024;

__global__ __launch_bounds__(kCompactThreads) void pages_compact(CompactArgs a) {
  constexpr int kAhead = 8;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first = (int64_t)blockIdx.x * kCompactThreads + tid, step = (int64_t)gridDim.x * kCompactThreads;
  __shared__ FreeBits s;
  const int words = (a.num_pages + 31) / 32;
  const int head = a.free_state[0], avail = a.free_state[1];
  // This thread's first page and cell, needed last: asked for now.
  const int held0 = first < a.num_pages ? a.shares[first] : 0, cell0 = first < a.cells ? a.table[first] : 0;
  for (int i = tid; i < words; i += kCompactThreads) s.bits[i] = 0;
  if (tid == 0) s.code = 0;
  __syncthreads();
  bool bad = bad_state(head, avail, a.num_pages);
  if (!bad)
    for (int k0 = tid; k0 < avail; k0 += kAhead * kCompactThreads) {
      int id[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = k0 + i * kCompactThreads;
        id[i] = k < avail ? a.free_pages[queue_at(head, k, a.num_pages)] : -1;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k0 + i * kCompactThreads >= avail) break;
        if (id[i] < 0 || id[i] >= a.num_pages || (atomicOr(&s.bits[id[i] >> 5], 1u << (id[i] & 31)) >> (id[i] & 31) & 1)) bad = true;
      }
    }
  if (bad) s.code = kBad;
  __syncthreads();
  // Free pages before each word: so many words a thread.
  const int per = (words + kCompactThreads - 1) / kCompactThreads, w0 = tid * per, w1 = min(w0 + per, words);
  int sum = 0;
  for (int w = w0; w < w1; ++w) sum += __popc(s.bits[w]);
  int at = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(at, d);
    if (lane >= d) at += u;
  }
  if (lane == 63) s.sums[wave] = at;
  __syncthreads();
  at -= sum;
#pragma unroll
  for (int w = 0; w < kCompactThreads / 64; ++w) at += w < wave ? s.sums[w] : 0;
  for (int w = w0; w < w1; ++w) {
    s.below[w] = at;
    at += __popc(s.bits[w]);
  }
  if (w0 < words && w1 == words) s.below[words] = at;
  __syncthreads();

  const int holes = free_below(s, a.limit);
  const int moves = a.num_pages - a.limit - (avail - holes);  // pages in use from the limit on
  int code = s.code;
  if (!code && moves > a.cap) code = kPages;
  if (!code && moves > holes) code = kExhausted;
  if (first == 0) {
    a.status[0] = code;
    a.status[1] = code ? 0 : moves;
    a.status[2] = code ? 0 : holes - moves;
    a.status[3] = code ? head : 0;
    a.status[4] = avail;
  }
  const auto is_free = [&](int p) { return s.bits[p >> 5] >> (p & 31) & 1; };
  // Where page p, in use, is afterwards.
  const auto moved = [&](int p) { return p < a.limit ? p : nth_free(s, p - a.limit - (free_below(s, p) - holes), words); };
  for (int64_t i = (code ? 0 : moves) + first; i < a.cap; i += step) a.src[i] = a.dst[i] = -1;
  if (code) return;
  for (int64_t i = first; i < a.num_pages; i += step) {
    const int p = (int)i;
    if (is_free(p)) {
      const int k = free_below(s, p);
      a.new_ids[p] = p;
      if (p >= a.limit) {
        a.free_out[holes - moves + (p - a.limit)] = p, a.shares_out[p] = 0;
      } else if (k < moves) {
        a.dst[k] = p;  // its holders come with the page that moves here
      } else {
        a.free_out[k - moves] = p, a.shares_out[p] = 0;
      }
    } else {
      const int to = moved(p);
      a.new_ids[p] = to;
      a.shares_out[to] = i == first ? held0 : a.shares[p];
      if (p >= a.limit) {
        a.src[p - a.limit - (free_below(s, p) - holes)] = p;
        a.free_out[holes - moves + (p - a.limit)] = p, a.shares_out[p] = 0;
      }
    }
  }
  for (int64_t i = avail + first; i < a.num_pages; i += step) a.free_out[i] = -1;
  for (int64_t i = first; i < a.cells; i += step) {
    const int id = i == first ? cell0 : a.table[i];
    a.table_out[i] = id >= a.limit && id < a.num_pages && !is_free(id) ? moved(id) : id;
  }
}

// ------------------------------------------------------------------ copy

// Pages src[k] to dst[k], k below the count, in every layer, and the bytes of their
// scales. A workgroup takes 32 KiB at a time: eight 16-byte loads in flight a thread.
// HBM bounds it, as much written as read: 220 MB 89 us, 4.9 TB/s, as a library's copy of
// 4 GiB; stores past the caches and four or sixteen loads in flight were no faster.
constexpr int kCopyThreads = 256, kCopyAhead = 8, kCopyPart = kCopyThreads * kCopyAhead * 16;

__global__ __launch_bounds__(kCopyThreads) void pages_copy(CopyArgs a) {
  const int n = a.count ? min(max(*a.count, 0), a.n) : a.n;
  const int parts = (int)((a.page_bytes + kCopyPart - 1) / kCopyPart);
  const int64_t items = (int64_t)n * a.layers * parts;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int part = (int)(it % parts);
    const int64_t at = it / parts;
    const int layer = (int)(at % a.layers), k = (int)(at / a.layers);
    const int src = a.src[k], dst = a.dst[k];
    if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages) continue;
    const uint8_t* from = a.kv + layer * a.layer_stride + src * a.page_bytes;
    uint8_t* to = a.kv + layer * a.layer_stride + dst * a.page_bytes;
    const int64_t b0 = (int64_t)part * kCopyPart + threadIdx.x * 16;
    uint4 v[kCopyAhead];
#pragma unroll
    for (int i = 0; i < kCopyAhead; ++i)
      if (b0 + i * (kCopyThreads * 16) < a.page_bytes) v[i] = ldg16_stream(from + b0 + i * (kCopyThreads * 16));
#pragma unroll
    for (int i = 0; i < kCopyAhead; ++i)
      if (b0 + i * (kCopyThreads * 16) < a.page_bytes) *reinterpret_cast<uint4*>(to + b0 + i * (kCopyThreads * 16)) = v[i];
    if (part == 0 && a.kv_scale) {
      uint8_t* s = a.kv_scale + layer * a.scale_layer_stride;
      for (int64_t b = threadIdx.x; b < a.scale_page_bytes; b += kCopyThreads)
        s[dst * a.scale_page_bytes + b] = s[src * a.scale_page_bytes + b];
    }
  }
}

}  // namespace

int launch_pages_fork(const PagesArgs& a, hipStream_t stream) {
  pages_fork<<<dim3((unsigned)std::max(a.n, 1)), kForkThreads, 0, stream>>>(a);
  return check_launch();
}

// Entries (of all lines, at most) that one workgroup takes back by itself.
constexpr int64_t kFewEntries = 4096;

int launch_pages_free(const PagesArgs& a, hipStream_t stream) {
  if ((int64_t)a.n * a.table_ld <= kFewEntries) {
    pages_end<<<1, kGatherThreads, 0, stream>>>(a);
    return check_launch();
  }
  pages_drop<<<dim3((unsigned)std::max(a.n, 1)), kForkThreads, 0, stream>>>(a);
  if (check_launch() != 0) return -3;
  pages_gather<<<1, kGatherThreads, 0, stream>>>(a);
  return check_launch();
}

int launch_pages_compact(const CompactArgs& a, hipStream_t stream) {
  const int64_t most = std::max<int64_t>(std::max<int64_t>(a.num_pages, a.cap), a.cells);
  const int64_t grid = std::min<int64_t>(256, (most + kCompactThreads - 1) / kCompactThreads);
  pages_compact<<<dim3((unsigned)std::max<int64_t>(grid, 1)), kCompactThreads, 0, stream>>>(a);
  return check_launch();
}

int launch_pages_copy(const CopyArgs& a, hipStream_t stream) {
  const int64_t items = (int64_t)a.n * a.layers * ((a.page_bytes + kCopyPart - 1) / kCopyPart);
  pages_copy<<<dim3((unsigned)std::max<int64_t>(1, std::min<int64_t>(items, 4096))), kCopyThreads, 0, stream>>>(a);
  return check_launch();
}

}  // namespace omni
