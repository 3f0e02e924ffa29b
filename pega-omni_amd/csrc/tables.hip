// The row tables of a serving step, built on the GPU from the request lengths
// (gfx950, wave64): positions, cache slots and sequence of every new row, the
// sequences' row and page ranges, their page lists, the pages that the step
// takes from the free queue and those that finished requests give back. What
// the engines' host Rows builder makes (crates/omni-qwen3-tts/src/model.rs:
// 266-303) and uploads row by row, from three numbers a request.
//
// Sequence s with first[s] tokens and count[s] new rows holds ceil(first / page)
// pages, in its table line, and needs ceil((first + count) / page); with a ring,
// of the indices below it. The k-th page that the step takes, in sequence order,
// is entry (head + k) % num_pages of the queue, and the k-th given back goes to
// entry (head + free + k) % num_pages: takes and returns never meet, so every
// workgroup can work out any row's page by itself. All offsets are prefix sums
// over the sequences, which each workgroup computes for itself: one launch, no
// order between workgroups, and the same bits every time.
#include "common.h"
#include "kernels.h"

#include <algorithm>

namespace omni {

namespace {

constexpr int kTabThreads = 256;
constexpr int kTabWaves = kTabThreads / 64;

// What a sequence adds to the step: rows, pages listed, pages taken, pages given back.
struct SeqShare {
  int rows, pages, taken, back, held, line, code;
};

__device__ __forceinline__ int pages_of(const TablesArgs& a, int tokens) {
  const int n = a.ring > 0 ? min(tokens, a.ring) : tokens;
  return n > 0 ? page_index(a.pd, n - 1) + 1 : 0;
}

__device__ __forceinline__ SeqShare seq_share(const TablesArgs& a, int s) {
  SeqShare r{};
  const int first = a.first[s], count = a.count[s];
  r.line = a.lines ? a.lines[s] : s;
  if (first < 0 || (count > 0 && first > 0x7fffffff - count) || r.line < 0 || r.line >= a.num_lines) {
    r.code = 1;
    return r;
  }
  r.held = pages_of(a, first);
  r.rows = max(count, 0);
  r.pages = count < 0 ? 0 : pages_of(a, first + r.rows);
  if (max(r.held, r.pages) > a.table_ld) {
    r.code = 4;
    return r;
  }
  if (a.free_pages) {
    r.taken = count < 0 ? 0 : r.pages - r.held;
    r.back = count < 0 ? r.held : 0;
  } else {
    r.held = r.pages;
  }
  return r;
}

// Inclusive sums over the workgroup's threads, in thread order.
__device__ __forceinline__ int4 scan4(int4 v, int4* wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int4 u = {__shfl_up(v.x, d), __shfl_up(v.y, d), __shfl_up(v.z, d), __shfl_up(v.w, d)};
    if (lane >= d) v = {v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w};
  }
  __syncthreads();
  if (lane == 63) wave_sums[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    const int4 u = wave_sums[w];
    v = {v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w};
  }
  return v;
}

// The first of n ends above x (n where none is).
__device__ __forceinline__ int owner(const int* ends, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__global__ __launch_bounds__(kTabThreads) void step_tables(TablesArgs a) {
  const int tid = threadIdx.x, wg = blockIdx.x;
  const int64_t step = (int64_t)gridDim.x * kTabThreads;
  __shared__ int4 s_wave[kTabWaves];
  __shared__ unsigned long long s_total[4];
  __shared__ unsigned s_codes;  // bit c: code c
  __shared__ int s_rows[kTabThreads], s_pages[kTabThreads], s_taken[kTabThreads], s_back[kTabThreads];
  __shared__ int s_first[kTabThreads], s_held[kTabThreads], s_line[kTabThreads];

  // Totals, in 64 bits, and whether the step can be made at all.
  if (tid < 4) s_total[tid] = 0;
  if (tid == 0) s_codes = 0;
  __syncthreads();
  unsigned long long rows = 0, pages = 0, taken = 0, back = 0;
  unsigned codes = 0;
  for (int s = tid; s < a.nseq; s += kTabThreads) {
    const SeqShare r = seq_share(a, s);
    if (r.code) codes |= 1u << r.code;
    rows += r.rows, pages += r.pages, taken += r.taken, back += r.back;
  }
  // Integer sums: the order of the additions does not change them.
  atomicAdd(&s_total[0], rows);
  atomicAdd(&s_total[1], pages);
  atomicAdd(&s_total[2], taken);
  atomicAdd(&s_total[3], back);
  if (codes) atomicOr(&s_codes, codes);
  __syncthreads();
  rows = s_total[0], pages = s_total[1], taken = s_total[2], back = s_total[3];
  codes = s_codes;
  const int head = a.free_pages ? a.free_state[0] : 0, avail = a.free_pages ? a.free_state[1] : 0;
  if (a.free_pages) {
    if (head < 0 || head >= a.num_pages || avail < 0 || avail > a.num_pages || avail + back > (unsigned)a.num_pages)
      codes |= 1u << 1;
    if (taken > (unsigned)max(avail, 0)) codes |= 1u << 5;
  }
  if (rows > (unsigned)a.row_cap) codes |= 1u << 2;
  if (pages > (unsigned)a.page_cap) codes |= 1u << 3;
  const int code = codes ? __ffs(codes) - 1 : 0;
  if (code) rows = pages = taken = back = 0;  // nothing is built, and the table and the queue stay

  if (wg == 0 && tid == 0) {
    a.status[0] = code;
    a.status[1] = (int)rows;
    a.status[2] = (int)pages;
    a.status[3] = a.free_pages ? code ? head : (int)(((int64_t)head + (int64_t)taken) % a.num_pages) : 0;
    a.status[4] = a.free_pages ? (int)(avail - (int64_t)taken + (int64_t)back) : 0;
    a.row_indptr[0] = 0;
    a.indptr[0] = 0;
  }
  for (int64_t r = (int64_t)rows + (int64_t)wg * kTabThreads + tid; r < a.row_cap; r += step)
    a.pos[r] = a.slots[r] = a.seq[r] = -1;
  if (code) {
    for (int64_t s = (int64_t)wg * kTabThreads + tid; s < a.nseq; s += step) a.row_indptr[s + 1] = a.indptr[s + 1] = 0;
    return;
  }

  const auto queue = [&](int64_t k) { return (int)((head + k) % a.num_pages); };
  int4 base{};  // rows, pages, taken and given back before these sequences
  for (int s0 = 0; s0 < a.nseq; s0 += kTabThreads) {
    const int n = min(kTabThreads, a.nseq - s0);
    SeqShare r{};
    if (tid < n) r = seq_share(a, s0 + tid);
    const int4 in = {r.rows, r.pages, r.taken, r.back};
    int4 end = scan4(in, s_wave);
    end = {base.x + end.x, base.y + end.y, base.z + end.z, base.w + end.w};
    s_rows[tid] = end.x, s_pages[tid] = end.y, s_taken[tid] = end.z, s_back[tid] = end.w;
    if (tid < n) {
      s_first[tid] = a.first[s0 + tid], s_held[tid] = r.held, s_line[tid] = r.line;
      if (wg == 0) a.row_indptr[s0 + tid + 1] = end.x, a.indptr[s0 + tid + 1] = end.y;
    }
    __syncthreads();
    const int4 top = {s_rows[n - 1], s_pages[n - 1], s_taken[n - 1], s_back[n - 1]};
    const auto before = [&](const int* ends, int i, int b) { return i > 0 ? ends[i - 1] : b; };
    const auto page_of = [&](int i, int j) {  // page j of sequence s0 + i
      return j < s_held[i] ? a.table[(int64_t)s_line[i] * a.table_ld + j]
                           : a.free_pages[queue((int64_t)before(s_taken, i, base.z) + j - s_held[i])];
    };
    // This workgroup's share of a range that goes on from `from`: every index x with x / 256 % gridDim.x == wg.
    const auto first_at = [&](int from) {
      const int64_t mine = (int64_t)wg * kTabThreads + tid;
      return from <= mine ? mine : mine + (from - mine + step - 1) / step * step;
    };
    for (int64_t x = first_at(base.x); x < top.x; x += step) {
      const int i = owner(s_rows, n, (int)x), p = s_first[i] + (int)x - before(s_rows, i, base.x);
      const int q = a.ring > 0 ? p % a.ring : p, j = page_index(a.pd, q);
      a.pos[x] = p;
      a.slots[x] = (int)page_slot(a.pd, page_of(i, j), q);
      a.seq[x] = s0 + i;
    }
    for (int64_t x = first_at(base.y); x < top.y; x += step) {
      const int i = owner(s_pages, n, (int)x);
      a.pages[x] = page_of(i, (int)x - before(s_pages, i, base.y));
    }
    for (int64_t x = first_at(base.z); x < top.z; x += step) {
      const int i = owner(s_taken, n, (int)x);
      a.table[(int64_t)s_line[i] * a.table_ld + s_held[i] + (int)x - before(s_taken, i, base.z)] = a.free_pages[queue(x)];
    }
    for (int64_t x = first_at(base.w); x < top.w; x += step) {
      const int i = owner(s_back, n, (int)x);
      a.free_pages[queue((int64_t)avail + x)] = a.table[(int64_t)s_line[i] * a.table_ld + (int)x - before(s_back, i, base.w)];
    }
    base = top;
    __syncthreads();
  }
}

}  // namespace

int launch_tables(const TablesArgs& a, hipStream_t stream) {
  const int most = std::max(std::max(a.row_cap, a.page_cap), a.nseq);
  const int grid = std::max(1, std::min(1024, (int)(((int64_t)most + kTabThreads - 1) / kTabThreads)));
  step_tables<<<grid, kTabThreads, 0, stream>>>(a);
  return check_launch();
}

}  // namespace omni
