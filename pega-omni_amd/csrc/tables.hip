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
  // More rows than a ring holds would give several of them one slot.
  if (first < 0 || (count > 0 && first > 0x7fffffff - count) || (a.ring > 0 && count > a.ring) || r.line < 0 ||
      r.line >= a.num_lines) {
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

// Sums of counts in 0 .. 2^31 - 1 that stop at 2^31 - 1 (still associative), so a
// total past int32 shows as one past every capacity.
__device__ __forceinline__ int add_sat(int x, int y) { return (int)min((uint32_t)x + (uint32_t)y, 0x7fffffffu); }
__device__ __forceinline__ int4 add_sat(int4 x, int4 y) {
  return {add_sat(x.x, y.x), add_sat(x.y, y.y), add_sat(x.z, y.z), add_sat(x.w, y.w)};
}

// Inclusive sums over the workgroup's threads, in thread order.
__device__ __forceinline__ int4 scan4(int4 v, int4* wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int4 u = {__shfl_up(v.x, d), __shfl_up(v.y, d), __shfl_up(v.z, d), __shfl_up(v.w, d)};
    if (lane >= d) v = add_sat(v, u);
  }
  if (lane == 63) wave_sums[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v = add_sat(v, wave_sums[w]);
  return v;
}

// Every workgroup: the sums over all sequences (one scan of as many sequences as
// threads gives totals and offsets; more sequences are added up first), then its
// share of each output, a row or page finding its sequence by bisection of the sums
// in LDS. Bytes bound nothing here (40 KB for 64 sequences of some 1500 tokens, a
// microsecond's worth for the largest steps): two memory round trips, the lengths
// and a page id, and the launch are what a call takes, 5.3 us for 64 sequences of
// one new token and 6.9 for 128, 24 of them prompts of 30-4096 (with 64-bit sums and a
// second pass over the sequences 14.6).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void step_tables(TablesArgs a) {
  constexpr int kWaves = THREADS / 64;
  const int tid = threadIdx.x, wg = blockIdx.x, first_x = wg * THREADS + tid, step = gridDim.x * THREADS;
  __shared__ int4 s_wave[kWaves];
  __shared__ int s_codes[kWaves];
  __shared__ int4 s_end[THREADS];            // rows, pages, taken and given back up to a sequence
  __shared__ int s_first[THREADS], s_held[THREADS];
  __shared__ int64_t s_line[THREADS];        // the sequence's line in the table

  const int head = a.free_pages ? a.free_state[0] : 0, avail = a.free_pages ? a.free_state[1] : 0;
  int codes = 0;  // bit c: code c
  if (a.free_pages && (head < 0 || head >= a.num_pages || avail < 0 || avail > a.num_pages)) codes |= 1 << 1;

  // Totals, and whether the step can be made at all.
  const bool one_scan = a.nseq <= THREADS;
  SeqShare r{};
  int4 sum{};
  for (int s = tid; s < a.nseq; s += THREADS) {
    r = seq_share(a, s);
    if (r.code) codes |= 1 << r.code;
    sum = add_sat(sum, int4{r.rows, r.pages, r.taken, r.back});
  }
  int4 end = scan4(sum, s_wave);
  s_end[tid] = end;
  for (int c = 1; c <= 5; ++c)
    if (__any(codes >> c & 1)) codes |= 1 << c;
  if ((tid & 63) == 0) s_codes[tid >> 6] = codes;
  __syncthreads();
  int4 total = s_end[THREADS - 1];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) codes |= s_codes[w];
  if (a.free_pages) {
    if (add_sat(max(avail, 0), total.w) > a.num_pages) codes |= 1 << 1;
    if (total.z > avail) codes |= 1 << 5;
  }
  if (total.x > a.row_cap) codes |= 1 << 2;
  if (total.y > a.page_cap) codes |= 1 << 3;
  const int code = codes ? __ffs(codes) - 1 : 0;
  if (code) total = int4{0, 0, 0, 0};  // nothing is built, and the table and the queue stay

  // Entry `head + k` of the queue, 0 <= k <= num_pages.
  const auto queue = [&](int k) {
    const uint32_t i = (uint32_t)head + (uint32_t)k;
    return i >= (uint32_t)a.num_pages ? i - (uint32_t)a.num_pages : i;
  };
  if (first_x == 0) {
    a.status[0] = code;
    a.status[1] = total.x;
    a.status[2] = total.y;
    a.status[3] = !a.free_pages ? 0 : code ? head : (int)queue(total.z);
    a.status[4] = !a.free_pages ? 0 : avail - total.z + total.w;
    a.row_indptr[0] = 0;
    a.indptr[0] = 0;
  }
  for (int64_t x = (int64_t)total.x + first_x; x < a.row_cap; x += step) a.pos[x] = a.slots[x] = a.seq[x] = -1;
  if (code) {
    for (int64_t s = first_x; s < a.nseq; s += step) a.row_indptr[s + 1] = a.indptr[s + 1] = 0;
    return;
  }

  int4 base{};  // the sums before the sequences at hand
  for (int s0 = 0; s0 < a.nseq; s0 += THREADS) {
    const int n = min(THREADS, a.nseq - s0);
    if (!one_scan) {
      __syncthreads();  // the last sequences' sums have been read
      r = SeqShare{};
      if (tid < n) r = seq_share(a, s0 + tid);
      end = add_sat(base, scan4(int4{r.rows, r.pages, r.taken, r.back}, s_wave));
      s_end[tid] = end;
    }
    if (tid < n) {
      s_first[tid] = a.first[s0 + tid], s_held[tid] = r.held, s_line[tid] = r.line * a.table_ld;
      if (wg == 0) a.row_indptr[s0 + tid + 1] = end.x, a.indptr[s0 + tid + 1] = end.y;
    }
    __syncthreads();
    const int4 top = s_end[n - 1];
    const auto before = [&](int i) { return i > 0 ? s_end[i - 1] : base; };
    // The sequence (of those at hand) whose range holds x; `of` picks the sum.
    const auto owner = [&](int x, auto of) {
      int lo = 0, hi = n;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (of(s_end[mid]) > x)
          hi = mid;
        else
          lo = mid + 1;
      }
      return lo;
    };
    const auto page_of = [&](int i, int j) {  // page j of sequence s0 + i
      return j < s_held[i] ? a.table[s_line[i] + j] : a.free_pages[queue(before(i).z + j - s_held[i])];
    };
    for (int64_t x = (int64_t)base.x + first_x; x < top.x; x += step) {
      const int i = owner((int)x, [](int4 v) { return v.x; }), p = s_first[i] + (int)x - before(i).x;
      const int q = a.ring > 0 ? p % a.ring : p, j = page_index(a.pd, q);
      const int id = page_of(i, j);
      a.pos[x] = p;
      a.seq[x] = s0 + i;
      a.slots[x] = (int)page_slot(a.pd, id, q);
    }
    for (int64_t x = (int64_t)base.y + first_x; x < top.y; x += step) {
      const int i = owner((int)x, [](int4 v) { return v.y; });
      a.pages[x] = page_of(i, (int)x - before(i).y);
    }
    for (int64_t x = (int64_t)base.z + first_x; x < top.z; x += step) {
      const int i = owner((int)x, [](int4 v) { return v.z; });
      a.table[s_line[i] + s_held[i] + (int)x - before(i).z] = a.free_pages[queue((int)x)];
    }
    for (int64_t x = (int64_t)base.w + first_x; x < top.w; x += step) {
      const int i = owner((int)x, [](int4 v) { return v.w; });
      a.free_pages[queue(avail + (int)x)] = a.table[s_line[i] + (int)x - before(i).w];
    }
    base = top;
  }
}

}  // namespace

// As many threads as sequences, to 1024: one scan gives every offset. us in 256 / 512 /
// 1024 threads: 286 sequences 11.6 / 7.7 / 8.6, 512 12.6 / 8.2 / 9.0, 1024 21.5 / 14.7 /
// 10.0, 4090 74 / 46 / 32.
int launch_tables(const TablesArgs& a, hipStream_t stream) {
  const int most = std::max(std::max(a.row_cap, a.page_cap), a.nseq);
  const auto grid = [&](int threads) { return (int)std::max<int64_t>(1, std::min<int64_t>(1 << 18, (int64_t)most + threads - 1) / threads); };
  if (a.nseq <= 256)
    step_tables<256><<<grid(256), 256, 0, stream>>>(a);
  else if (a.nseq <= 512)
    step_tables<512><<<grid(512), 512, 0, stream>>>(a);
  else
    step_tables<1024><<<grid(1024), 1024, 0, stream>>>(a);
  return check_launch();
}

}  // namespace omni
