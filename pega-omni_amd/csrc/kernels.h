// Launch interface between the C ABI (capi.cpp) and the HIP kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "indexing.h"

namespace omni {

typedef uint16_t bf16_t;

// The HIP status of this thread's last launch, kept for error messages.
inline thread_local hipError_t g_launch_status = hipSuccess;
inline int check_launch() {
  g_launch_status = hipGetLastError();
  return g_launch_status == hipSuccess ? 0 : -3;
}

// What a launch holds: fewer than 2^32 threads in x, at most 65,535 workgroups in y and z.
constexpr int64_t kMostGridThreads = (1LL << 32) - 1;
constexpr int kMostGridYZ = 65535;
inline bool grid_holds(int64_t x, int threads, int64_t y = 1) {
  return x * threads <= kMostGridThreads && y <= kMostGridYZ;
}

// Everything a decode launch reads; passed by value as the kernel argument.
struct DecodeArgs {
  const bf16_t* qkv;
  int64_t q_stride;  // elements between consecutive qkv rows
  const bf16_t* kv;
  const int32_t* pos;  // len_mode 0: per-row positions; 1: per-sequence last page lengths
  const int32_t* seq;
  const int32_t* indptr;
  const int32_t* pages;
  bf16_t* out;
  float* ws_o;   // [rows][hq][splits][128] split outputs (normalised)
  float* ws_lse; // [rows][hq][splits] split log2-sum-exp
  int hq, hk;
  int ragged;
  PageDiv pd;   // page size and its divisor
  int context;  // cap on keys per row
  int len_mode;
  int chunk, splits;
  float scale_log2;  // softmax scale times log2(e)
  int fp8;           // 1: kv slots are FP8 E4M3 with f32 scales (lm_attend's cache)
  int64_t slot_bytes;  // bytes per FP8 slot: 2 hk 128 + 2 hk 4
  int group_heads;     // K/V heads per workgroup of the head-group kernels (0 = pick from the shape)
  int dense_per, dense_base, dense_span;  // dense rows (len_mode 2): slot (n / per) * span + t
  // Fused rotary (rope != 0, decode rows only): q and the row's own key are
  // rotated in the kernel (Qwen3: normalised first; FP8 ring: K and V
  // quantized), and the split holding the row's new key writes it into slot
  // slots[n] of kv_w (the cache kv points to) and takes it from registers.
  int rope;
  const bf16_t* q_norm;
  const bf16_t* k_norm;
  const int32_t* slots;
  bf16_t* kv_w;
  float eps, theta;
  float coef;  // FP8 ring (lm_rope): pair i turns by p * exp(i * coef)
};

int launch_decode(const DecodeArgs& a, int rows, hipStream_t stream);

// The allocation-free decode entry point's split-partial workspace: a
// file-scope device array of this many bytes per GPU.
constexpr int64_t kNoAllocScratchBytes = 16LL << 20;
constexpr int kMaxDevices = 64;
// Device address of that array on the current device (looked up once per
// device); 0 on success, -1 if the lookup fails.
int noalloc_scratch(float** ptr);

// Copy of whole cache slots (prefix K/V reuse): slot dst[r] takes slot src[r].
int launch_copy_slots(void* kv, const int32_t* src, const int32_t* dst, int tokens, int slot_bytes,
                      hipStream_t stream);

int launch_gather_kv(const void* kv, int hk, const int32_t* indptr, const int32_t* pages, PageDiv pd,
                     const int32_t* seq_ids, const int32_t* lens, const int32_t* out_indptr, int nseq, void* out,
                     hipStream_t stream);

// Tiled MFMA attention (prefill and DiT).
struct TiledArgs {
  const bf16_t* q;
  int64_t q_stride;  // elements between query rows
  // paged source (mode 0): kv slots [2 hk][128]
  const bf16_t* kv;
  const int32_t* pos;
  const int32_t* seq;
  const int32_t* indptr;
  const int32_t* pages;
  const int32_t* work;  // 4 int32 per tile: seq, first row, rows, unused
  PageDiv pd;
  // dense source (mode 1): k, v [slots][hk][128]
  const bf16_t* k;
  const bf16_t* v;
  const int32_t* kv_len_at;
  int q_len;
  int causal;
  int64_t q_bstride, kv_bstride, out_bstride;
  bf16_t* out;
  int hq, hk;
  float scale_log2;  // any finite value
  uint32_t q_sign;   // set by the launch: flips the signs of two bf16 of Q where the scale is negative
  // Tail split (dense, uniform key ranges): items >= split_from run as
  // split_k key chunks each, writing f32 partials to ws (one segment per
  // chunk: O[kTiledRows][128] then (m, l)[kTiledRows]); 0 chunks = no split.
  int split_from, split_k;
  float* ws;
  // Row halves (no split): the last `halved` items (prefill: all or none) run
  // as two workgroups of kTiledRows / 2 packed rows each; 0 = none.
  int halved;
  // All items run as four workgroups of a quarter of the rows each (no split).
  int quarters;
  // All but DiT: P carried as two bf16 terms (hi + lo) through P.V.
  int exact_p;
  // packed prompts (mode 2), cross attention: elements between rows of k and of v
  int64_t k_stride, v_stride;
  // Several rows per sequence: an item is (sequence, first row, rows, kv head, split,
  // splits, segment of ws, split tile); splits are of split_tiles key tiles, and of a
  // split tile's, how many it used goes to `used`.
  const uint8_t* kv8;       // the 8-bit cache (pd: blocks per page)
  const uint8_t* kv_scale;
  const int32_t* of;        // cross: the source of each sequence (null: the sequence)
  const int32_t* first;     // and its first row and rows
  const int32_t* len;
  int split_tiles;
  int splits_listed;          // (tile, kv head) pairs that are split
  int64_t segments;           // their splits
  const int32_t* split_items; // (first row, rows + 2^9 splits, kv head, first segment) of each
  int32_t* used;
};
constexpr int kMultiItem = 8;  // int32 per item
// Query heads of a K/V head that such tiles are built for.
constexpr bool multi_tiles_hold(int G) { return (G >= 1 && G <= 8) || G == 16; }

// Packed (position, head) query rows per MFMA tile: one 8-wave workgroup, one per CU.
constexpr int kTiledRows = 256;
// Bytes of one partial segment of the tail split: O (f32) and (m, l) per packed row.
constexpr int kTiledThreads = kTiledRows * 2;  // a wave for each 32 rows
constexpr int64_t kSegmentBytes = (int64_t)kTiledRows * (128 + 2) * 4;

// Prefill work list: a header of kPrefillWorkHeader int32 (entries 0..8: the
// item ranges of the 8 XCDs, range x = [h[x], h[x + 1])) then 4 int32 per
// (tile, kv head) item: sequence, first row, rows, kv head.
constexpr int kPrefillWorkHeader = 16;
constexpr int kXcds = 8;
int launch_prefill(const TiledArgs& a, int items, hipStream_t stream);
// Packed prompts: items are (sequence's first row, first row, rows, kv head).
constexpr int64_t kMostPromptStride = 1LL << 22;  // elements: 128 rows stay below 2^30 bytes
int launch_prompt(const TiledArgs& a, int items, hipStream_t stream);
// Several rows per sequence over a source of launch_rows: items of kMultiItem fields, as TiledArgs has them.
int launch_multi_tiles(const TiledArgs& a, int source, int items, hipStream_t stream);

// Rotary embedding + K/V scatter (the step before attention).
struct RopeArgs {
  bf16_t* qkv;
  int64_t ld;  // elements between qkv rows
  const bf16_t* q_norm;
  const bf16_t* k_norm;
  const int32_t* pos;    // [rows], or [rows][3] (t, h, w) for M-RoPE
  const int32_t* slots;  // [rows] cache slot of each row
  bf16_t* kv;            // bf16 slots [2 hk][128]
  void* kv_bytes;        // FP8 slots of slot_bytes
  int64_t slot_bytes;
  bf16_t* k_cache;  // M-RoPE: separate caches [slots][hk][128]
  bf16_t* v_cache;
  int rows, hq, hk;
  int per, base, span;  // dense rows: seq n / per at position base + n % per, slot seq * span + pos
  int mrope_hw;
  float eps, theta, coef;
};
// Head-64 ring attentions (Mimi, Qwen3-TTS codec, depformer).
struct ShortArgs {
  const bf16_t* qkv;
  const int32_t* pos;
  const int32_t* lines;  // session -> line of the per-session state
  void* state;           // Mimi / codec rings: state + lines[s] * stride bytes
  int64_t stride;
  bf16_t* ws;            // depformer workspace [seqs][8][K | V][heads * 64]
  bf16_t* out;
  bf16_t* qkv_rw;        // Mimi rotary: the qkv rows, q turned in place
  int rows, heads, T, context, step;
  float scale, theta;
  float coef;            // Mimi rotary: pair i turns by p * exp(i * coef)
};
constexpr int kShortMimi = 0, kShortCodec = 1, kShortDep = 2, kShortMimiRope = 3;
int launch_short(const ShortArgs& a, int kind, hipStream_t stream);

constexpr int kRopeQwen3 = 0, kRopeQwen3Dense = 1, kRopeHidream = 2, kRopeLm = 3;
int launch_rope(const RopeArgs& a, int mode, hipStream_t stream);
int launch_dit(const TiledArgs& a, int batch, hipStream_t stream);
// Items and the tail split launch_dit would use for a call (split_k = 0: none).
void dit_split(const TiledArgs& a, int batch, int resident, int* items, int* split_from, int* split_k);
// Whether a call of `items` tiles should run them as row quarters, and the
// items launch_prefill should run as row halves otherwise (all or none).
bool tiled_quarters(long long items, int resident);
int prefill_halves(long long items, int resident);
// Items launch_dit should run as row halves when no split is used (0: none).
int dit_halves(const TiledArgs& a, int batch, int resident);

// Row tables of a step, built on the GPU (tables.hip).
struct TablesArgs {
  const int32_t* first;  // [nseq] positions in the cache before the step
  const int32_t* count;  // [nseq] new rows; negative: the request is done
  const int32_t* lines;  // [nseq] table line of each sequence, or null (line s)
  int nseq;
  PageDiv pd;
  int ring;  // > 0: position p lives at index p % ring
  int32_t* table;  // [num_lines][table_ld] page ids
  int64_t table_ld;
  int num_lines;
  int32_t* free_pages;  // queue of num_pages entries, or null: every page is in the table
  int num_pages;
  const int32_t* free_state;  // {first free entry, free entries}
  int row_cap, page_cap;
  int32_t *pos, *slots, *seq;   // [row_cap]
  int32_t *row_indptr, *indptr; // [nseq + 1]
  int32_t* pages;               // [page_cap]
  int32_t* status;              // {code, rows, pages, first free entry, free entries}
};
int launch_tables(const TablesArgs& a, hipStream_t stream);

// Pages of a cache (pages.hip): forked, given back, compacted, copied.
constexpr int kMostLines = 1 << 18;  // of a table: a bit each in LDS
constexpr int kMostPool = 1 << 19;   // pages of a pool that is compacted: likewise, and a sum for 32

struct PagesArgs {
  const int32_t* parents;  // fork: [n] table lines
  const int32_t* lines;    // [n] the children, or the lines that end
  const int32_t* tokens;   // [n]; negative: nothing to do
  int n;
  PageDiv pd;
  const int32_t* table;  // [num_lines][table_ld]
  int32_t* table_out;    // the same
  int64_t table_ld;
  int num_lines;
  int32_t* free_pages;
  int num_pages;
  const int32_t* free_state;
  int32_t* shares;       // [num_pages] lines that hold a page beside the first
  int32_t *src, *dst;    // fork: [n] pages to copy
  int32_t* status;       // {code, pages taken or given back, pages shared or dropped, first free entry, free entries}
};
int launch_pages_fork(const PagesArgs& a, hipStream_t stream);
int launch_pages_free(const PagesArgs& a, hipStream_t stream);

struct CompactArgs {
  const int32_t* table;
  int32_t* table_out;  // may be the table
  int64_t cells;       // of the table
  const int32_t* free_pages;
  int32_t* free_out;
  int num_pages, limit;
  const int32_t* free_state;
  const int32_t* shares;
  int32_t* shares_out;
  int32_t* new_ids;  // [num_pages]
  int32_t *src, *dst;
  int cap;  // entries of src and dst
  int32_t* status;
};
int launch_pages_compact(const CompactArgs& a, hipStream_t stream);

struct CopyArgs {
  uint8_t* kv;
  int64_t page_bytes, layer_stride;  // multiples of 16
  uint8_t* kv_scale;                 // may be null
  int64_t scale_page_bytes, scale_layer_stride;
  int layers, num_pages;
  const int32_t *src, *dst;  // pairs with a page outside the pool are none
  int n;
  const int32_t* count;  // pairs that count, or null: n
};
int launch_pages_copy(const CopyArgs& a, hipStream_t stream);

// The 8-bit block cache (q8.hip): blocks of 16 tokens, [2 hk heads][2048]
// bytes (K heads [16 tokens][128 dims], V heads [128 dims][16 tokens]) and one
// biased power-of-two exponent per (block, head).
constexpr int kQ8Block = 16;
constexpr int kQ8HeadBytes = kQ8Block * 128;
constexpr int kQ8E4m3 = 0, kQ8Int8 = 1;

struct RopeQ8Args {
  const bf16_t* qkv;
  int64_t ld;
  const bf16_t* q_norm;
  const bf16_t* k_norm;
  const int32_t* pos;
  const int32_t* slots;  // negative: the row is skipped
  bf16_t* q;
  int64_t q_ld;
  bf16_t* k;  // may be null
  int64_t k_ld;
  uint8_t* kv;
  uint8_t* kv_scale;
  int format;
  int rows, hq, hk;
  float eps;
  double inv_theta64;  // theta^(-1/64): pair i turns by pos * inv_theta64^i
};
int launch_rope_q8(const RopeQ8Args& a, hipStream_t stream);  // -2: more rows or heads than a grid holds, nothing launched

struct DecodeQ8Args {
  const bf16_t* q;
  int64_t q_stride;
  const uint8_t* kv;
  const uint8_t* kv_scale;
  const int32_t* pos;  // negative: the row stores zeros
  const int32_t* seq;
  const int32_t* indptr;
  const int32_t* pages;
  bf16_t* out;
  float* ws_o;    // [rows][hq][splits][128]
  float* ws_lse;  // [rows][hq][splits]
  int format;
  int hq, hk;
  int ragged;
  PageDiv pd;  // blocks per page
  int chunk, splits;
  int per_round;   // rows whose workgroups fill the GPU once; 0: rows in their order
  int len_shift;   // row lengths >> len_shift fit 6 bits (longer ones count as 63)
  float scale_log2;
};
constexpr int kQ8Threads = 256;  // of every workgroup of the 8-bit cache's kernels
// Whether decode's grid and (of splits) the merge's hold a call.
inline bool decode_q8_fits(int rows, int hq, int splits) {
  return grid_holds(splits, kQ8Threads) && (splits == 1 || grid_holds((int64_t)rows * hq, kQ8Threads));
}
int launch_decode_q8(DecodeQ8Args a, int rows, hipStream_t stream);

// Groups of rows that see the same keys (rows.hip): an item is (sequence, first row,
// rows, its first row in the workspace).
constexpr int kRowsThreads = 256;
// (row, head) pairs that a workgroup of rows_merge takes: with many splits its four waves
// share them.
constexpr int kRowsMergeMany = 32;
constexpr int rows_merged(int splits) { return splits > kRowsMergeMany ? 2 : 8; }
constexpr int kRowsBf16 = 2;  // source: bf16 rows, beside kQ8E4m3 and kQ8Int8

struct RowsArgs {
  const bf16_t* q;
  int64_t q_stride;
  // the 8-bit cache
  const uint8_t* kv;
  const uint8_t* kv_scale;
  const int32_t* pos;  // negative: the row stores zeros
  const int32_t* indptr;
  const int32_t* pages;
  PageDiv pd;  // blocks per page
  // bf16 sources: rows first[e] .. + len[e] - 1 of k and v, e = of[sequence] (null: the sequence)
  const bf16_t* k;
  const bf16_t* v;
  int64_t k_stride, v_stride;
  const int32_t* of;
  const int32_t* first;
  const int32_t* len;
  bf16_t* out;
  const int32_t* items;
  float* ws_o;       // [workspace rows][hq][splits][128]
  float* ws_lse;     // [workspace rows][hq][splits]
  int32_t* ws_used;  // splits that each group takes
  int hq, hk;
  int g16;  // set by the launch: divides a packed column by hq / hk
  int chunk, splits;
  float scale_log2;
};
// groups: of at most 16, and of at most 32 packed rows; their items one list behind the other.
int launch_rows(const RowsArgs& a, int source, const int* groups, hipStream_t stream);

}  // namespace omni
