// Attention of a few rows that see the same keys (gfx950, wave64): several new rows
// of a sequence over the 8-bit block cache, or rows over an encoder's bf16 states.
// What a row sees is its own affair (keys 0..pos, or all of a source), but the keys
// are read once for all rows of a group.
//
// A group is at most 16 NC packed (row, head) columns of one K/V head: R = 16 NC / G
// rows. One workgroup per (group, K/V head, split of the keys); its waves take the
// split's 32-key tiles in turn, each with running maxima, sums and O of its own, and
// the four are merged through LDS at the end. Lane l is column n = l % 16 of a block
// of 16 columns, and group g = l / 16 of v_mfma_f32_16x16x32_bf16's operands:
//   S^T (16 keys x 16 columns), two of them: row 4 x + r of product j is key
//     8 x + 4 j + r of the tile, so that a lane ends with keys 8 g .. 8 g + 7 for its
//     column, in order, which is P^T's operand as it stands.
//   O^T (16 dims x 16 columns) += V^T . P^T. The cache holds V as [dim][token]; bf16
//     rows of V pass through the wave's own 8 KiB of LDS, from which transposing
//     reads take eight keys of a dim.
// K and V operands are made once a tile and serve NC columns blocks. P is carried as
// two bf16 terms (hi + lo, 16 bits) and is at most 1 on the way: the running base
// stands 8 (log2) above the maximum that moved it. What a row's later keys hold does
// not reach it: their scores go, and as 0 times a NaN of V is NaN, those count as 0 in
// the tiles that not all rows see whole, and come back in the end for the rows that see
// them (up to 0.25 us where most tiles are such: 41 groups of 32 over 137-785 keys, 9.3 us).
//
// The keys' bytes bound it where groups are many: 64 sequences of 4 rows over 200-2400
// tokens of 16q/8kv, E4M3, 31.0 us, 5.5 TB/s (a row per workgroup, each reading the keys
// again: 70); 48 sources of 100-1500 bf16 rows, 5 rows each, 31.3 us, 5.1 TB/s. A group
// alone is bound by its chain (rows, page ids, exponents, K, V, the waves' exchange): 5
// rows over 2400 tokens 6.8 us and 3.7 of merge. 16 columns a workgroup because that is
// the product's width; a second block of 16 costs 14 % more time a tile, registers then
// allowing two workgroups a CU in place of four. Two groups of 32 in place of a tile for
// 33 to 64 packed rows, and eight waves a group in place of four, were no faster.
#include "common.h"
#include "kernels.h"
#include "q8_bytes.h"
#include "rotary.h"

#include <algorithm>

namespace omni {

namespace {

constexpr int kThreads = kRowsThreads, kWaves = kThreads / 64;
constexpr int kTile = 32;  // keys per step: two blocks of the cache
constexpr int kBlocksPerTile = kTile / kQ8Block;
constexpr int kIds = 64 / kBlocksPerTile;  // tiles whose blocks a wave looks up at once
constexpr int kBf16 = 2;                   // beside kQ8E4m3 and kQ8Int8

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// ds_read_b64_tr_b16: within each 16 lanes, lane i receives element i % 4 of the
// 8-byte chunks that lanes 4 e + i / 4 address, e = 0..3.
__device__ __forceinline__ bf16x4 lds_read_tr(const bf16_t* p) {
  typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p));
}

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
constexpr int kBufferFlags = 0x00020000;  // resource word 3 of raw buffer loads

// A raw buffer over a wave-uniform base, `bytes` long: what lies past that is read as zeros.
__device__ __forceinline__ i32x4 buffer_rsrc(const void* base, int bytes) {
  const uint64_t b = (uint64_t)base;
  return i32x4{__builtin_amdgcn_readfirstlane((int)b), __builtin_amdgcn_readfirstlane((int)(b >> 32)),
               __builtin_amdgcn_readfirstlane(bytes), kBufferFlags};
}
// Sixteen bytes at offset off of a buffer, read once: nontemporal (bit 1 of the last operand).
__device__ __forceinline__ uint4 ldb16_stream(i32x4 rsrc, int off) {
  const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)(uint32_t)rsrc[0] | (uint64_t)(uint32_t)rsrc[1] << 32), 0, rsrc[2], rsrc[3]);
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 2));
}
// The same to LDS, lane l's to lds + 16 l (lds wave-uniform). The compiler does not
// see these loads, nor M0's and the resource's hazards: s_nop 4 covers those, and
// the wave waits for the loads by itself.
__device__ __forceinline__ void dma16_stream(i32x4 rsrc, int off, const void* lds) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds"
               :
               : "v"(off), "s"(rsrc), "{m0}"((uint32_t)(uintptr_t)(lds_void*)lds)
               : "memory");
}

// The larger of v over the 16 lanes of a DPP row.
template <int CTRL>
__device__ __forceinline__ int dpp_max(int v) {
  return max(v, __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ int row16_max(int v) {
  return dpp_max<kRowMirror>(dpp_max<kRowHalfMirror>(dpp_max<kQuadSwap2>(dpp_max<kQuadSwap1>(v))));
}

// c / G for packed columns: 0 <= c < 32, 1 <= G <= 16 (g16 = 65536 / G + 1).
__device__ __forceinline__ int row_of_column(int c, int g16) { return c * g16 >> 16; }

// v, so that what follows from it is worked out here and not held in registers through a loop.
__device__ __forceinline__ int here(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Waves per SIMD that a kernel's registers (bf16: its LDS) leave room for.
constexpr int room(int src, int nc) { return nc == 2 || src == kBf16 ? 2 : 4; }

template <int SRC, int NC>
__global__ __launch_bounds__(kThreads, room(SRC, NC)) void rows_attn(RowsArgs a) {
  constexpr bool Q8 = SRC != kBf16;
  constexpr int FMT = Q8 ? SRC : kQ8E4m3;
  const int slot = blockIdx.x % a.splits, unit = blockIdx.x / a.splits;
  const int kh = unit % a.hk, group = unit / a.hk, split = spread_split(slot, unit, a.splits);
  const int4 item = reinterpret_cast<const int4*>(a.items)[group];  // sequence, first row, rows, row of the workspace
  const int G = a.hq / a.hk, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
  const int nrows = item.z;

  // Columns: row c / G of the group, head c % G. Keys that each sees; a column that is none sees what the last does.
  int64_t src0 = 0;  // bf16: the source's first row
  int src_len = 0;
  const int32_t* pg = nullptr;
  if constexpr (Q8) {
    pg = a.pages + a.indptr[item.x];
  } else {
    const int e = a.of ? a.of[item.x] : item.x;
    src0 = a.first[e], src_len = max(a.len[e], 0);
  }
  int lim[NC], most = 0, not_least = -INT_MAX;
  bf16x8 q[NC][4];  // product step kk holds dims 64 (kk / 2) + 16 g + 8 (kk % 2) .. + 7
#pragma unroll
  for (int b = 0; b < NC; ++b) {
    const int c = 16 * b + col, i = row_of_column(c, a.g16);
    const bool mine = i < nrows;
    lim[b] = -1;
    if (mine) {
      lim[b] = Q8 ? max(a.pos[item.y + i], -1) + 1 : src_len;
      most = max(most, lim[b]), not_least = max(not_least, -lim[b]);
    }
    const bf16_t* qp = a.q + (int64_t)(item.y + (mine ? i : 0)) * a.q_stride + (int64_t)(kh * G + c - i * G) * kHead;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      q[b][kk] = __builtin_bit_cast(bf16x8, ldg16(qp + 64 * (kk >> 1) + 16 * grp + 8 * (kk & 1)));
  }
  most = __builtin_amdgcn_readfirstlane(row16_max(most));
  const int least = -__builtin_amdgcn_readfirstlane(row16_max(not_least));

  const int split_len = most > 0 ? split_len_of(a.chunk, a.splits, most) : 0;
  const int used = most > 0 ? (most - 1) / split_len + 1 : 0;
  if (a.splits > 1 && split == 0 && kh == 0 && tid == 0) a.ws_used[group] = used;
  const int packed = nrows * G;
  if (used == 0) {
    if (split == 0)
      for (int i = tid; i < packed * kHead; i += kThreads)
        a.out[((int64_t)(item.y + i / kHead / G) * a.hq + kh * G + i / kHead % G) * kHead + i % kHead] = 0;
    return;
  }
  if (split >= used) return;
  const int t0 = split * split_len, t1 = (int)min((int64_t)most, (int64_t)t0 + split_len);
#pragma unroll
  for (int b = 0; b < NC; ++b) lim[b] = lim[b] < 0 ? t1 : lim[b];
  const int tiles = (t1 - t0 + kTile - 1) / kTile;
  const int mine = (tiles - wave + kWaves - 1) / kWaves;  // tiles wave, wave + 4, ..

  // 8-bit: blocks of kIds of the wave's tiles at a time: lane 2 k + b holds block b of tile k and its two exponents.
  const int64_t row_blocks = 2LL * a.hk;
  int ids = 0, exps = 0;
  auto next_blocks = [&](int k0) __attribute__((always_inline)) {
    const int tile = wave + kWaves * (k0 + (lane >> 1));
    const int b = (int)min((int64_t)(t0 / kQ8Block) + (int64_t)tile * kBlocksPerTile + (lane & 1), (int64_t)((t1 - 1) / kQ8Block));
    ids = (int)page_slot(a.pd, pg[page_index(a.pd, b)], b);
    const uint8_t* e = a.kv_scale + ids * row_blocks + kh;
    exps = e[0] | e[a.hk] << 16;
  };
  // One buffer for the waves' tiles of V (bf16: two each, of 8 KiB) and, in the end,
  // their parts of a block of columns (8.25 KiB each).
  constexpr int kPart = 16 * (kHead + 4), kVTile = kTile * kHead;
  __shared__ __align__(16) float s_buf[kWaves * (Q8 ? kPart : kVTile)];
  __shared__ float s_m[kWaves][16], s_l[kWaves][16];
  // E4M3: the first key of a wave's that holds a NaN in dim d of V, among the keys that
  // not all rows see, once there is one at all.
  constexpr bool NANS = Q8 && FMT == kQ8E4m3;
  __shared__ int s_nan[NANS ? kWaves : 1][kHead];
  bool bad = false;
  bf16_t* v_lds = reinterpret_cast<bf16_t*>(s_buf) + wave * (2 * kVTile);

  // bf16: a tile's rows from a scalar base, each lane's first one at a constant offset
  // (bytes); those past the last key are read as zeros.
  const int k_off = Q8 ? 0 : (2 * (col & 4) + (col & 3)) * 2 * (int)a.k_stride + 32 * grp + 2 * (col & 8);
  auto tile_rows = [&](const bf16_t* base, int64_t stride, int k) __attribute__((always_inline)) {
    const int n0 = t0 + (wave + kWaves * k) * kTile, rows = min(t1 - n0, kTile);
    return buffer_rsrc(base + (src0 + n0) * stride + (int64_t)kh * kHead, (rows - 1) * 2 * (int)stride + 2 * kHead);
  };
  uint4 kr[Q8 ? 2 : 4][2], vr[Q8 ? 4 : 1];
  auto load_k = [&](int k) __attribute__((always_inline)) {
    if constexpr (Q8) {
      const uint8_t* kb = a.kv + kh * kQ8HeadBytes + (2 * (col & 4) + (col & 3)) * kHead + 16 * grp + 8 * (col & 8);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int64_t block = __builtin_amdgcn_readlane(ids, 2 * (k & (kIds - 1)) + b);
#pragma unroll
        for (int j = 0; j < 2; ++j) kr[j][b] = ldg16_stream(kb + block * row_blocks * kQ8HeadBytes + 4 * j * kHead);
      }
    } else {
      // Rows 0-7 of the product, then 8-15, whole lines of 128 bytes, eight lanes a key; columns n and n + 8 trade halves.
      const auto rsrc = tile_rows(a.k, a.k_stride, k);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = k_off + (16 * i + 4 * j) * 2 * (int)a.k_stride;
          kr[2 * j][i] = ldb16_stream(rsrc, at), kr[2 * j + 1][i] = ldb16_stream(rsrc, at + 128);
        }
    }
  };
  auto load_v = [&](int k) __attribute__((always_inline)) {
    if constexpr (Q8) {
      const int64_t block = from_lane(ids, 2 * (k & (kIds - 1)) + (grp >> 1));
      const uint8_t* vb = a.kv + (block * row_blocks + a.hk + kh) * kQ8HeadBytes + (16 * (grp & 1) + col) * kQ8Block;
#pragma unroll
      for (int i = 0; i < 4; ++i) vr[i] = ldg16_stream(vb + i * 32 * kQ8Block);
    } else {
      // To LDS, four rows a load. 32-byte unit u of row r lies in unit u ^ (r % 4 + 4 (r / 8 % 2)):
      // the 8 rows x 32 bytes that 32 lanes of a transposing read take are disjoint banks.
      const auto rsrc = tile_rows(a.v, a.v_stride, k);
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the tile before has been read
#pragma unroll
      for (int i = 0; i < 8; ++i)
        dma16_stream(rsrc, (4 * i + grp) * 2 * (int)a.v_stride + 32 * ((col >> 1) ^ (grp | (i >> 1 & 1) << 2)) + 16 * (col & 1),
                     v_lds + (k & 1) * kVTile + 4 * i * kHead);
    }
  };

  f32x4 o[NC][8];
  float m[NC], l[NC];
#pragma unroll
  for (int b = 0; b < NC; ++b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[b][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[b] = -INFINITY, l[b] = 0.f;
  }
  if (mine > 0) {
    if constexpr (Q8)
      next_blocks(0);
    else
      load_v(0);
    load_k(0);
  }
  for (int k = 0; k < mine; ++k) {
    // 8-bit: V of this tile, then (when its scores are taken) K of the next: one of the
    // two is always in flight. bf16: V and K of the next tile when this one's scores are
    // taken; V, whose loads the compiler does not see, is waited for below.
    if constexpr (Q8) load_v(k);
    int e2 = 0;
    if constexpr (Q8) e2 = from_lane(exps, 2 * (k & (kIds - 1)) + (grp >> 1));
    const int n0 = t0 + (wave + kWaves * k) * kTile, left = t1 - n0;  // keys from this tile on
    float s[NC][8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 d[NC];
#pragma unroll
      for (int b = 0; b < NC; ++b) d[b] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (Q8)
        trade_halves(kr[j][0], kr[j][1]);
      else
        trade_halves(kr[2 * j][0], kr[2 * j][1]), trade_halves(kr[2 * j + 1][0], kr[2 * j + 1][1]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        bf16x8 ka;
        if constexpr (Q8) {
          const uint4& w = kr[j][kk >> 1];
          ka = kk & 1 ? bf16_of<FMT>(w.z, w.w) : bf16_of<FMT>(w.x, w.y);
        } else {
          ka = __builtin_bit_cast(bf16x8, kr[2 * j + (kk >> 1)][kk & 1]);
        }
#pragma unroll
        for (int b = 0; b < NC; ++b) d[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, q[b][kk], d[b], 0, 0, 0);
      }
#pragma unroll
      for (int b = 0; b < NC; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][4 * j + r] = d[b][r];
    }
    if constexpr (!Q8) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): V of this tile; K has been used, so that nothing younger is in flight
      asm volatile("" ::: "memory");       // V's reads stay behind it
    }
    if (k + 1 < mine) {
      if (Q8 && ((k + 1) & (kIds - 1)) == 0) next_blocks(k + 1);
      if constexpr (!Q8) load_v(k + 1);
      load_k(k + 1);
    }
    const float ks = Q8 ? pow2_biased(e2 & 0xff) * a.scale_log2 : a.scale_log2, vs = Q8 ? pow2_biased(e2 >> 16) : 1.f;
#pragma unroll
    for (int b = 0; b < NC; ++b)
#pragma unroll
      for (int t = 0; t < 8; ++t) s[b][t] *= ks;
    if (n0 + kTile > least) {  // keys that some row does not see
      const int key = n0 + 8 * ((NANS ? here(lane) : lane) >> 4);
#pragma unroll
      for (int b = 0; b < NC; ++b)
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (key + t >= lim[b]) s[b][t] = -INFINITY;
    }
    if constexpr (Q8) {
      if (left < kTile) {  // nothing past the last key that any row sees counts, whatever it holds
        const int tokens = left - kQ8Block * ((NANS ? here(lane) : lane) >> 5);  // of this lane's block
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int n_ok = min(max(tokens - 4 * w, 0), 4);
          const uint32_t stay = n_ok == 4 ? ~0u : (1u << (8 * n_ok)) - 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) (&vr[i].x)[w] &= stay;
        }
      }
    }
    bf16x8 ph[NC], pl[NC];
#pragma unroll
    for (int b = 0; b < NC; ++b) {
      float mx = s[b][0];
#pragma unroll
      for (int t = 1; t < 8; ++t) mx = fmaxf(mx, s[b][t]);
      mx = max_of_groups(mx);
      const bool grow = mx > m[b];
      if (__any(grow)) {
        const float to = mx + 8.f, alpha = grow ? fast_exp2(m[b] - to) : 1.f;
        m[b] = grow ? to : m[b];
        l[b] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[b][i] *= alpha;
      }
      const float base = m[b] == -INFINITY ? 0.f : m[b];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        s[b][t] = fast_exp2(s[b][t] - base);
        l[b] += s[b][t];
        s[b][t] *= vs;
      }
      const uint4 hi = pack8(s[b]);
      float rest[8];
      widen8(hi, rest);
#pragma unroll
      for (int t = 0; t < 8; ++t) rest[t] = s[b][t] - rest[t];
      ph[b] = __builtin_bit_cast(bf16x8, hi), pl[b] = __builtin_bit_cast(bf16x8, pack8(rest));
    }
    if constexpr (NANS) {
      // A NaN times the weight 0 of a row that does not see its key is NaN: where such
      // rows are it counts as 0 here, and the rows that do see it get it in the end.
      if (__builtin_expect(n0 + kTile > least, 1)) {
        uint32_t low = 0x7f7f7f7fu, one = 0x01010101u;  // in registers: half the bytes of code, which a small call waits for
        asm volatile("" : "+s"(low), "+s"(one));
        const auto nans = [&](uint32_t x) { return (x & low) + one; };  // bit 7 of a byte of 0x7f or 0xff
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) any |= nans((&vr[i].x)[w]);
        if (__builtin_expect(__any((any & 0x80808080u) != 0), 0)) {
          const int ln = here(lane);
          if (!bad) s_nan[wave][ln] = s_nan[wave][ln + 64] = INT_MAX;
          bad = true;
          const int dim = ln & 31, key = n0 + (ln & 32) / (32 / kQ8Block);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            int first = INT_MAX;
#pragma unroll
            for (int w = 3; w >= 0; --w) {
              const uint32_t x = (uint32_t)here((int)(&vr[i].x)[w]), nan = nans(x) & 0x80808080u;
              if (nan) first = key + 4 * w + ((__ffs(nan) - 8) >> 3);
              (&vr[i].x)[w] = x & ~((nan >> 7) * 0xffu);
            }
            atomicMin(&s_nan[wave][32 * i + dim], first);
          }
        }
      }
    }
    const auto weigh = [&](int i, const bf16x8& v) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < NC; ++b) {
        o[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph[b], o[b][i], 0, 0, 0);
        o[b][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl[b], o[b][i], 0, 0, 0);
      }
    };
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // Even groups keep tokens 0-7 of their dim and take those of the odd group's, and the other way round.
        const auto a0 = __builtin_amdgcn_permlane16_swap(vr[i].x, vr[i].z, false, false);
        const auto a1 = __builtin_amdgcn_permlane16_swap(vr[i].y, vr[i].w, false, false);
        weigh(2 * i, bf16_of<FMT>(a0[0], a1[0]));
        weigh(2 * i + 1, bf16_of<FMT>(a0[1], a1[1]));
      }
    } else {
      const bf16_t* vt = v_lds + (k & 1) * kVTile;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bf16x4 part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 8 * grp + 4 * h + (col >> 2), f = (r & 3) | (r >> 3 & 1) << 2;
          part[h] = lds_read_tr(vt + r * kHead + 16 * (i ^ f) + 4 * (col & 3));
        }
        weigh(i, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
      }
    }
  }

  // The waves' parts, merged, a block of columns at a time: O rows [column][dim], then
  // (m, l). A wave without a tile has m = -inf and zeros.
#pragma unroll
  for (int b = 0; b < NC; ++b) {
    if (16 * b >= packed) break;
    l[b] += xor_lane(l[b], 16);
    l[b] += xor_lane(l[b], 32);
    __syncthreads();  // V's tiles and the block before have been read
#pragma unroll
    for (int i = 0; i < 8; ++i)
      *reinterpret_cast<f32x4*>(s_buf + wave * kPart + col * (kHead + 4) + 16 * i + 4 * grp) = o[b][i];
    if (NANS && __builtin_expect(bad, 0)) {  // a NaN for the rows that see its key
#pragma unroll 1
      for (int d = 4 * grp; d < kHead; d += (d & 3) == 3 ? 13 : 1)
        if (s_nan[wave][d] < lim[b]) s_buf[wave * kPart + col * (kHead + 4) + d] = NAN;
    }
    if (grp == 0) s_m[wave][col] = m[b], s_l[wave][col] = l[b];
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 16 * kHead / 4 / kThreads; ++it) {  // four dims of a column a thread
      const int x = tid + it * kThreads, g = x / (kHead / 4), d = 4 * (x & (kHead / 4 - 1)), c = 16 * b + g;
      if (c >= packed) break;
      float wm[kWaves], top = -INFINITY, den = 0.f;
      f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) wm[w] = s_m[w][g], top = fmaxf(top, wm[w]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float e = fast_exp2(wm[w] - base);
        num += *reinterpret_cast<const f32x4*>(s_buf + w * kPart + g * (kHead + 4) + d) * e;
        den = fmaf(s_l[w][g], e, den);
      }
      const int row = row_of_column(c, a.g16), head = kh * G + c - row * G;
      const int64_t h = (int64_t)(item.y + row) * a.hq + head;
      if (used == 1) {
        uint2 w = make_uint2(pack_bf16x2(num[0] / den, num[1] / den), pack_bf16x2(num[2] / den, num[3] / den));
        if (Q8 && a.pos[item.y + row] < 0) w = make_uint2(0, 0);  // a row that is none, among rows that see keys
        *reinterpret_cast<uint2*>(a.out + h * kHead + d) = w;
      } else {
        // den = 0: the row sees nothing of this split (or every score is -inf): it weighs nothing beside the others.
        const int64_t at = ((int64_t)(item.w + row) * a.hq + head) * a.splits + split;
        *reinterpret_cast<f32x4*>(a.ws_o + at * kHead + d) = den == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : num / den;
        if (d == 0) a.ws_lse[at] = base + __log2f(den);
      }
    }
  }
}

// The splits of a group's rows, merged: sum of o_i 2^(lse_i - max) over the sum of
// those weights. 32 lanes of 4 dims a (row, head), kMergeBatch splits at a time, asked
// for before their weights are known. Bound by a round trip a batch, so that four waves
// take the batches in turn, and wave 0 joins them, where there are many: 5 rows over 60,000
// tokens of 16q/8kv in 62 splits, with the attention, 24.9 -> 20.8 us, 5 over 40,000 states of
// 4 heads in 59 19.7 -> 15.7; with 20 splits two batches of one wave are faster.
constexpr int kMergeBatch = 16;

template <bool Q8, int WAVES>
__global__ __launch_bounds__(kThreads) void rows_merge(RowsArgs a, int parts) {
  constexpr int kMergeRows = kThreads / 32 / WAVES;
  static_assert(kMergeRows == rows_merged(WAVES > 1 ? kRowsMergeMany + 1 : kRowsMergeMany), "as the grid has it");
  const int group = blockIdx.x / parts, wave = WAVES > 1 ? threadIdx.x >> 6 : 0, t = WAVES > 1 ? threadIdx.x & 63 : threadIdx.x;
  const int x = (blockIdx.x % parts) * kMergeRows + (t >> 5), head = x % a.hq;
  const int used = a.ws_used[group];
  const int4 item = reinterpret_cast<const int4*>(a.items)[group];
  if ((blockIdx.x % parts) * kMergeRows >= item.z * a.hq) return;
  const bool live = x / a.hq < item.z;
  const int row = live ? x / a.hq : 0;
  if (WAVES == 1 && !live) return;
  const bool none = Q8 && a.pos[item.y + row] < 0;
  const int lane = threadIdx.x & 31;
  const int64_t h = (int64_t)(item.w + row) * a.hq + head;
  const float* lse = a.ws_lse + h * a.splits;
  const float* part = a.ws_o + h * a.splits * kHead + 4 * lane;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, den = 0.f;
  for (int i0 = kMergeBatch * wave, begun = 0; i0 < used || !begun; i0 += kMergeBatch * WAVES, begun = 1) {
    f32x4 o[kMergeBatch];
    float e[kMergeBatch];
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      const int i = min(i0 + j, (begun ? used : a.splits) - 1);  // the first are asked for before it is known how many count
      e[j] = lse[i];
      o[j] = *reinterpret_cast<const f32x4*>(part + (int64_t)i * kHead);
    }
    if (!begun && used <= 1) return;
    float mx = top;
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) mx = i0 + j < used ? fmaxf(mx, e[j]) : mx;
    const float base = mx == -INFINITY ? 0.f : mx, alpha = fast_exp2(top - base);
    top = mx;
    num *= alpha, den *= alpha;
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j)
      if (i0 + j < used) {  // what was asked for beyond may be anything
        const float w = fast_exp2(e[j] - base);
        num += o[j] * w, den += w;
      }
  }
  if (WAVES > 1 && used > kMergeBatch) {  // else wave 0 had them all
    __shared__ float s_part[WAVES > 1 ? WAVES - 1 : 1][6][64];
    if (wave > 0) {
      s_part[wave - 1][4][t] = den, s_part[wave - 1][5][t] = top;
#pragma unroll
      for (int e = 0; e < 4; ++e) s_part[wave - 1][e][t] = num[e];
    }
    __syncthreads();
    float mx = top;
#pragma unroll
    for (int v = 0; v < WAVES - 1; ++v) mx = fmaxf(mx, s_part[v][5][t]);
    const float base = mx == -INFINITY ? 0.f : mx, own = fast_exp2(top - base);
    num *= own, den *= own;
#pragma unroll
    for (int v = 0; v < WAVES - 1; ++v) {
      const float e = fast_exp2(s_part[v][5][t] - base);
      den = fmaf(s_part[v][4][t], e, den);
#pragma unroll
      for (int d = 0; d < 4; ++d) num[d] = fmaf(s_part[v][d][t], e, num[d]);
    }
  }
  if (wave > 0 || !live) return;
  uint2 w = make_uint2(pack_bf16x2(num[0] / den, num[1] / den), pack_bf16x2(num[2] / den, num[3] / den));
  if (none) w = make_uint2(0, 0);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)(item.y + row) * a.hq + head) * kHead + 4 * lane) = w;
}

template <int SRC>
int launch(const RowsArgs& a, const int* groups, hipStream_t stream) {
  RowsArgs x = a;
  x.g16 = 65536 / (a.hq / a.hk) + 1;
  for (int c = 0; c < 2; ++c) {
    if (groups[c] == 0) continue;
    const int64_t grid = (int64_t)groups[c] * a.hk * a.splits;
    if (c == 0)
      rows_attn<SRC, 1><<<(unsigned)grid, kThreads, 0, stream>>>(x);
    else
      rows_attn<SRC, 2><<<(unsigned)grid, kThreads, 0, stream>>>(x);
    if (check_launch() != 0) return -3;
    if (a.splits > 1) {
      const int rows = std::max((c + 1) * 16 / (a.hq / a.hk), 1), per = rows_merged(a.splits);
      const int parts = (rows * a.hq + per - 1) / per;
      const unsigned wgs = (unsigned)((int64_t)groups[c] * parts);
      if (a.splits > kRowsMergeMany)
        rows_merge<SRC != kBf16, 4><<<wgs, kThreads, 0, stream>>>(x, parts);
      else
        rows_merge<SRC != kBf16, 1><<<wgs, kThreads, 0, stream>>>(x, parts);
      if (check_launch() != 0) return -3;
    }
    x.items += 4 * (int64_t)groups[c], x.ws_used += groups[c];
  }
  return 0;
}

}  // namespace

int launch_rows(const RowsArgs& a, int source, const int* groups, hipStream_t stream) {
  return source == kRowsBf16 ? launch<kBf16>(a, groups, stream)
         : source == kQ8E4m3 ? launch<kQ8E4m3>(a, groups, stream)
                             : launch<kQ8Int8>(a, groups, stream);
}

}  // namespace omni
