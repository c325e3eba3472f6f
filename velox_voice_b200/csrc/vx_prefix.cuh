// Attention over shared prefixes and own tokens: how the work is cut, for the kernels that do the parts of it (vx_prefix_attn.cu,
// vx_prefix_tiles.cu).
//
// A SPAN is one kind of keys: those of the groups' prefixes, the sequences' own tokens, or both in a row (joint).  Its owners (groups,
// sequences, sequences) have runs of rows; row rho of an owner and a key head stands for token rho / per_kv of its run and query head
// rho % per_kv, so that all query heads that share a key head read its keys together.  Rows are cut into tiles, keys into chunks.  An
// item is one tile, one chunk and one key head; it leaves (m, l, O) of its rows -- a maximum or a number near it, sum of 2^(x - m), sum of
// 2^(x - m) v, with x = scale log2(e) q.k -- as part `part0 + chunk` in scratch, from which a last kernel joins the parts of a row:
//   out = sum_c 2^(m_c - m) O_c / sum_c 2^(m_c - m) l_c,  m = max_c m_c.
// The number of chunks is fixed on the host from the width of the tables; how many of them hold keys is known on the device only, and
// both sides derive it from the same lengths, so empty parts are neither written nor read.
//
// Places that no row of a tile sees are filled with zeros.  New tokens of a sequence lie in one tile with rows that see them and rows that do
// not, and a probability of 0 times a value that is not finite would reach the latter: where such a tile holds one, its product with the
// values is formed another way.
#pragma once

#include "vx_paged.cuh"

namespace vx {

struct PrefixParams {
  PagedCache cache;               // (a cache in 4 bits: page size and number of pages only)
  Fp4Cache fp4;
  KvRows rows;
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  __nv_bfloat16* out;
  int64_t o_row, o_head;
  int32_t q_heads, kv_heads;
  FastDiv per_kv;
  int32_t groups, group_size;     // group_size: equal groups, 0 with group_offsets
  const int32_t* group_offsets;
  PagedTable prefix;
  const int32_t* prefix_lengths;
  float scale2;                   // scale log2(e); a cache in 4 bits: times 256 k_scale, see e4m3_as_half
  float v_factor;                 // of a cache in 4 bits: 256 v_scale
  float2* part_ml;                // [parts][rows][q_heads]
  float* part_o;                  // [parts][rows][q_heads][head_dim]
  int* status;
};

enum SpanKind : int32_t { kSpanPrefix = 0, kSpanOwn = 1, kSpanJoint = 2 };
constexpr int kSpanAlign = 128;  // own keys of a joint span begin at the next multiple of this behind the prefix

// One span as a kernel walks it.
struct Span {
  int32_t kind;
  int32_t slots;      // row tiles there can be; a slot without rows is skipped
  int32_t equal;      // tiles per owner where all have as many rows; 0: found from the offsets
  int32_t chunk;      // keys per chunk
  int32_t chunks;     // 0: the span is not walked
  int32_t part0;      // first part in scratch; -1: the only part there is, its rows go to `out`
};
constexpr Span kNoSpan{0, 1, 1, 1, 0, 0};

__device__ __forceinline__ int sequence_row0(const PrefixParams& p, int s) {
  return p.rows.row_offsets ? min(max(p.rows.row_offsets[s], 0), p.rows.rows) : s;
}
__device__ __forceinline__ int group_sequence0(const PrefixParams& p, int g) {
  return p.group_offsets ? min(max(p.group_offsets[g], 0), p.rows.sequences) : g * p.group_size;
}
// first row of owner o (o = number of owners: the end of the last)
__device__ __forceinline__ int owner_row0(const PrefixParams& p, bool sequences, int o) {
  return sequence_row0(p, sequences ? o : group_sequence0(p, o));
}

// group of a sequence, -1: none; all lanes of the warp ask for the same one
__device__ __forceinline__ int group_of(const PrefixParams& p, int s) {
  if (p.groups == 0) return -1;
  if (!p.group_offsets) return s / p.group_size;
  const int g = find_by_warp(p.groups, s, [&](int o) { return p.group_offsets[o]; });
  return s >= p.group_offsets[g] && s < p.group_offsets[g + 1] ? g : -1;
}

// Keys of the prefix of group g, and own keys that the i-th token behind `length` others of its sequence sees: as far as the tables reach.
__device__ __forceinline__ int prefix_keys(const PrefixParams& p, int g) {
  const int cap = p.prefix.pages * static_cast<int>(p.cache.page_size.d);
  return g < 0 ? 0 : min(max(p.prefix_lengths[g], 0), cap);
}
__device__ __forceinline__ int own_keys(const PrefixParams& p, int length, int64_t i) {
  const int cap = p.rows.table.pages * static_cast<int>(p.cache.page_size.d);
  return length < 0 ? 0 : static_cast<int>(min(length + i + 1, static_cast<int64_t>(cap)));
}
// Tokens of sequence s in front of its first row that the call has, as far as the table reaches: those of the cache and, where its offset lies
// in front of the call's rows, those between; negative: it takes no part.
__device__ __forceinline__ int tokens_before(const PrefixParams& p, int s) {
  const int length = p.rows.lengths[s];
  if (length < 0 || !p.rows.row_offsets) return length;
  const int64_t cap = static_cast<int64_t>(p.rows.table.pages) * static_cast<int>(p.cache.page_size.d);
  return static_cast<int>(min(length + max(-static_cast<int64_t>(p.rows.row_offsets[s]), static_cast<int64_t>(0)), cap));
}
__device__ __forceinline__ int align_keys(int n) { return (n + kSpanAlign - 1) / kSpanAlign * kSpanAlign; }

// First row of a tile of a run of so many rows, -1: it has none.  (Compared before it is multiplied: offsets that do not ascend ask for any tile.)
__device__ __forceinline__ constexpr int first_row(int tile, int tm, int rows) { return tile >= 0 && rows > 0 && tile <= (rows - 1) / tm ? tile * tm : -1; }

// Rows of an item.
struct ItemRows {
  int owner;
  int row0, rows;   // first token of the owner's run, rows (token, head of the key head's group) of the run
  int rho0;         // first row of the tile
};

// Owner and tile of a slot.  With offsets, owner o has the slots [base(o), base(o + 1)), base(o) = floor(row0(o) per_kv / TM) + o: enough for
// its tiles, and found by a search without a pass over all owners.  All lanes of the warp ask for the same slot.
template <int TM>
__device__ __forceinline__ bool find_rows(const PrefixParams& p, const Span& sp, int slot, ItemRows& it) {
  const int per = static_cast<int>(p.per_kv.d);
  const bool sequences = sp.kind != kSpanPrefix;
  const int owners = sequences ? p.rows.sequences : p.groups;
  int tile;
  if (sp.equal) {
    it.owner = slot / sp.equal;
    tile = slot - it.owner * sp.equal;
  } else {
    auto base = [&](int o) { return static_cast<int>(static_cast<int64_t>(owner_row0(p, sequences, o)) * per / TM) + o; };
    it.owner = find_by_warp(owners, slot, base);  // the largest with base(o) <= slot
    tile = slot - base(it.owner);
  }
  if (it.owner >= owners) return false;
  it.row0 = owner_row0(p, sequences, it.owner);
  const int n = owner_row0(p, sequences, it.owner + 1) - it.row0;
  it.rows = n * per;
  it.rho0 = first_row(tile, TM, it.rows);
  return it.rho0 >= 0;
}

// The tiles of a span counted by a warp, without the slots that have no rows: a kernel whose CTAs take items in turn shares them out evenly.
struct SpanTiles {
  int block;   // owners per lane
  int before;  // tiles of the owners in front of this lane's
  int tiles;   // all of them
  int row0, rows;  // with one owner per lane: its run
};
__device__ __forceinline__ int scan_by_warp(int n) {  // the sum up to this lane, its own included
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, n, x);
    if (lane >= x) n += y;
  }
  return n;
}
template <int TM>
__device__ __forceinline__ int owner_tiles(const PrefixParams& p, bool sequences, int o, int& row0, int& rows) {
  row0 = owner_row0(p, sequences, o);
  rows = (owner_row0(p, sequences, o + 1) - row0) * static_cast<int>(p.per_kv.d);
  return rows > 0 ? (rows - 1) / TM + 1 : 0;
}
template <int TM>
__device__ __forceinline__ SpanTiles count_tiles(const PrefixParams& p, const Span& sp) {
  const bool sequences = sp.kind != kSpanPrefix;
  const int owners = sequences ? p.rows.sequences : p.groups, lane = threadIdx.x & 31;
  SpanTiles st{};
  if (sp.chunks == 0) return st;
  if (sp.equal) {
    st.tiles = owners * sp.equal;
    return st;
  }
  st.block = (owners + 31) / 32;
  int n = 0;
#pragma unroll 4
  for (int i = 0; i < st.block; ++i)
    if (lane * st.block + i < owners) n += owner_tiles<TM>(p, sequences, lane * st.block + i, st.row0, st.rows);
  const int sum = scan_by_warp(n);
  st.before = sum - n;
  st.tiles = min(max(__shfl_sync(0xffffffffu, sum, 31), 0), sp.slots);  // (offsets that do not ascend)
  return st;
}
// Rows of tile t; all lanes of the warp ask for the same one.
template <int TM>
__device__ __forceinline__ bool find_tile(const PrefixParams& p, const Span& sp, const SpanTiles& st, int t, ItemRows& it) {
  const bool sequences = sp.kind != kSpanPrefix;
  const int owners = sequences ? p.rows.sequences : p.groups, lane = threadIdx.x & 31;
  int tile = 0;
  if (sp.equal) {
    it.owner = t / sp.equal;
    tile = t - it.owner * sp.equal;
  } else {
    const int src = 31 - __clz(__ballot_sync(0xffffffffu, lane == 0 || st.before <= t));  // the lane that counted it
    const int before = __shfl_sync(0xffffffffu, st.before, src);
    it.row0 = __shfl_sync(0xffffffffu, st.row0, src);
    it.rows = __shfl_sync(0xffffffffu, st.rows, src);
    it.owner = src;
    tile = t - before;
    if (st.block > 1) {  // 32 of its owners at a time
      it.owner = -1;
      int first = before;
      for (int o = src * st.block, end = min(o + st.block, owners); o < end; o += 32) {
        int row0, rows;
        const int n = o + lane < end ? owner_tiles<TM>(p, sequences, o + lane, row0, rows) : 0, sum = scan_by_warp(n), all = __shfl_sync(0xffffffffu, sum, 31);
        if (t < first + all) {
          const int k = __ffs(__ballot_sync(0xffffffffu, t < first + sum)) - 1;
          it.owner = o + k;
          it.row0 = __shfl_sync(0xffffffffu, row0, k);
          it.rows = __shfl_sync(0xffffffffu, rows, k);
          tile = t - first - __shfl_sync(0xffffffffu, sum - n, k);
          break;
        }
        first += all;
      }
      if (it.owner < 0) return false;
    }
  }
  if (sp.equal) {
    it.row0 = owner_row0(p, sequences, it.owner);
    it.rows = (owner_row0(p, sequences, it.owner + 1) - it.row0) * static_cast<int>(p.per_kv.d);
  }
  it.rho0 = first_row(tile, TM, it.rows);
  return it.rho0 >= 0;
}

// Not 0 if one of the two bf16 values of a word is an infinity or NaN, gathered in `sum` (0 x is 0 or NaN).
__device__ __forceinline__ void note_not_finite(uint32_t& sum, uint32_t two) { asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(two), "r"(0u)); }
__device__ __forceinline__ bool any_not_finite(uint32_t sum) { return (sum & 0x7fff7fffu) != 0; }

// A cache in 4 bits: probabilities are formed in fp16 as 2^(x - reference), the reference this far below a maximum (see vx_prefix_fp4.cu).
constexpr float kFp4Below = 7.0f;

// What the kernels for few rows walk.
struct RowsParams {
  PrefixParams p;
  Span span[2];
  int32_t warps[2];      // of a CTA per item of the span: 1, 2 or 4; a cache in 4 bits, one span: 8 or 16 too, a CTA of so many
  int32_t first_blocks;  // CTAs of span[0]; those of span[1] follow
  int32_t beside;        // the launch in front is the tile kernel of this call, see prefix_rows_kernel
};
constexpr int PR_WARPS = 4;
// Launches prefix_rows_fp4_kernel with `blocks` CTAs of RB blocks of eight rows.
int launch_rows_fp4(const RowsParams& rp, int head_dim, int rb, int64_t blocks, void* stream);
int rows_fp4_ctas(int rb, int head_dim);  // per SM

// Launches prefix_tiles_kernel on the spans that have chunks.
constexpr int kSlotRows = 128;  // rows of a slot of prefix_tiles_kernel
int launch_prefix_tiles(const PrefixParams& p, int head_dim, bool paired, bool fp4, const Span& first, const Span& second, void* stream);

}  // namespace vx
