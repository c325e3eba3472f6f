// Attention over shared prefixes and own tokens on the 5th-generation tensor cores (the cut of the work: vx_prefix.cuh; few rows and keys:
// vx_prefix_attn.cu).
//
// One CTA per SM goes through its items.  It has two SLOTS of 128 rows with tensor memory of their own; while the softmax of one slot works,
// the tensor cores have the products of the other.
//   PAIRED     both slots take one item of 256 rows, 128 keys a tile: every K and V tile is loaded once for both.  For many rows per owner,
//              where the products are the bound.  Tensor memory of a slot: S (128 columns, P in bf16 over it) | O (head_dim).  (Tiles of 64 keys
//              and two S here too, an MMA issuer per slot: 2,125 us against 1,815 for 6,906 tokens of four prompts behind 16,384; a product of
//              64 columns reads all of Q from shared memory for half the work.)
//   otherwise  each slot has a stream of items of its own, 64 keys a tile, and the tiles of the two take turns.  For few rows, where the keys'
//              bytes are the bound: smaller tiles hold less of the shared memory while their softmax runs, so more of it is for copies in
//              flight (with tiles of 128 keys a third of the time was lost), and S is double-buffered, so that the softmax of a slot
//              finds its next S.  Tensor memory of a slot: S0 | S1 (64 columns each, P over them) | O.
// Roles:
//   warps 0..3, 4..7  softmax of slot 0, 1: a query row per thread straight out of tensor memory
//   warps 8..11       loaders, K and V into rings of the stream, page by page (cp.async, 16 bytes; keys that are not there are filled with zeros
//                     and marked in a bit mask).  PAIRED each takes a quarter of every tile (with whole tiles in turn a tile was 2 us late); else
//                     two warps per stream take its tiles in turn (with quarters 1,500 of 1,950 cycles went into what a tile costs whatever its
//                     size, and the loaders were the bound).
//   warps 12, 15      MMA issuers.  A thread that issues is held while its products run, so the slots of two streams have one each: what it
//                     has to wait for and to look up between two tiles passes under the other's products (one issuer for both spent 60 % of its
//                     time between products).  PAIRED has one for both slots, whose products must not mix: two issuers without turns
//                     took 27 % longer, with turns 8 %.
//   warps 13, 14      one per stream of items: looks them up, hands them to the other roles through a ring and loads their queries
//                     (PAIRED the second warp loads those of the second slot)
// All roles run on into the next item as far as their rings and buffers let them, so that what an item costs to begin (its place in the tables,
// its queries, its first keys) passes under the one before it.
// Q, K and V lie in shared memory in rows of 128 bytes with the 128-byte swizzle, 64 columns a panel; V is read as an MN-major operand.
// P is the A operand in tensor memory, so that shared memory is read for K, Q and V only.  S of a tile is issued behind the P V product that
// reads P from the same columns, by the same thread: the tensor cores take its products in order.
// The reference maximum of a row moves only when a tile's maximum exceeds it by more than 8 in units of log2 (probabilities stay below
// 2^8); then the row's sum and its O are scaled before P is handed over.
// What bounds it.  PAIRED: the round trip of a slot -- 2,000 cycles of softmax (1,024 of them exponentials: 128 x 128 at 16 a cycle for each of
// two slots), then P V and the next S, 1,024 cycles of the tensor cores, with hand-over and the other slot's products in between: 3,900 cycles
// a tile of 256 rows by 128 keys: 6,906 tokens of four prompts behind 16,384 (32 query heads on 8 key heads of 128) take 1,780 us with pauses
// between the calls, 1.12 PFLOP/s, and 2,040, 0.98, in calls one after the other, where the power cap lowers the clock.  Otherwise: bytes from L2
// and HBM where there are many keys (128 rows a head over 90,000 keys, 84 us, 4.4 TB/s), the softmax of a tile (some 1,950 cycles) where keys are shared by many
// rows, and what a CTA costs to begin and end where an SM has a few tiles only (16 groups of 100 rows over 64 keys, one tile each: 11 us at head_dim 64).
// Every wait on a barrier is bounded.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "vx_common.cuh"
#include "vx_prefix.cuh"
#include "vx_ptx.cuh"
#include "vx_quant_math.cuh"

namespace vx {
namespace {

constexpr int PT_THREADS = 16 * 32;
constexpr int PT_MASKS = 16;               // tiles of a stream whose masks are kept: more than a ring of keys holds and a slot has begun
constexpr int PT_ITEMS = 4;                // items of a stream that are known ahead
constexpr int PT_Q_PANEL = kSlotRows * 128;  // 64 bf16 of every row
constexpr uint32_t PT_TM_SLOT = 256, PT_TM_O = 128, PT_TM_COLS = 512;

template <int D, bool PAIRED>
struct TileShape {
  static constexpr int kKeys = PAIRED ? 128 : 64;
  static constexpr int kBuffers = PAIRED ? 1 : 2;             // of S
  static constexpr int kPanel = kKeys * 128;                  // 64 bf16 of every key
  static constexpr int kTile = D / 64 * kPanel;               // bytes of a K or V tile
  static constexpr int kQ = D / 64 * PT_Q_PANEL;              // of a slot's queries
  static constexpr int kStreams = PAIRED ? 1 : 2;
  static constexpr int kParts = PAIRED ? 4 : 1;               // loaders that share a tile
  // P of a tile handed over in halves, so that the products of the first run under the exponentials of the second.  Gains where the products are
  // short (16 utterances of 3,116 to 5,510 frames, 9,894 tokens of 66 prompts, head_dim 64: 363 -> 339 us) and loses where an issuer that waits for the
  // second half keeps the other slot's products waiting (6,906 tokens of four prompts behind 16,384, head_dim 128: 1,710 -> 1,755).
  static constexpr bool kHalves = PAIRED && D == 64;
  static constexpr int kStagesK = D == 128 ? 3 : 5, kStagesV = D == 128 ? 2 : 5;  // of a stream
  static constexpr int kSmem = 2 * kQ + kStreams * (kStagesK + kStagesV) * kTile + 1024;
};

struct TilesParams {
  PrefixParams p;
  Span span[2];
};

// What the roles know of an item.  Its keys are those from v0 on of the row prefix keys (padded to p128) | own keys.
struct TileItem {
  int tiles;              // 0: the stream ends
  int n[2];               // tiles that the slots of a pair take
  int head, row0, rows, rho0;
  int v0, p128, p_keys, o_keys;
  int group, sequence, length;
  int part;
};

template <class Shape>
struct TileBarriers {
  uint64_t k_full[Shape::kStreams][Shape::kStagesK], k_empty[Shape::kStreams][Shape::kStagesK];
  uint64_t v_full[Shape::kStreams][Shape::kStagesV], v_empty[Shape::kStreams][Shape::kStagesV];
  uint64_t p_half[2];  // kHalves: the first half of a tile's P
  uint64_t s_full[2][Shape::kBuffers], p_full[2][Shape::kBuffers], pv_done[2][Shape::kBuffers], q_full[2], q_empty[2];
  uint64_t mask_full[2][PT_MASKS], item_full[2][PT_ITEMS], item_empty[2][PT_ITEMS];
  alignas(16) uint16_t mask[2][PT_MASKS][Shape::kKeys / 16];
  TileItem item[2][PT_ITEMS];
  uint32_t tmem_base;
};

// bf16 x bf16 -> fp32, A K-major; B K-major or MN-major (b_mn)
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void mma_bf16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
// The barrier is arrived at once for this thread when its copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// A whole 32-byte sector from one lane: lanes write rows of their own.
__device__ __forceinline__ void store32(float* dst, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// The factor of a row's scores and its reference maximum.  2^(scale2 s - m) has the product unrounded and m rounded: it is off by 2^(half a unit of m),
// the same for all keys of the row and in its sum, which leaves the range where m is 2^31 or more.  From 2^30 on scale2 without its mantissa
// stands in, and products are exact: two different scores are 64 or more in log2 apart there, 32 with the smaller factor, so that the
// largest takes all of the weight either way.
constexpr float PT_LARGE = 1073741824.0f;
__device__ __forceinline__ float without_mantissa(float x) { return __uint_as_float(__float_as_uint(x) & 0x7f800000u); }
// such a reference maximum in units of log2, for the parts of a row and where it moves
__device__ __forceinline__ float in_log2(float m, float factor, float scale2) {
  return factor == scale2 ? m : m * __uint_as_float((__float_as_uint(scale2) & 0x007fffffu) | 0x3f800000u);
}
// bits [0, n) of a word
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1); }

// Item n of a span, heads next to each other, then tiles, then chunks; false: there is nothing to do for it.  All lanes of the warp.
template <bool PAIRED, int KEYS>
__device__ bool find_tile_item(const PrefixParams& p, const Span& sp, const SpanTiles& st, uint32_t n, TileItem& t) {
  constexpr int TM = PAIRED ? 2 * kSlotRows : kSlotRows;
  const uint32_t kv = static_cast<uint32_t>(p.kv_heads), tile = n / kv, tiles = static_cast<uint32_t>(st.tiles);
  t.head = static_cast<int>(n - tile * kv);
  const int chunk = static_cast<int>(tile / tiles);
  ItemRows r;
  if (!find_tile<TM>(p, sp, st, static_cast<int>(tile - static_cast<uint32_t>(chunk) * tiles), r)) return false;
  t.row0 = r.row0; t.rows = r.rows; t.rho0 = r.rho0;
  t.group = t.sequence = t.length = 0;
  t.p_keys = t.o_keys = 0;
  if (sp.kind == kSpanPrefix) {
    t.group = r.owner;
    t.p_keys = prefix_keys(p, r.owner);
  } else {
    t.sequence = r.owner;
    t.length = tokens_before(p, r.owner);
    if (t.length < 0) return false;
    if (sp.kind == kSpanJoint) {
      t.group = group_of(p, r.owner);
      t.p_keys = prefix_keys(p, t.group);
    }
    t.o_keys = own_keys(p, t.length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(min(r.rho0 + TM, r.rows) - 1))));
  }
  t.p128 = align_keys(t.p_keys);
  const int64_t v0 = static_cast<int64_t>(chunk) * sp.chunk, end = sp.kind == kSpanPrefix ? t.p_keys : static_cast<int64_t>(t.p128) + t.o_keys;
  if (v0 >= end) return false;
  t.v0 = static_cast<int>(v0);
  auto tiles_to = [&](int64_t e) {  // of the chunk, for rows that see keys up to e
    if (e > v0 + sp.chunk) e = v0 + sp.chunk;
    return e <= v0 ? 0 : static_cast<int>((e - v0 + KEYS - 1) / KEYS);
  };
  t.tiles = tiles_to(end);
  if (PAIRED) {
    const bool other = r.rows - r.rho0 > kSlotRows;
    t.n[0] = t.n[1] = t.tiles;
    if (!other) t.n[1] = 0;
    else if (sp.kind != kSpanPrefix)
      t.n[0] = tiles_to(static_cast<int64_t>(t.p128) + own_keys(p, t.length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(r.rho0 + kSlotRows - 1)))));
  } else {
    t.n[0] = t.n[1] = t.tiles;
  }
  t.part = sp.part0 < 0 ? -1 : sp.part0 + chunk;
  return true;
}

// Whether one of the keys [from, to) of a tile has a value that is not finite.  All lanes of the warp.
template <int D, int PANEL>
__device__ __forceinline__ bool values_not_finite(const uint8_t* tile, int from, int to) {
  const int lane = threadIdx.x & 31;
  uint32_t sum = 0;
#pragma unroll 4
  for (int key = from + (lane >> 3); key < to; key += 4)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const uint4 w = *reinterpret_cast<const uint4*>(tile + i * PANEL + key * 128 + (lane & 7) * 16);
      note_not_finite(sum, w.x);
      note_not_finite(sum, w.y);
      note_not_finite(sum, w.z);
      note_not_finite(sum, w.w);
    }
  return __any_sync(0xffffffffu, any_not_finite(sum));
}

// O of this lane's row behind a tile, into `o`: P of the tile (tensor memory, bf16) times the values of the keys that the row sees (those of
// the mask `there` below `sees`), added to what tensor memory holds (`first`: nothing).  For tiles that values_not_finite is true of; all
// lanes of the warp.
template <int D, int KEYS>
__device__ __noinline__ void add_tile_apart(float* o, uint32_t o_tmem, uint32_t p_tmem, bool first, const uint32_t* there, int sees, const uint8_t* tile) {
#pragma unroll 1
  for (int i = 0; i < D / 16; ++i) {
    uint32_t x[16];
    tc_ld_x16(o_tmem + 16 * i, x);
    tc_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) o[16 * i + e] = first ? 0.0f : __uint_as_float(x[e]);
  }
#pragma unroll 1
  for (int i = 0; i < KEYS / 32; ++i) {
    uint32_t x[16];
    tc_ld_x16(p_tmem + 16 * i, x);
    tc_wait_ld();
#pragma unroll 1
    for (int e = 0; e < 32; ++e) {
      uint32_t two = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) two = k == e >> 1 ? x[k] : two;
      const float w = __uint_as_float(e & 1 ? two & 0xffff0000u : two << 16);
      const int key = 32 * i + e;
      if (!((there[i] >> e) & 1) || key >= sees) continue;
#pragma unroll 1
      for (int c = 0; c < D / 8; ++c) {
        const uint4 u = *reinterpret_cast<const uint4*>(tile + (c >> 3) * (KEYS * 128) + key * 128 + (((c & 7) ^ (key & 7)) << 4));
        const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[8 * c + 2 * k] += w * __uint_as_float(v[k] << 16);
          o[8 * c + 2 * k + 1] += w * __uint_as_float(v[k] & 0xffff0000u);
        }
      }
    }
    __syncwarp();
  }
}
template <int D>
__device__ __noinline__ void put_back(const float* o, uint32_t o_tmem) {
#pragma unroll 1
  for (int i = 0; i < D / 16; ++i) {
    uint32_t x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(o[16 * i + e]);
    tc_st_x16(o_tmem + 16 * i, x);
  }
  tc_wait_st_all();
}

template <int D, bool PAIRED>
__global__ void __launch_bounds__(PT_THREADS, 1) prefix_tiles_kernel(const __grid_constant__ TilesParams tp) {
  using Shape = TileShape<D, PAIRED>;
  constexpr int BN = Shape::kKeys, NB = Shape::kBuffers, NK = Shape::kStagesK, NV = Shape::kStagesV;
  constexpr int STREAMS = PAIRED ? 1 : 2;
  constexpr unsigned ALL = 0xffffffffu;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const q_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* const k_ring = q_s + 2 * Shape::kQ;
  uint8_t* const v_ring = k_ring + STREAMS * NK * Shape::kTile;
  __shared__ TileBarriers<Shape> bar;
  const PrefixParams& p = tp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp < 2) {  // each lane some barriers
    const int s = warp;  // slot, stream
    for (int i = lane; i < PT_MASKS; i += 32) mbar_init(&bar.mask_full[s][i], Shape::kParts);
    if (lane < PT_ITEMS) {
      mbar_init(&bar.item_full[s][lane], 1);
      mbar_init(&bar.item_empty[s][lane], 4 / STREAMS + 1 + 8 / STREAMS + (PAIRED ? 1 : 0));  // warps that read an item: loaders, MMA issuer, softmax, the second slot's queries
    }
    if (lane < NB) {
      mbar_init(&bar.s_full[s][lane], 1);
      mbar_init(&bar.p_full[s][lane], 4);
      mbar_init(&bar.pv_done[s][lane], 1);
    }
    if (lane == 0) {
      mbar_init(&bar.q_full[s], 64 / STREAMS);  // threads that load queries
      mbar_init(&bar.q_empty[s], 1);
      mbar_init(&bar.p_half[s], 4);
    }
    if (s < STREAMS && lane < NK) {
      mbar_init(&bar.k_full[s][lane], 32 * Shape::kParts);  // threads of the loaders that share a tile
      mbar_init(&bar.k_empty[s][lane], 1);
    }
    if (s < STREAMS && lane < NV) {
      mbar_init(&bar.v_full[s][lane], 32 * Shape::kParts);
      mbar_init(&bar.v_empty[s][lane], 1);
    }
    mbar_fence_init();
  }
  if (warp == 12) {
    tmem_alloc(&bar.tmem_base, PT_TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bar.tmem_base;
  pdl_wait();
  pdl_launch_dependents();
  // Registers: 128 a thread at launch, 512 for a thread of each of the four warpgroups.  The softmax, which holds a row of S, takes more in
  // two of them, the other two leave as many (2 n + 2 (256 - n) = 512); every warp of a warpgroup passes the same setmaxnreg.
  constexpr int SOFTMAX_REGS = PAIRED ? 192 : 168;

  // The items of a stream, one after another: waits for the next, copies it, hands its place back.
  struct Items {
    int at = 0;
    uint32_t phase = 0;
  };
  auto next_item = [&](int stream, Items& c, TileItem& t) {
    if (!__all_sync(ALL, mbar_wait_spin(&bar.item_full[stream][c.at], c.phase, p.status, 48))) return false;
    t = bar.item[stream][c.at];
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar.item_empty[stream][c.at]);
    if (++c.at == PT_ITEMS) { c.at = 0; c.phase ^= 1; }
    return true;
  };

  if (warp >= 8 && warp < 12) {
    // =========================== loaders ===========================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(256 - SOFTMAX_REGS));
    constexpr int PARTS = Shape::kParts, TEAM = 4 / STREAMS / PARTS;  // loaders that share a tile, that take tiles in turn
    constexpr int MINE = BN / PARTS, GROUPS = MINE / 16, PER_LANE = MINE / 32;
    const int stream = (warp - 8) / (4 / STREAMS), part = (warp - 8) % PARTS, rank = (warp - 8) / PARTS % TEAM;
    constexpr int LANES = D / 8;           // lanes that share a key
    constexpr int KEYS = 32 / LANES;       // keys per instruction
    const int piece = lane % LANES, sub = lane / LANES;
    const uint32_t at = (piece >> 3) * Shape::kPanel + (part * MINE + sub) * 128, swz = ((piece & 7) ^ sub) << 4;  // (key & 7 = sub + a multiple of KEYS)
    const bool whole_pages = p.cache.page_size.d % 16 == 0;  // 16 keys from a multiple of 16 on lie on one page
    bool ok = true;
    // Where this warp's keys of a tile are, a table entry looked up per lane: with whole pages lane i has the first of keys [16 i, 16 i + 16) and
    // how many of them there are, otherwise keys lane and lane + 32.
    int page[PER_LANE], n = 0;
    uint32_t place[PER_LANE];
    TileItem t;
    t.tiles = 0;
    auto look_up = [&](int tile) {
      const int v = t.v0 + tile * BN;
      const bool own = v >= t.p128;
      const int first = v - (own ? t.p128 : 0) + part * MINE, end = own ? t.o_keys : t.p_keys;
      const PagedTable& table = own ? p.rows.table : p.prefix;
      const int32_t* const row = table.table + static_cast<int64_t>(own ? t.sequence : t.group) * table.ld;
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) {
        const int j = first + (whole_pages ? 16 * lane : lane + 32 * e);
        if (e == 0) n = whole_pages && lane < GROUPS ? min(max(end - j, 0), 16) : 0;
        page[e] = -1;
        if (whole_pages ? e == 0 && n > 0 : j < end) {
          uint32_t index;
          p.cache.page_size.divmod(static_cast<uint32_t>(j), index, place[e]);
          page[e] = row[index];  // (keys end where the table does)
        }
      }
    };
    struct Where {
      int64_t off[PER_LANE];  // -1: not there (whole pages: see n)
      int n, head;
    };
    auto where = [&](const PagedTensor& c) {
      Where w;
#pragma unroll
      for (int e = 0; e < PER_LANE; ++e) w.off[e] = page[e] >= 0 ? page[e] * c.page + place[e] * c.token : (whole_pages ? 0 : -1);
      w.n = n;
      w.head = t.head;
      return w;
    };
    auto copy = [&](uint64_t* full, uint32_t dst, const PagedTensor& c, const Where& w) {
      const __nv_bfloat16* const base = c.p + w.head * c.head + piece * 8;
      if (whole_pages) {
        const int64_t step = KEYS * c.token;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int in = __shfl_sync(ALL, w.n, g);
          const __nv_bfloat16* src = base + __shfl_sync(ALL, w.off[0], g) + sub * c.token;
          if (in == 16) {
#pragma unroll
            for (int i = 0; i < 16 / KEYS; ++i) {
              cp_async16(dst + g * 2048 + i * (KEYS * 128) + (swz ^ (((i * KEYS) & 7) << 4)), src);
              src += step;
            }
          } else {
#pragma unroll 1
            for (int i = 0; i < 16 / KEYS; ++i) {
              const bool there = i * KEYS + sub < in;
              cp_async16(dst + g * 2048 + i * (KEYS * 128) + (swz ^ (((i * KEYS) & 7) << 4)), there ? src : base, there);
              src += step;
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) {
#pragma unroll 1
          for (int i = 0; i < 32 / KEYS; ++i) {
            const int64_t o = __shfl_sync(ALL, w.off[e], i * KEYS + sub);
            cp_async16(dst + e * 4096 + i * (KEYS * 128) + (swz ^ (((i * KEYS) & 7) << 4)), base + (o < 0 ? 0 : o), o >= 0);
          }
        }
      }
      cp_async_arrive(full);
    };
    const uint32_t k_at = smem_u32(k_ring) + stream * NK * Shape::kTile + at, v_at = smem_u32(v_ring) + stream * NV * Shape::kTile + at;
    // K of tile m, then V of the tile before (PAIRED: its stage is free later than that of the next K) or of the same
    auto load_v = [&](int m, const Where& w) {
      const int vs = m % NV;
      ok = __all_sync(ALL, mbar_wait(&bar.v_empty[stream][vs], (m / NV + 1) & 1, p.status, 53));
      if (ok) copy(&bar.v_full[stream][vs], v_at + vs * Shape::kTile, p.cache.v, w);
    };
    Items items;
    Where v_due;
    int first = 0;   // tile of the stream that the item begins with
    while (ok) {
      ok = next_item(stream, items, t);
      if (!ok || t.tiles == 0) break;
      int tile = (rank - first % TEAM + TEAM) % TEAM;  // this warp's are tiles rank, rank + TEAM, ... of the stream
      if (tile < t.tiles) look_up(tile);
      for (; ok && tile < t.tiles; tile += TEAM) {
        const int m = first + tile, ks = m % NK;
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e)
          if (page[e] >= p.cache.pages) page[e] = -1;
        if (page[0] < 0) n = 0;
        const Where k_where = where(p.cache.k), v_where = where(p.cache.v);
        // which keys are there, in a word per lane (whole pages: 16 keys, else 32)
        uint32_t there[PER_LANE];
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) there[e] = whole_pages ? low_bits(n) : __ballot_sync(ALL, page[e] >= 0);
        if (tile + TEAM < t.tiles) look_up(tile + TEAM);
        // (the m-th tile is the m / stages-th use of its stage)
        ok = __all_sync(ALL, mbar_wait(&bar.k_empty[stream][ks], (m / NK + 1) & 1, p.status, 40));
        if (!ok) break;
        copy(&bar.k_full[stream][ks], k_at + ks * Shape::kTile, p.cache.k, k_where);
        // (the softmax has read the mask PT_MASKS tiles of the stream before this one: PT_MASKS is more than NK + the tiles of a slot whose S is
        // issued and whose P is not read)
        uint16_t* const mask = bar.mask[stream][m % PT_MASKS] + part * (MINE / 16);
        if (whole_pages) {
          if (lane < GROUPS) mask[lane] = static_cast<uint16_t>(there[0]);
        } else if (lane == 0) {
#pragma unroll
          for (int e = 0; e < PER_LANE; ++e) reinterpret_cast<uint32_t*>(mask)[e] = there[e];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.mask_full[stream][m % PT_MASKS]);
        if (!PAIRED) load_v(m, v_where);
        else if (m > 0) load_v(m - 1, v_due);
        v_due = v_where;
      }
      first += t.tiles;
    }
    if (PAIRED && ok && first > 0) load_v(first - 1, v_due);
    cp_async_wait_all();
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(256 - SOFTMAX_REGS));
    if (warp == 12 || (warp == 15 && !PAIRED)) {
      // =========================== MMA issuers ===========================
      const bool leader = elect_one();
      const int slot = warp == 12 ? 0 : 1;
      // Descriptors: the low word is the shared address >> 4 and, for V (MN-major), the distance of its panels of 64 columns above bit 16; the
      // high word has the distance of 8-row groups, version and swizzle.  Low words come out of a shuffle, so that the compiler knows
      // them to be the same in all lanes and forms the descriptors in uniform registers.
      const uint32_t idesc_s = idesc_bf16(128, BN, false), idesc_o = idesc_bf16(128, D, true);
      const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
      auto desc = [&](uint32_t lo) { return (static_cast<uint64_t>(desc_hi) << 32) | lo; };
      const uint32_t q_lo = smem_u32(q_s) >> 4, k_lo = smem_u32(k_ring) >> 4, v_lo = smem_u32(v_ring) >> 4;
      bool ok = true;
      // (the copies are writes of the generic proxy: the fence orders them before the products that read them)
      auto landed = [&](uint64_t* full, int stage, int phase) {
        const bool there = __all_sync(ALL, mbar_wait_spin(&full[stage], phase & 1, p.status, 42));
        if (leader) fence_proxy_async_smem();
        return there;
      };
      auto issue_s = [&](int slot, int buffer, int stage) {
        const uint32_t qa = __shfl_sync(ALL, q_lo + slot * (Shape::kQ >> 4), 0);
        const uint32_t kt = __shfl_sync(ALL, k_lo + stage * (Shape::kTile >> 4), 0), ts = __shfl_sync(ALL, tmem_base + slot * PT_TM_SLOT + buffer * BN, 0);
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_bf16_ss(ts, desc(qa + (i >> 2) * (PT_Q_PANEL >> 4) + (i & 3) * 2), desc(kt + (i >> 2) * (Shape::kPanel >> 4) + (i & 3) * 2), idesc_s, i != 0);
          tc_commit(&bar.s_full[slot][buffer]);
        }
      };
      auto issue_o = [&](int slot, int buffer, int stage, bool first, int from, int to) {  // P of these 16s of keys is there
        const uint32_t vt = __shfl_sync(ALL, v_lo + stage * (Shape::kTile >> 4), 0) | (static_cast<uint32_t>(Shape::kPanel >> 4) << 16);
        const uint32_t tm = __shfl_sync(ALL, tmem_base + slot * PT_TM_SLOT, 0), ps = __shfl_sync(ALL, tm + buffer * BN, 0);
        tc_fence_after();
        if (leader) {
#pragma unroll
          for (int i = from; i < to; ++i)  // 16 keys are two groups of eight rows
            mma_bf16_ts(tm + PT_TM_O, ps + i * 8, desc(vt + i * ((16 * 128) >> 4)), idesc_o, !(first && i == 0));
        }
      };
      Items items;
      TileItem t;
      uint32_t q_phase = 0;
      auto wait_q = [&](int i) {
        const bool there = __all_sync(ALL, mbar_wait_spin(&bar.q_full[i], q_phase, p.status, 41));
        q_phase ^= 1;
        if (leader) fence_proxy_async_smem();
        return there;
      };
      if (PAIRED) {
        // Step x: P V of tile x and S of tile x + 1, slot by slot.
        int x = -1, ks = 0, vs = 0;
        uint32_t k_phase = 0, v_phase = 0, p_phase = 0;  // p_phase: a bit per slot
        bool has[2] = {false, false}, fresh = false, last[2] = {false, false};  // of tile x: which slots take it, first and last of the item
        auto take_p = [&](int s, int stage, bool first) {
          const uint32_t phase = (p_phase >> s) & 1;
          p_phase ^= 1u << s;
          constexpr int FIRST = Shape::kHalves ? BN / 32 : 0;
          bool there = true;
          if (Shape::kHalves) {
            there = __all_sync(ALL, mbar_wait_spin(&bar.p_half[s], phase, p.status, 56));
            if (there) issue_o(s, 0, stage, first, 0, FIRST);
          }
          there = there && __all_sync(ALL, mbar_wait_spin(&bar.p_full[s][0], phase, p.status, 43));
          if (there) issue_o(s, 0, stage, first, FIRST, BN / 16);
          return there;
        };
        auto step = [&](bool more, bool has0, bool has1, bool first, bool last0, bool last1, bool end) {  // tile x + 1: whether there is one, ...
          if (x >= 0) ok = landed(bar.v_full[0], vs, v_phase);
          if (ok && has[0]) {
            ok = take_p(0, vs, fresh);
            if (ok && last[0] && leader) tc_commit(&bar.pv_done[0][0]);
          }
          if (ok && first) ok = wait_q(0);
          if (ok && more) ok = landed(bar.k_full[0], ks, k_phase);
          if (ok && has0) issue_s(0, 0, ks);
          if (ok && has[1]) {
            ok = take_p(1, vs, fresh);
            if (ok && last[1] && leader) tc_commit(&bar.pv_done[1][0]);
          }
          if (!ok) return;
          if (has1) issue_s(1, 0, ks);
          if (leader) {
            if (x >= 0) tc_commit(&bar.v_empty[0][vs]);
            if (more) tc_commit(&bar.k_empty[0][ks]);
            if (end) tc_commit(&bar.q_empty[0]);
          }
          if (x >= 0 && ++vs == NV) { vs = 0; v_phase ^= 1; }
          if (++ks == NK) { ks = 0; k_phase ^= 1; }
          ++x;
          has[0] = has0; has[1] = has1; fresh = first; last[0] = last0; last[1] = last1;
        };
        while (ok) {
          ok = next_item(0, items, t);
          if (!ok || t.tiles == 0) break;
          for (int j = 0; ok && j < t.tiles; ++j) step(true, j < t.n[0], j < t.n[1], j == 0, j + 1 == t.n[0], j + 1 == t.n[1], j + 1 == t.tiles);
        }
        if (ok && x >= 0) step(false, false, false, false, false, false, false);
      } else {
        // Up to two S ahead of P V.
        int left = 0, open = 0;        // tiles of the item whose S is to come; tiles whose P V is to come
        int ks = 0, vs = 0;
        uint32_t k_phase = 0, v_phase = 0, s_buffer = 0, o_buffer = 0, p_phase = 0, firsts = 0;  // firsts: a bit per open tile: first of its item
        bool first = false;
        while (ok) {
          if (left == 0 && open == 0) {
            ok = next_item(slot, items, t);
            if (!ok || t.tiles == 0) break;
            left = t.tiles;
            first = true;
          }
          if (left > 0 && open < NB) {
            ok = (!first || wait_q(slot)) && landed(bar.k_full[slot], ks, k_phase);
            if (!ok) break;
            issue_s(slot, s_buffer, slot * NK + ks);
            s_buffer ^= 1;
            --left;
            if (leader) {
              tc_commit(&bar.k_empty[slot][ks]);
              if (left == 0) tc_commit(&bar.q_empty[slot]);
            }
            if (++ks == NK) { ks = 0; k_phase ^= 1; }
            firsts |= (first ? 1u : 0u) << open;
            ++open;
            first = false;
            continue;
          }
          ok = landed(bar.v_full[slot], vs, v_phase) && __all_sync(ALL, mbar_wait_spin(&bar.p_full[slot][o_buffer], (p_phase >> o_buffer) & 1, p.status, 43));
          if (!ok) break;
          p_phase ^= 1u << o_buffer;
          issue_o(slot, o_buffer, slot * NV + vs, (firsts & 1) != 0, 0, BN / 16);
          if (leader) {
            tc_commit(&bar.pv_done[slot][o_buffer]);
            tc_commit(&bar.v_empty[slot][vs]);
          }
          if (++vs == NV) { vs = 0; v_phase ^= 1; }
          o_buffer ^= 1;
          firsts >>= 1;
          --open;
        }
      }
    } else if (warp < 15) {
      // =========================== items and queries ===========================
      const int slot = warp - 13, stream = PAIRED ? 0 : slot;
      constexpr int LANES = D / 8, ROWS = 32 / LANES;
      const int piece = lane % LANES, sub = lane / LANES;
      uint32_t q_phase = 0;
      bool ok = true;
      // The queries of the slot's rows [rho0, rho0 + 128) of `rows`, by whole warps of them: rows that do not exist are zeros.
      auto load_q = [&](int row0, int rows, int rho0, int head) {
        ok = __all_sync(ALL, mbar_wait(&bar.q_empty[stream], q_phase ^ 1, p.status, 50));
        if (!ok) return;
        q_phase ^= 1;
        const int n_rows = min((rows - rho0 + 31) / 32 * 32, kSlotRows);
        const uint32_t dst = smem_u32(q_s) + slot * Shape::kQ + (piece >> 3) * PT_Q_PANEL;
        const __nv_bfloat16* const src = p.q + row0 * p.q_row + head * static_cast<int64_t>(p.per_kv.d) * p.q_head + piece * 8;
#pragma unroll 4
        for (int r = sub; r < n_rows; r += ROWS) {
          const bool there = rho0 + r < rows;
          uint32_t tok, hq;
          p.per_kv.divmod(static_cast<uint32_t>(there ? rho0 + r : 0), tok, hq);
          cp_async16(dst + r * 128 + (((piece & 7) ^ (r & 7)) << 4), src + tok * p.q_row + hq * p.q_head, there);
        }
        cp_async_arrive(&bar.q_full[stream]);
      };
      if (PAIRED && slot == 1) {  // the second slot's
        Items items;
        TileItem t;
        while (ok) {
          ok = next_item(stream, items, t);
          if (!ok || t.tiles == 0) break;
          load_q(t.row0, t.rows, t.rho0 + kSlotRows, t.head);
        }
        cp_async_wait_all();
      } else {
        const uint32_t n_streams = gridDim.x * STREAMS, first = blockIdx.x * STREAMS + static_cast<uint32_t>(stream);
        int at = 0;
        uint32_t phase = 0;
        auto hand_out = [&](const TileItem& t, bool writer) {
          ok = __all_sync(ALL, mbar_wait(&bar.item_empty[stream][at], phase ^ 1, p.status, 49));
          if (!ok) return;
          if (writer) bar.item[stream][at] = t;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.item_full[stream][at]);
          if (++at == PT_ITEMS) { at = 0; phase ^= 1; }
        };
        // A stream has an item of every round, in turn from both ends of it: with causal rows the later tiles have more keys.  (The host saw to
        // it that items are below 2^31.)
        constexpr int TM = PAIRED ? 2 * kSlotRows : kSlotRows;
        SpanTiles st0{}, st1{};
        uint32_t items0 = 0, items = 0;  // of the first span, of both
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {  // (one copy of the code: what is fetched for the first time counts here)
          st0 = st1;
          items0 = items;
          st1 = count_tiles<TM>(p, tp.span[e]);
          items += static_cast<uint32_t>(st1.tiles * tp.span[e].chunks * p.kv_heads);
        }
#pragma unroll 1
        for (uint32_t n0 = 0, odd = 0; n0 < items && ok; n0 += n_streams, odd ^= 1) {
          const uint32_t n = n0 + (odd ? n_streams - 1 - first : first);
          if (n >= items) continue;
          const bool second = n >= items0;
          TileItem t;
          if (!find_tile_item<PAIRED, BN>(p, tp.span[second], second ? st1 : st0, second ? n - items0 : n, t)) continue;
          hand_out(t, lane == 0);
          if (ok) load_q(t.row0, t.rows, t.rho0, t.head);
        }
        TileItem end;
        end.tiles = 0;
        if (ok) hand_out(end, lane == 0);
        cp_async_wait_all();
      }
    }
  } else {
    // =========================== softmax: a row per thread ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
    constexpr int W = BN / 32;              // words of a row's mask, pieces of 32 keys
    const int slot = warp >> 2, quad = warp & 3, stream = PAIRED ? 0 : slot;
    const uint32_t tm = tmem_base + slot * PT_TM_SLOT + (static_cast<uint32_t>(quad * 32) << 16);
    const float NEG_INF = __int_as_float(0xff800000);
    Items items;
    TileItem t;
    int masks = 0;                          // tiles of the stream up to this item
    uint32_t units = 0, mine_done = 0;      // tiles of the slot so far: unit n has buffer n % NB, phase n / NB; its items so far
    bool ok = true;
    while (true) {
      ok = next_item(stream, items, t);
      if (!ok || t.tiles == 0) break;
      const int rho = t.rho0 + (PAIRED ? slot * kSlotRows : 0) + quad * 32 + lane;
      uint32_t tok, hq;
      p.per_kv.divmod(static_cast<uint32_t>(rho), tok, hq);
      const bool there = rho < t.rows;
      const bool idle = rho - lane >= t.rows;  // a warp without rows: whatever its P holds stays in its own rows of O
      const int limit = there ? own_keys(p, t.length, static_cast<int>(tok)) : t.o_keys;
      const int warp_limit = __shfl_sync(ALL, limit, 0);  // limits ascend with the rows
      float factor = p.scale2, m_ref = NEG_INF, l = 0.0f;
      float o_apart[D];    // O behind the tile before, where that was formed apart (in local memory)
      bool apart = false;
      const int mine = PAIRED ? (slot ? t.n[1] : t.n[0]) : t.tiles;
      // One tile.  LATE: it has own tokens that rows of the warp see and others do not.
      auto do_tile = [&](auto late, int u) {
        constexpr bool LATE = decltype(late)::value;
        const uint32_t buffer = units % NB, parity = (units / NB) & 1;
        const uint32_t tb = tm + buffer * BN;
        if (idle) {
          ok = __all_sync(ALL, mbar_wait(&bar.s_full[slot][buffer], parity, p.status, 47));
          if (ok && lane == 0) {
            if (Shape::kHalves) mbar_arrive(&bar.p_half[slot]);
            mbar_arrive(&bar.p_full[slot][buffer]);
          }
          return;
        }
        // which keys of the tile this row sees: as a rule all of them
        const int mk = masks + u;
        const bool marked = mbar_wait(&bar.mask_full[stream][mk % PT_MASKS], (mk / PT_MASKS) & 1, p.status, 44);
        const uint32_t* const words = reinterpret_cast<const uint32_t*>(bar.mask[stream][mk % PT_MASKS]);
        const int v = t.v0 + u * BN;
        uint32_t seen[W], both = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          seen[i] = words[i];
          both &= seen[i];
        }
        bool masked = both != 0xffffffffu;
        if (LATE) {
          masked = true;
#pragma unroll
          for (int i = 0; i < W; ++i) seen[i] &= low_bits(limit - (v - t.p128) - 32 * i);
        }
        const bool formed = mbar_wait(&bar.s_full[slot][buffer], parity, p.status, 45);
        ok = __all_sync(ALL, marked && formed);
        if (!ok) return;
        tc_fence_after();
        uint32_t sc[W][32];
        float m4[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
        auto largest = [&](int i) {
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((seen[i] >> e) & 1)) sc[i][e] = 0xff800000u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) m4[(e >> 1) & 3] = max3(m4[(e >> 1) & 3], __uint_as_float(sc[i][e]), __uint_as_float(sc[i][e + 1]));
        };
        tc_ld_32x32b_x32(tb, sc[0]);
        if (W == 4) tc_ld_32x32b_x32(tb + 32, sc[1]);
        tc_wait_ld();
#pragma unroll
        for (int i = W / 2; i < W; ++i) tc_ld_32x32b_x32(tb + 32 * i, sc[i]);
#pragma unroll
        for (int i = 0; i < W / 2; ++i) largest(i);
        tc_wait_ld();
#pragma unroll
        for (int i = W / 2; i < W; ++i) largest(i);
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const float m_tile = mx * factor;
        const bool moves = m_tile > m_ref + 8.0f;
        // P V of the tile before has to be complete before O is touched (with one buffer this tile's S was issued behind it)
        auto o_is_there = [&] {
          if (NB > 1) ok = __all_sync(ALL, mbar_wait(&bar.pv_done[slot][(units - 1) % NB], ((units - 1) / NB) & 1, p.status, 46));
          tc_fence_after();
          return ok;
        };
        if (__any_sync(ALL, moves || (LATE && apart))) {
          float alpha = 1.0f;
          if (moves) {
            const float before = in_log2(m_ref, factor, p.scale2);
            factor = p.scale2;
            m_ref = mx * factor;
            alpha = ex2(before - m_ref);  // 0 for -inf
            if (fabsf(m_ref) >= PT_LARGE) {
              factor = without_mantissa(factor);
              m_ref = mx * factor;
            }
          }
          l *= alpha;
          if (u > 0) {
            if (!o_is_there()) return;
            if (LATE && apart) put_back<D>(o_apart, tm + PT_TM_O);
            if (LATE) apart = false;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              uint32_t o[16];
              tc_ld_x16(tm + PT_TM_O + 16 * i, o);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tc_st_x16(tm + PT_TM_O + 16 * i, o);
            }
          }
        }
        const float ref = m_ref == NEG_INF ? 0.0f : m_ref;
        const uint64_t k2 = pack_f32x2(factor, factor), n2 = pack_f32x2(-ref, -ref);
        uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
        for (int i = 0; i < W; ++i) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sc[i][e]), __uint_as_float(sc[i][e + 1])), k2, n2), x0, x1);
            x0 = ex2(x0);
            x1 = ex2(x1);
            sum[(e >> 1) & 1] = add_f32x2(sum[(e >> 1) & 1], pack_f32x2(x0, x1));
            pk[e >> 1] = pack_bf16(x0, x1);
          }
          tc_st_x16(tb + 16 * i, pk);  // over S, which is in registers
          if (Shape::kHalves && !LATE && i == W / 2 - 1) {
            tc_wait_st_all();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.p_half[slot]);
          }
        }
        float a0, a1, b0, b1;
        unpack_f32x2(sum[0], a0, a1);
        unpack_f32x2(sum[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
        tc_wait_st_all();
        if (LATE) {
          ok = __all_sync(ALL, mbar_wait(&bar.v_full[stream][mk % NV], (mk / NV) & 1, p.status, 54));
          if (!ok) return;
          const uint8_t* const values = v_ring + (stream * NV + mk % NV) * Shape::kTile;
          if (values_not_finite<D, Shape::kPanel>(values, max(warp_limit - (v - t.p128), 0), min(t.o_keys - (v - t.p128), BN))) {
            if (u > 0 && !o_is_there()) return;
            add_tile_apart<D, BN>(o_apart, tm + PT_TM_O, tb, u == 0, words, limit - (v - t.p128), values);
            apart = true;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (Shape::kHalves && LATE) mbar_arrive(&bar.p_half[slot]);
          mbar_arrive(&bar.p_full[slot][buffer]);
        }
      };
      // the late tiles begin with the one that has the first own token that the first row does not see
      const int first_late = warp_limit >= t.o_keys ? mine : min(max(t.p128 + warp_limit - t.v0, 0) / BN, mine);
      // A slot that took none of the last tiles may be far ahead of the loaders, where the phase of a mask says nothing yet: its first S tells
      // that they have come here.
      if (PAIRED && mine > 0 && !idle) ok = __all_sync(ALL, mbar_wait(&bar.s_full[slot][units % NB], (units / NB) & 1, p.status, 55));
      int u = 0;
      for (; ok && u < first_late; ++u, ++units) do_tile(std::false_type{}, u);
      for (; ok && u < mine; ++u, ++units) do_tile(std::true_type{}, u);
      masks += t.tiles;
      if (!ok) break;
      if (mine == 0) continue;
      // P V of the last tile (PAIRED: said of that one only)
      ok = __all_sync(ALL, mbar_wait(&bar.pv_done[slot][(units - 1) % NB], (PAIRED ? mine_done : (units - 1) / NB) & 1, p.status, 46));
      if (!ok) break;
      ++mine_done;
      if (idle) continue;
      tc_fence_after();
      if (apart) put_back<D>(o_apart, tm + PT_TM_O);
      const int64_t row = t.row0 + static_cast<int>(tok), qh = t.head * static_cast<int64_t>(p.per_kv.d) + hq;
      if (t.part >= 0) {
        const int64_t at = (static_cast<int64_t>(t.part) * p.rows.rows + row) * p.q_heads + qh;
        if (there) p.part_ml[at] = make_float2(in_log2(m_ref, factor, p.scale2), l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tc_ld_32x32b_x32(tm + PT_TM_O + 32 * i, o);
          tc_wait_ld();
          if (there) {
#pragma unroll
            for (int e = 0; e < 4; ++e) store32(p.part_o + at * D + 32 * i + 8 * e, &o[8 * e]);
          }
        }
      } else {
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        __nv_bfloat16* const dst = p.out + row * p.o_row + qh * p.o_head;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tc_ld_32x32b_x32(tm + PT_TM_O + 32 * i, o);
          tc_wait_ld();
          if (there) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // (rows of `out` are 16-byte aligned)
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[k] = pack_bf16(__uint_as_float(o[8 * e + 2 * k]) * inv, __uint_as_float(o[8 * e + 2 * k + 1]) * inv);
              reinterpret_cast<uint4*>(dst + 32 * i)[e] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem_base, PT_TM_COLS);
  }
}

template <int D, bool PAIRED>
int launch(const TilesParams& tp, int64_t items, cudaStream_t st) {  // `items`: at most
  int dev = 0;
  VX_CUDA_OK(cudaGetDevice(&dev));
  static std::atomic<uint64_t> attr_done{0};
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !(attr_done.load(std::memory_order_acquire) & (1ull << dev))) {
    VX_CUDA_OK(cudaFuncSetAttribute(prefix_tiles_kernel<D, PAIRED>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileShape<D, PAIRED>::kSmem));
    if (cached) attr_done.fetch_or(1ull << dev, std::memory_order_release);
  }
  const int64_t ctas = PAIRED ? items : (items + 1) / 2;
  VX_CUDA_OK(launch_dependent(prefix_tiles_kernel<D, PAIRED>, dim3(static_cast<unsigned>(ctas < sm_count() ? ctas : sm_count())), dim3(PT_THREADS),
                              TileShape<D, PAIRED>::kSmem, st, tp));
  return 0;
}

}  // namespace

int launch_prefix_tiles(const PrefixParams& p, int head_dim, bool paired, const Span& a, const Span& b, void* stream) {
  const TilesParams tp{p, {a, b}};
  const int64_t first = static_cast<int64_t>(a.slots) * a.chunks * p.kv_heads;
  const int64_t items = first + static_cast<int64_t>(b.slots) * b.chunks * p.kv_heads;
  if (items >= (1ll << 31)) return fail(-1, "too much work for one call (%lld items)", (long long)items);
  const auto st = static_cast<cudaStream_t>(stream);
  if (head_dim == 64) return paired ? launch<64, true>(tp, items, st) : launch<64, false>(tp, items, st);
  return paired ? launch<128, true>(tp, items, st) : launch<128, false>(tp, items, st);
}

}  // namespace vx
