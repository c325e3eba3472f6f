// Attention over shared prefixes and own tokens for many rows per owner and key head, on the 5th-generation tensor cores (the cut of the
// work: vx_prefix.cuh; few rows: vx_prefix_attn.cu).
//
// A CTA takes up to 256 rows of one owner and key head against one chunk of keys, in tiles of 128 keys, as two SLOTS of 128 rows with
// tensor memory of their own: S = Q K^T (128 x 128, fp32), P (bf16, over S) and O (128 x head_dim).  While the softmax of one slot works, the
// tensor cores have the products of the other.  With 128 rows or fewer both slots hold the same rows and take the key tiles in turn; their
// two results are joined through shared memory at the end.
//   warps 0..3, 4..7  softmax of slot 0, 1: a query row per thread straight out of tensor memory
//   warps 8..11       loaders: 32 keys of every tile each, page by page (cp.async, 16 bytes; keys that are not there are filled with zeros
//                     and marked in a word per 32 keys)
//   warp 12           MMA issuer
// Q, K and V lie in shared memory in rows of 128 bytes with the 128-byte swizzle, 64 columns a panel; V is read as an MN-major operand.
// P is the A operand in tensor memory, so that shared memory is read for K, Q and V only.
// The reference maximum of a row moves only when a tile's maximum exceeds it by more than 8 in units of log2 (probabilities stay below
// 2^8); then the row's sum and its O are scaled before P is handed over.
// Every wait on a barrier is bounded.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "vx_common.cuh"
#include "vx_prefix.cuh"
#include "vx_ptx.cuh"
#include "vx_quant_math.cuh"

namespace vx {
namespace {

constexpr int PT_BN = 128;                 // keys per tile
constexpr int PT_PANEL = 128 * 128;        // 128 rows of 64 bf16
constexpr int PT_THREADS = 16 * 32;         // (warps 13..15 only fill the fourth warpgroup)
constexpr int PT_MASKS = 8;                // tiles whose masks are kept
constexpr uint32_t PT_TM_SLOT = 256, PT_TM_O = 128, PT_TM_COLS = 512;

template <int D>
struct TileShape {
  static constexpr int kPanels = D / 64;
  static constexpr int kTile = kPanels * PT_PANEL;   // bytes of a K or V tile and of a slot's Q
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kSmem = (2 + kStages) * kTile + 1024;
};

struct TilesParams {
  PrefixParams p;
  Span span[2];
  int32_t first_items;
};

template <int NS>
struct TileBarriers {
  uint64_t q_full, full[NS], empty[NS], s_full[2], p_full[2], o_full[2], mask_full[PT_MASKS];
  uint32_t mask[PT_MASKS][4];
  uint32_t tmem_base;
  float2 ml[128];  // slot 1's, joined by slot 0
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
// bits [0, n) of a word
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1); }

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1) prefix_tiles_kernel(const __grid_constant__ TilesParams tp) {
  using Shape = TileShape<D>;
  constexpr int NS = Shape::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const q_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* const ring = q_s + 2 * Shape::kTile;
  __shared__ TileBarriers<NS> bar;
  const PrefixParams& p = tp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_wait();
  pdl_launch_dependents();
  int n = static_cast<int>(blockIdx.x);
  const bool second = n >= tp.first_items;
  if (second) n -= tp.first_items;
  const Span& sp = tp.span[second];
  const int head = n % p.kv_heads;
  n /= p.kv_heads;
  const int chunk = n / sp.slots;
  Item it;
  if (!find_item<kTileRows>(p, sp, n - chunk * sp.slots, chunk, it)) return;
  const bool dual = it.rows - it.rho0 > 128;
  // key tiles: of the CTA and of its slots
  const int tiles = (it.keys - it.key0 + PT_BN - 1) / PT_BN;
  int n_slot[2];
  if (dual) {
    n_slot[1] = tiles;
    n_slot[0] = tiles;
    if (sp.own) {  // what the last row of slot 0 sees
      const int k0 = min(own_keys(p, it.length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(it.rho0 + 127)))), it.keys) - it.key0;
      n_slot[0] = k0 <= 0 ? 0 : (k0 + PT_BN - 1) / PT_BN;
    }
  } else {
    n_slot[0] = (tiles + 1) >> 1;
    n_slot[1] = tiles >> 1;
  }

  if (threadIdx.x == 0) {
    mbar_init(&bar.q_full, dual ? 8 : 4);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bar.full[s], 128);  // the loaders' threads
      mbar_init(&bar.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar.s_full[s], 1);
      mbar_init(&bar.p_full[s], 4);
      mbar_init(&bar.o_full[s], 1);
    }
    for (int s = 0; s < PT_MASKS; ++s) mbar_init(&bar.mask_full[s], 4);
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
  // Registers: 128 a thread at launch, 512 for a thread of each of the four warpgroups.  The softmax, which holds a row of S, takes 192 in
  // two of them, the other two leave 64 each (2 x 192 + 2 x 64 = 512); every warp of a warpgroup passes the same setmaxnreg.

  if (warp >= 8 && warp < 12) {
    // =========================== loaders ===========================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // Order: K0, K1, V0, K2, V1, ..., V(tiles - 1), each into the next stage of the ring.
    const int w = warp - 8;
    const PagedTable& table = sp.own ? p.rows.table : p.prefix;
    const __nv_bfloat16* const kb = p.cache.k.p + head * p.cache.k.head;
    const __nv_bfloat16* const vb = p.cache.v.p + head * p.cache.v.head;
    constexpr int LANES = D / 8;           // lanes that share a key
    constexpr int KEYS = 32 / LANES;       // keys per instruction
    const int piece = lane % LANES, sub = lane / LANES;
    const uint32_t ring_u = smem_u32(ring) + (piece >> 3) * PT_PANEL;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto load = [&](const __nv_bfloat16* base, int64_t off) {
      ok = __all_sync(0xffffffffu, mbar_wait(&bar.empty[stage], phase ^ 1, p.status, 40));
      if (!ok) return;
      const uint32_t dst = ring_u + stage * Shape::kTile;
#pragma unroll
      for (int i = 0; i < 32 / KEYS; ++i) {
        const int key = i * KEYS + sub;
        const int64_t o = __shfl_sync(0xffffffffu, off, key);
        cp_async16(dst + (w * 32 + key) * 128 + (((piece & 7) ^ (key & 7)) << 4), base + (o < 0 ? 0 : o) + piece * 8, o >= 0);
      }
      cp_async_arrive(&bar.full[stage]);
      if (++stage == NS) { stage = 0; phase ^= 1; }
    };
    int64_t v_prev = -1;  // the tile before
    for (int t = 0; t <= tiles && ok; ++t) {
      int64_t k_off = -1, v_off = -1;
      if (t < tiles) {
        const int j = it.key0 + t * PT_BN + w * 32 + lane;
        if (j < it.keys) {
          uint32_t index, slot;
          p.cache.page_size.divmod(static_cast<uint32_t>(j), index, slot);
          const int page = page_of(table, it.owner, index, p.cache.pages);
          if (page >= 0) {
            k_off = page * p.cache.k.page + slot * p.cache.k.token;
            v_off = page * p.cache.v.page + slot * p.cache.v.token;
          }
        }
        const uint32_t there = __ballot_sync(0xffffffffu, k_off >= 0);
        load(kb, k_off);
        if (!ok) break;
        // (the softmax is done with the tile PT_MASKS before this one: its P was there before the stage just filled was free)
        if (lane == 0) {
          bar.mask[t % PT_MASKS][w] = there;
          mbar_arrive(&bar.mask_full[t % PT_MASKS]);
        }
      }
      if (t > 0) load(vb, v_prev);
      v_prev = v_off;
    }
    cp_async_wait_all();
  } else if (warp >= 12) {
    // =========================== MMA issuer ===========================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 12) {
    const bool leader = elect_one();
    const uint32_t idesc_s = idesc_bf16(128, PT_BN, false), idesc_o = idesc_bf16(128, 64, true);
    const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    auto desc = [&](uint32_t lo) { return (static_cast<uint64_t>(desc_hi) << 32) | lo; };
    const uint32_t q_lo = smem_u32(q_s) >> 4, ring_lo = smem_u32(ring) >> 4;
    bool ok = mbar_wait_spin(&bar.q_full, 0, p.status, 41);
    tc_fence_after();
    auto k_stage = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
    auto v_stage = [&](int j) { return j < tiles - 1 ? 2 * j + 2 : 2 * j + 1; };
    // (the copies are writes of the generic proxy: the fence orders them before the products that read them)
    auto landed = [&](int i) {
      const bool there = mbar_wait_spin(&bar.full[i % NS], (i / NS) & 1, p.status, 42);
      fence_proxy_async_smem();
      return there;
    };
    auto issue_s = [&](int slot, int j) {
      const uint32_t qa = q_lo + (dual ? slot : 0) * (Shape::kTile >> 4), kt = ring_lo + (k_stage(j) % NS) * (Shape::kTile >> 4);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint32_t off = (i >> 2) * (PT_PANEL >> 4) + (i & 3) * 2;
        if (leader) mma_bf16_ss(tmem_base + slot * PT_TM_SLOT, desc(qa + off), desc(kt + off), idesc_s, i != 0);
      }
      if (leader) tc_commit(&bar.s_full[slot]);
    };
    auto issue_o = [&](int slot, int j, bool first) {
      const uint32_t vt = ring_lo + (v_stage(j) % NS) * (Shape::kTile >> 4), tm = tmem_base + slot * PT_TM_SLOT;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int i = 0; i < PT_BN / 16; ++i)
          if (leader) mma_bf16_ts(tm + PT_TM_O + h * 64, tm + i * 8, desc(vt + h * (PT_PANEL >> 4) + i * ((16 * 128) >> 4)), idesc_o, !(first && i == 0));
    };
    auto release = [&](int i) {
      if (leader) tc_commit(&bar.empty[i % NS]);
    };
    if (dual) {
      ok = ok && landed(0);
      if (ok) {
        tc_fence_after();
        if (n_slot[0] > 0) issue_s(0, 0);
        issue_s(1, 0);
        release(0);
      }
      for (int j = 0; j < tiles && ok; ++j) {
        ok = landed(v_stage(j));
        for (int slot = 0; slot < 2 && ok; ++slot) {
          if (j >= n_slot[slot]) continue;
          ok = mbar_wait_spin(&bar.p_full[slot], j & 1, p.status, 43);
          if (!ok) break;
          tc_fence_after();
          issue_o(slot, j, j == 0);
          if (j + 1 < n_slot[slot]) {
            ok = landed(k_stage(j + 1));
            if (!ok) break;
            tc_fence_after();
            issue_s(slot, j + 1);
          } else if (leader) {
            tc_commit(&bar.o_full[slot]);
          }
        }
        release(v_stage(j));
        if (j + 1 < tiles) release(k_stage(j + 1));
      }
    } else {
      for (int j = 0; j < 2 && j < tiles && ok; ++j) {
        ok = landed(k_stage(j));
        if (!ok) break;
        tc_fence_after();
        issue_s(j, j);
        release(k_stage(j));
      }
      for (int j = 0; j < tiles && ok; ++j) {
        const int slot = j & 1;
        ok = landed(v_stage(j)) && mbar_wait_spin(&bar.p_full[slot], (j >> 1) & 1, p.status, 43);
        if (!ok) break;
        tc_fence_after();
        issue_o(slot, j, j < 2);
        release(v_stage(j));
        if (j + 2 < tiles) {
          ok = landed(k_stage(j + 2));
          if (!ok) break;
          tc_fence_after();
          issue_s(slot, j + 2);
          release(k_stage(j + 2));
        } else if (leader) {
          tc_commit(&bar.o_full[slot]);
        }
      }
    }
    }
  } else {
    // =========================== softmax: a row per thread ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int slot = warp >> 2, quad = warp & 3, local = quad * 32 + lane;
    const uint32_t tm = tmem_base + slot * PT_TM_SLOT + (static_cast<uint32_t>(quad * 32) << 16);
    const int rho = it.rho0 + (dual ? slot * 128 : 0) + local;
    uint32_t tok, hq;
    p.per_kv.divmod(static_cast<uint32_t>(rho), tok, hq);
    const bool there = rho < it.rows;
    const int64_t row = it.row0 + static_cast<int>(tok), qh = head * static_cast<int64_t>(p.per_kv.d) + hq;
    if (dual || slot == 0) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (there ? row * p.q_row + qh * p.q_head : 0));
      uint8_t* const dst = q_s + slot * Shape::kTile + local * 128;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (there) u = src[i];
        *reinterpret_cast<uint4*>(dst + (i >> 3) * PT_PANEL + (((i & 7) ^ (local & 7)) << 4)) = u;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.q_full);
    }
    const int limit = there && sp.own ? own_keys(p, it.length, static_cast<int>(tok)) : it.keys;
    const bool idle = rho - lane >= it.rows;  // a warp without rows: whatever its P holds stays in its own rows of O
    const float NEG_INF = __int_as_float(0xff800000);
    float m_ref = NEG_INF, l = 0.0f;
    bool ok = true;
    const int mine = n_slot[slot];
    for (int u = 0; u < mine; ++u) {
      const int t = dual ? u : 2 * u + slot;
      if (idle) {
        ok = __all_sync(0xffffffffu, mbar_wait_spin(&bar.s_full[slot], u & 1, p.status, 47));
        if (!ok) break;
        if (lane == 0) mbar_arrive(&bar.p_full[slot]);
        continue;
      }
      // which keys of the tile this row sees
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&bar.mask_full[t % PT_MASKS], (t / PT_MASKS) & 1, p.status, 44));
      if (!ok) break;
      uint32_t seen[4];
      bool all = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        seen[i] = bar.mask[t % PT_MASKS][i] & low_bits(limit - it.key0 - t * PT_BN - 32 * i);
        all = all && seen[i] == 0xffffffffu;
      }
      const bool masked = __any_sync(0xffffffffu, !all);
      ok = __all_sync(0xffffffffu, mbar_wait_spin(&bar.s_full[slot], u & 1, p.status, 45));
      if (!ok) break;
      tc_fence_after();
      uint32_t sc[4][32];
      tc_ld_32x32b_x32(tm, sc[0]);
      tc_ld_32x32b_x32(tm + 32, sc[1]);
      tc_wait_ld();
      tc_ld_32x32b_x32(tm + 64, sc[2]);
      tc_ld_32x32b_x32(tm + 96, sc[3]);
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
      largest(0);
      largest(1);
      tc_wait_ld();
      largest(2);
      largest(3);
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      const float m_tile = mx * p.scale2;
      const bool moves = m_tile > m_ref + 8.0f;
      if (__any_sync(0xffffffffu, moves)) {
        const float alpha = moves ? ex2(m_ref - m_tile) : 1.0f;  // 0 for m_ref = -inf
        if (moves) m_ref = m_tile;
        l *= alpha;
        if (u > 0) {  // (S of this tile was issued behind P V of the one before: O is complete)
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tc_ld_32x32b_x32(tm + PT_TM_O + 32 * i, o);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tc_st_x16(tm + PT_TM_O + 32 * i, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
            tc_st_x16(tm + PT_TM_O + 32 * i + 16, *reinterpret_cast<uint32_t(*)[16]>(&o[16]));
          }
        }
      }
      const float ref = m_ref == NEG_INF ? 0.0f : m_ref;
      const uint64_t k2 = pack_f32x2(p.scale2, p.scale2), n2 = pack_f32x2(-ref, -ref);
      uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
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
        tc_st_x16(tm + 16 * i, pk);  // over S, which is in registers
      }
      float a0, a1, b0, b1;
      unpack_f32x2(sum[0], a0, a1);
      unpack_f32x2(sum[1], b0, b1);
      l += (a0 + a1) + (b0 + b1);
      tc_wait_st_all();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.p_full[slot]);
    }
    if (ok && mine > 0) ok = __all_sync(0xffffffffu, mbar_wait_spin(&bar.o_full[slot], 0, p.status, 46));
    tc_fence_after();
    const int64_t at = (static_cast<int64_t>(sp.part0 + chunk) * p.rows.rows + row) * p.q_heads + qh;
    if (dual) {
      if (ok && mine > 0) {
        if (there) p.part_ml[at] = make_float2(m_ref, l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tc_ld_32x32b_x32(tm + PT_TM_O + 32 * i, o);
          tc_wait_ld();
          if (there) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              reinterpret_cast<uint4*>(p.part_o + at * D + 32 * i)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
      }
    } else {
      // Slot 1's sums to slot 0 through the shared memory of Q, which every S has been formed of by now (the last of them was issued ahead
      // of slot 1's last P V).  16-byte pieces of a row in an order that depends on the row, so that lanes hit different banks.
      if (slot == 1 && ok && mine > 0) {
        bar.ml[local] = make_float2(m_ref, l);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tc_ld_32x32b_x32(tm + PT_TM_O + 32 * i, o);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(q_s + local * (D * 4) + (((8 * i + e) ^ (local & 7)) << 4)) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        }
      }
      named_bar_sync(1, 256);
      if (slot == 0 && ok) {
        const bool other = n_slot[1] > 0;
        const float2 ml = other ? bar.ml[local] : make_float2(NEG_INF, 0.0f);
        const float m = fmaxf(m_ref, ml.x), ref = m == NEG_INF ? 0.0f : m;
        const float wa = ex2(m_ref - ref), wb = ex2(ml.x - ref);
        if (there) p.part_ml[at] = make_float2(m, wa * l + (other ? wb * ml.y : 0.0f));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          uint32_t o[32];
          tc_ld_32x32b_x32(tm + PT_TM_O + 32 * i, o);
          tc_wait_ld();
          if (there) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float4 x = make_float4(0, 0, 0, 0);
              if (other) x = *reinterpret_cast<const float4*>(q_s + local * (D * 4) + (((8 * i + e) ^ (local & 7)) << 4));
              float4 y;
              y.x = wa * __uint_as_float(o[4 * e]) + wb * x.x;
              y.y = wa * __uint_as_float(o[4 * e + 1]) + wb * x.y;
              y.z = wa * __uint_as_float(o[4 * e + 2]) + wb * x.z;
              y.w = wa * __uint_as_float(o[4 * e + 3]) + wb * x.w;
              reinterpret_cast<float4*>(p.part_o + at * D + 32 * i)[e] = y;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem_base, PT_TM_COLS);
  }
}

template <int D>
int launch(const TilesParams& tp, int64_t items, cudaStream_t st) {
  int dev = 0;
  VX_CUDA_OK(cudaGetDevice(&dev));
  static std::atomic<uint64_t> attr_done{0};
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !(attr_done.load(std::memory_order_acquire) & (1ull << dev))) {
    VX_CUDA_OK(cudaFuncSetAttribute(prefix_tiles_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileShape<D>::kSmem));
    if (cached) attr_done.fetch_or(1ull << dev, std::memory_order_release);
  }
  VX_CUDA_OK(launch_dependent(prefix_tiles_kernel<D>, dim3(static_cast<unsigned>(items)), dim3(PT_THREADS), TileShape<D>::kSmem, st, tp));
  return 0;
}

}  // namespace

int launch_prefix_tiles(const PrefixParams& p, int head_dim, const Span& prefix, const Span& own, void* stream) {
  TilesParams tp{p, {prefix, own}, 0};
  const int64_t first = static_cast<int64_t>(prefix.slots) * prefix.chunks * p.kv_heads;
  const int64_t items = first + static_cast<int64_t>(own.slots) * own.chunks * p.kv_heads;
  if (items >= (1ll << 31)) return fail(-1, "too much work for one call (%lld items)", (long long)items);
  tp.first_items = static_cast<int32_t>(first);
  const auto st = static_cast<cudaStream_t>(stream);
  return head_dim == 64 ? launch<64>(tp, items, st) : launch<128>(tp, items, st);
}

}  // namespace vx
