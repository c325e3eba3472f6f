// Attention of new tokens over a shared prefix and their own tokens in a paged cache:
//
//   out[r, h] = sum_j softmax_j(scale q[r, h] . k_j) v_j
//   keys: tokens [0, prefix_lengths[g]) of the group's pages, own tokens t <= lengths[s] + i of the sequence
//
// How the work is cut: vx_prefix.cuh.  This file has the kernel for few rows per owner and key head, the kernel that joins the parts, and
// the entry points.
//
// prefix_rows_kernel: up to 16 rows against one chunk of keys, by one, two or four of a CTA's four warps; each takes 16 keys in turn through a
// ring of its own in shared memory (cp.async, two or three stages of 16 keys and their values), so that no warp waits for another before the
// end, where their sums are joined.  Keys and values are the m16 side of m16n8k16 products: eight rows fill one, and nothing is computed for
// rows that do not exist.  With lane = 4 g + c:
//   S^T = K Q^T: the order of the terms of a sum over head_dim is free.  A lane reads 16 bytes = 8 values of keys g and g + 8 at 8 (c + 4 i);
//     the registers are the A fragments of two products whose 16 "k" are the values 8 (c + 4 i) + {0, 1, 2, 3} (then {4, ..., 7}) of the
//     four c; Q is read in the same order.
//   O^T += V^T P^T: the accumulators hold P^T by keys; transposed in 8 x 8 blocks (movmatrix) they are the B fragment.  A lane reads 8 values
//     of each of the keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 at 64 b + 8 g and pairs two keys' values with byte permutes; product j of block b has
//     columns 64 b + 8 g + 2 j (rows g of its A) and 64 b + 8 g + 2 j + 1 (rows g + 8).
// (ldmatrix gives the same fragments from rows of 16 bytes; with the reads above the pieces of a key lie in shared memory as they lie in the
// cache.  mma.sync and not tcgen05: its M is 128 rows, of which these calls have 1 to 16.)
// The reference maximum of a row moves only when a score exceeds it by more than 8 (probabilities stay below 2^8), so most steps
// need a vote and no shuffles; sums are kept per lane until the end.
// What bounds it: HBM where there is enough to read -- with the tile kernel, which has the prefixes, and the join, 566 MB of a batch of 149
// sequences over eight prompts take 100 us, 5.7 TB/s -- and else the latency of a CTA and its issue slots: 16 groups of ten hypotheses, 8
// heads of 64, take 6.7 us over 64 frames, 16 over 1,000 and 34 over 3,750 (123 MB, 3.7 TB/s; issue slots 57 % busy).

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "vx_common.cuh"
#include "vx_prefix.cuh"
#include "vx_ptx.cuh"

namespace vx {
namespace {

constexpr int PR_WARPS = 4;

// CTAs of prefix_rows_kernel per SM, as many as its registers allow: what a CTA needs before and behind its keys passes under the others'
// keys.  (16 groups of ten hypotheses, head_dim 64: over 64 frames 8.5 us with 2 or 3, 6.7 with 4, over 1,000 16 with any, over 3,750 37.5, 37.5 and 33.6.)
constexpr int rows_ctas(int blocks, int head_dim) { return head_dim == 64 ? 4 : (blocks == 2 ? 2 : 3); }

struct RowsParams {
  PrefixParams p;
  Span span[2];
  int32_t warps[2];      // of a CTA per item of the span: 1, 2 or 4
  int32_t first_blocks;  // CTAs of span[0]; those of span[1] follow
  int32_t beside;        // the launch in front is the tile kernel of this call, see below
};

__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// 8 x 8 block of 16-bit values, lane 4 g + c holding (g, 2 c) and (g, 2 c + 1): the same of its transpose
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ld_shared16(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// 16 keys and their values per stage of a warp's ring.
template <int D>
struct RowsShape {
  static constexpr int kHalf = 16 * D * 2;                       // bytes of the keys of a stage
  static constexpr int kStages = D == 128 ? 2 : 3;
  static constexpr int kRing = kStages * 2 * kHalf;              // of a warp
  static constexpr int kSmem = PR_WARPS * kRing;
};

// RB blocks of eight rows.
template <int D, int RB>
__global__ void __launch_bounds__(PR_WARPS * 32, rows_ctas(RB, D)) prefix_rows_kernel(const __grid_constant__ RowsParams rp) {
  using Shape = RowsShape<D>;
  constexpr int NS = Shape::kStages;
  constexpr int KC = D / 32;               // 16-byte pieces of a key per lane
  constexpr int VB = D / 64;               // and of a value
  constexpr int TM = 8 * RB;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 ml_s[PR_WARPS][TM];
  __shared__ uint32_t there_s[PR_WARPS][NS];  // bit k: key k of a stage is there
  const PrefixParams& p = rp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  // Beside the tile kernel of the same call: that one lets this launch start only behind its own wait, so everything in front of both is
  // complete, and neither reads what the other writes.  The wait comes at the end then: whoever waits for this kernel waits for both.
  struct Behind {
    const bool last;
    __device__ ~Behind() {
      if (last) pdl_wait();
    }
  } behind{rp.beside != 0};
  if (!rp.beside) pdl_wait();
  pdl_launch_dependents();  // (behind the wait: see the kernel that joins the parts)
  int n = static_cast<int>(blockIdx.x);
  const bool second = n >= rp.first_blocks;
  if (second) n -= rp.first_blocks;
  const Span& sp = rp.span[second];
  const int warps = rp.warps[second], team = warp / warps, rank = warp - team * warps;  // the warps of an item
  n = n * (PR_WARPS / warps) + team;
  const int head = n % p.kv_heads;  // heads of a token lie next to each other
  n /= p.kv_heads;
  const int chunk = n / sp.slots;
  if (chunk >= sp.chunks) return;
  const bool own = sp.kind == kSpanOwn;
  ItemRows it;
  if (!find_rows<TM>(p, sp, n - chunk * sp.slots, it)) return;
  const int length = own ? tokens_before(p, it.owner) : 0;
  // keys [key0, keys): those of the chunk that the tile's last row sees
  int keys = own ? own_keys(p, length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(min(it.rho0 + TM, it.rows) - 1)))) : prefix_keys(p, it.owner);
  if (static_cast<int64_t>(chunk) * sp.chunk >= keys) return;
  const int key0 = chunk * sp.chunk;
  keys = static_cast<int>(min(static_cast<int64_t>(keys), static_cast<int64_t>(key0) + sp.chunk));
  const PagedTable& table = own ? p.rows.table : p.prefix;
  const __nv_bfloat16* const kb = p.cache.k.p + head * p.cache.k.head;
  const __nv_bfloat16* const vb = p.cache.v.p + head * p.cache.v.head;
  const int blocks = it.rows - it.rho0 > 8 ? RB : 1;  // that have rows

  // The ring: the copies of a step are one group, a warp waits for its own.
  const int STEP = 16 * warps;
  constexpr int LANES = D / 8, KEYS = 32 / LANES;  // lanes per key, keys per copy instruction
  const int piece = lane % LANES, sub = lane / LANES;
  const uint32_t ring = smem_u32(smem) + warp * Shape::kRing;
  const bool whole_pages = p.cache.page_size.d % 16 == 0;  // the 16 keys of a step lie on one page
  int j_load = key0 + rank * 16;
  auto fetch = [&](int stage) {  // the next 16 keys of this warp
    const uint32_t dst = ring + stage * 2 * Shape::kHalf;
    // Where they are: the first of them when they lie on one page (the others follow it), else key j_load + lane, handed around below.
    int64_t k_off = -1, v_off = -1;
    {
      const int j = j_load + (whole_pages ? 0 : lane & 15);
      if (j < keys) {
        uint32_t index, slot;
        p.cache.page_size.divmod(static_cast<uint32_t>(j), index, slot);
        const int page = page_of(table, it.owner, index, p.cache.pages);
        if (page >= 0) {
          k_off = page * p.cache.k.page + slot * p.cache.k.token;
          v_off = page * p.cache.v.page + slot * p.cache.v.token;
        }
      }
    }
    uint32_t there;
    if (whole_pages) {
      const int n = k_off >= 0 ? keys - j_load : 0;
      there = n >= 16 ? 0xffffu : (1u << n) - 1;
      const __nv_bfloat16* ka = kb + (n > 0 ? k_off + sub * p.cache.k.token : 0) + piece * 8;
      const __nv_bfloat16* va = vb + (n > 0 ? v_off + sub * p.cache.v.token : 0) + piece * 8;
#pragma unroll
      for (int i = 0; i < 16 / KEYS; ++i) {
        const int key = i * KEYS + sub;
        const bool in = key < n;
        cp_async16(dst + key * (D * 2) + ((piece ^ ((key & 1) << 2)) << 4), in ? ka : kb, in);
        cp_async16(dst + Shape::kHalf + key * (D * 2) + ((piece ^ (((key >> 1) & 3) << 1)) << 4), in ? va : vb, in);
        ka += KEYS * p.cache.k.token;
        va += KEYS * p.cache.v.token;
      }
    } else {
      there = __ballot_sync(0xffffffffu, k_off >= 0) & 0xffffu;
#pragma unroll 1
      for (int i = 0; i < 16 / KEYS; ++i) {
        const int key = i * KEYS + sub;
        const int64_t ko = __shfl_sync(0xffffffffu, k_off, key), vo = __shfl_sync(0xffffffffu, v_off, key);
        cp_async16(dst + key * (D * 2) + ((piece ^ ((key & 1) << 2)) << 4), kb + (ko < 0 ? 0 : ko) + piece * 8, ko >= 0);
        cp_async16(dst + Shape::kHalf + key * (D * 2) + ((piece ^ (((key >> 1) & 3) << 1)) << 4), vb + (vo < 0 ? 0 : vo) + piece * 8, vo >= 0);
      }
    }
    if (lane == 0) there_s[warp][stage] = there;
    j_load += STEP;
  };
#pragma unroll 1
  for (int i = 0; i < NS - 1; ++i) {
    if (j_load < keys) fetch(i);
    cp_async_commit();
  }

  // queries: row 8 r + g, the pieces of this lane
  uint32_t q[RB][KC][4];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int rho = it.rho0 + 8 * r + g;
    uint32_t tok, hq;
    p.per_kv.divmod(static_cast<uint32_t>(rho), tok, hq);
    const __nv_bfloat16* src = p.q + static_cast<int64_t>(it.row0 + static_cast<int>(tok)) * p.q_row + (head * static_cast<int64_t>(p.per_kv.d) + hq) * p.q_head;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (rho < it.rows) u = *reinterpret_cast<const uint4*>(src + 8 * (c + 4 * i));
      q[r][i][0] = u.x; q[r][i][1] = u.y; q[r][i][2] = u.z; q[r][i][3] = u.w;
    }
  }
  // keys that row 8 r + 2 c + e sees; the first row of the tile sees fewest
  int limit[RB][2], min_limit = keys;
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      limit[r][e] = own ? own_keys(p, length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(it.rho0 + 8 * r + 2 * c + e)))) : keys;
  if (own) min_limit = own_keys(p, length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(it.rho0))));

  const float NEG_INF = __int_as_float(0xff800000);
  float m_ref[RB][2], l[RB][2], o[RB][VB][4][4];  // of rows 8 r + 2 c + e
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m_ref[r][0] = m_ref[r][1] = NEG_INF;
    l[r][0] = l[r][1] = 0.0f;
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[r][b][j][0] = o[r][b][j][1] = o[r][b][j][2] = o[r][b][j][3] = 0.0f;
  }

  // where this lane reads its fragments in a stage
  const uint32_t k_at = g * (D * 2) + ((c ^ ((g & 1) << 2)) << 4);                                // keys g, g + 8: pieces c + 4 i
  const uint32_t v_at = Shape::kHalf + 2 * c * (D * 2) + ((g ^ (c << 1)) << 4);                   // keys 2 c + e + 8 f: pieces g + 8 b
  auto step = [&](const uint32_t there, const uint32_t at, const int j0) {
    float s[RB][4];  // [2 b + e]: key 8 b + g, row 8 r + 2 c + e
#pragma unroll
    for (int r = 0; r < RB; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.0f;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      uint32_t k0[4], k1[4];
      ld_shared16(at + (k_at ^ ((i & 1) << 6)) + (i >> 1) * 128, k0);
      ld_shared16(at + (k_at ^ ((i & 1) << 6)) + (i >> 1) * 128 + 8 * (D * 2), k1);
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r < blocks) {
          mma_bf16_16816(s[r], k0[0], k1[0], k0[1], k1[1], q[r][i][0], q[r][i][1]);
          mma_bf16_16816(s[r], k0[2], k1[2], k0[3], k1[3], q[r][i][2], q[r][i][3]);
        }
    }
    const bool late = j0 + 16 > min_limit && min_limit < keys;  // keys that rows of the tile do not see
    // scores in units of log2; keys that are not there or that the row does not see count as -inf
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] *= p.scale2;
    if (j0 + 16 > min_limit || there != 0xffffu) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((there >> (8 * (e >> 1) + g)) & 1) || j0 + 8 * (e >> 1) + g >= limit[r][e & 1]) s[r][e] = NEG_INF;
    }
    bool moves = false;
    float mx[RB][2];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[r][e] = fmaxf(s[r][e], s[r][2 + e]);
        moves = moves || mx[r][e] > m_ref[r][e] + 8.0f;
      }
    if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[r][e] = fmaxf(mx[r][e], __shfl_xor_sync(0xffffffffu, mx[r][e], x));
          const float m_new = fmaxf(m_ref[r][e], mx[r][e]);
          const float alpha = m_new == NEG_INF ? 1.0f : ex2(m_ref[r][e] - m_new);
          m_ref[r][e] = m_new;
          l[r][e] *= alpha;
#pragma unroll
          for (int b = 0; b < VB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[r][b][j][e] *= alpha;
              o[r][b][j][2 + e] *= alpha;
            }
        }
    }
    uint32_t pt[RB][2];  // P^T as B fragments
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const float ref0 = m_ref[r][0] == NEG_INF ? 0.0f : m_ref[r][0], ref1 = m_ref[r][1] == NEG_INF ? 0.0f : m_ref[r][1];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float x0 = ex2(s[r][2 * b] - ref0), x1 = ex2(s[r][2 * b + 1] - ref1);
        l[r][0] += x0;
        l[r][1] += x1;
        pt[r][b] = transpose8x8(pack_bf16(x0, x1));
      }
    }
#pragma unroll
    for (int b = 0; b < VB; ++b) {
      uint32_t v[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) ld_shared16(at + v_at + b * 128 + ((e & 1) + 8 * (e >> 1)) * (D * 2), v[e]);
      if (late) {
        uint32_t sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j) note_not_finite(sum, v[e][j]);
        if (__any_sync(0xffffffffu, any_not_finite(sum))) {
          // Row by row, with zeros for the values of the keys that the row does not see.
#pragma unroll
          for (int r = 0; r < RB; ++r) {
#pragma unroll 1
            for (int n = 0; n < 8; ++n) {
              const int lim0 = __shfl_sync(0xffffffffu, limit[r][0], n >> 1), lim1 = __shfl_sync(0xffffffffu, limit[r][1], n >> 1);
              const int sees = (n & 1 ? lim1 : lim0) - j0 - 2 * c;  // of the keys from 2 c on
              const uint32_t in0 = (sees > 0 ? 0xffffu : 0u) | (sees > 1 ? 0xffff0000u : 0u), in1 = (sees > 8 ? 0xffffu : 0u) | (sees > 9 ? 0xffff0000u : 0u);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_bf16_16816(t, __byte_perm(v[0][j], v[1][j], 0x5410) & in0, __byte_perm(v[0][j], v[1][j], 0x7632) & in0,
                               __byte_perm(v[2][j], v[3][j], 0x5410) & in1, __byte_perm(v[2][j], v[3][j], 0x7632) & in1, pt[r][0], pt[r][1]);
                if (c == n >> 1) {
                  if (n & 1) {
                    o[r][b][j][1] += t[1];
                    o[r][b][j][3] += t[3];
                  } else {
                    o[r][b][j][0] += t[0];
                    o[r][b][j][2] += t[2];
                  }
                }
              }
            }
          }
          continue;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a0 = __byte_perm(v[0][j], v[1][j], 0x5410), a1 = __byte_perm(v[0][j], v[1][j], 0x7632);
        const uint32_t a2 = __byte_perm(v[2][j], v[3][j], 0x5410), a3 = __byte_perm(v[2][j], v[3][j], 0x7632);
#pragma unroll
        for (int r = 0; r < RB; ++r)
          if (r < blocks) mma_bf16_16816(o[r][b][j], a0, a1, a2, a3, pt[r][0], pt[r][1]);
      }
    }
  };
  int stage = 0;
#pragma unroll 1
  for (int j0 = key0 + rank * 16; j0 < keys; j0 += STEP) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    // the stage behind (that of the step before, which every lane has read) is filled again
    if (j_load < keys) fetch(stage == 0 ? NS - 1 : stage - 1);
    cp_async_commit();
    step(there_s[warp][stage], ring + stage * 2 * Shape::kHalf, j0);
    if (++stage == NS) stage = 0;
  }
  named_bar_sync(1 + team, 32 * warps);  // every warp of the item is done with its ring: the sums go there

  // the warps' parts of a row
  constexpr int PITCH = D + 4;
  static_assert(TM * PITCH * 4 <= Shape::kRing, "the sums of a warp fit in its ring");
  float* const o_s = reinterpret_cast<float*>(smem);
  constexpr int OWN = Shape::kRing / 4;
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], x);
      const int lr = 8 * r + 2 * c + e;
      if (g == 0) ml_s[warp][lr] = make_float2(m_ref[r][e], l[r][e]);
#pragma unroll
      for (int b = 0; b < VB; ++b) {  // columns 64 b + 8 g + 2 j + {0, 1}
        float* dst = o_s + warp * OWN + lr * PITCH + 64 * b + 8 * g;
        reinterpret_cast<float4*>(dst)[0] = make_float4(o[r][b][0][e], o[r][b][0][2 + e], o[r][b][1][e], o[r][b][1][2 + e]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(o[r][b][2][e], o[r][b][2][2 + e], o[r][b][3][e], o[r][b][3][2 + e]);
      }
    }
  named_bar_sync(1 + team, 32 * warps);
  constexpr int PIECES = D / 4;
  for (int i = rank * 32 + lane; i < TM * PIECES; i += 32 * warps) {
    const int lr = i / PIECES, col = (i % PIECES) * 4, rho = it.rho0 + lr;
    if (rho >= it.rows) break;
    float m = NEG_INF, sum = 0.0f;
    for (int w = team * warps; w < (team + 1) * warps; ++w) m = fmaxf(m, ml_s[w][lr].x);
    const float ref = m == NEG_INF ? 0.0f : m;
    float4 acc = make_float4(0, 0, 0, 0);
    for (int w = team * warps; w < (team + 1) * warps; ++w) {
      const float a = ex2(ml_s[w][lr].x - ref);
      const float4 x = *reinterpret_cast<const float4*>(o_s + w * OWN + lr * PITCH + col);
      sum += a * ml_s[w][lr].y;
      acc.x += a * x.x; acc.y += a * x.y; acc.z += a * x.z; acc.w += a * x.w;
    }
    uint32_t tok, hq;
    p.per_kv.divmod(static_cast<uint32_t>(rho), tok, hq);
    const int64_t row = it.row0 + static_cast<int>(tok), qh = head * static_cast<int64_t>(p.per_kv.d) + hq;
    const int64_t at = (static_cast<int64_t>(sp.part0 + chunk) * p.rows.rows + row) * p.q_heads + qh;
    if (col == 0) p.part_ml[at] = make_float2(m, sum);
    *reinterpret_cast<float4*>(p.part_o + at * D + col) = acc;
  }
}

template <int D, int RB>
int launch_rows(const RowsParams& rp, int64_t blocks, cudaStream_t st) {
  int dev = 0;
  VX_CUDA_OK(cudaGetDevice(&dev));
  static std::atomic<uint64_t> attr_done{0};
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !(attr_done.load(std::memory_order_acquire) & (1ull << dev))) {
    VX_CUDA_OK(cudaFuncSetAttribute(prefix_rows_kernel<D, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsShape<D>::kSmem));
    if (cached) attr_done.fetch_or(1ull << dev, std::memory_order_release);
  }
  VX_CUDA_OK(launch_dependent(prefix_rows_kernel<D, RB>, dim3(static_cast<unsigned>(blocks)), dim3(PR_WARPS * 32), RowsShape<D>::kSmem, st, rp));
  return 0;
}

// The parts of every row joined, and zeros for the rows that have none.  WARPS warps of a block of eight share a row and query head, a slice of
// the parts each; a warp requests the sums of PARTS parts (at head_dim 64 half a warp has one) together with their maxima, weighs them (maximum,
// then 2^(m_c - m)) and adds them up; shared memory joins the warps.  Many rows of up to four parts, four at a time: fewer
// registers, more rows on an SM (16 utterances with 124 hypotheses of 30 to 60 tokens: a call of 93 us against 103; 32 rows of two parts: 10 against 8).  What a row is, is looked up ahead of the wait: the kernels in front let
// this one start behind a wait of their own, so all that was there before this call is complete.
// What bounds it: one round trip to the parts in L2, or their bytes where rows are many: 64 rows of 32 heads of 128 with 17 parts (18 MB) are done 7 us
// after the kernel in front (a lane that requested one part after the other: 11), 32 rows with 2 parts 2 us.
struct JoinParams {
  PrefixParams p;
  Span span[2];
  int32_t first;  // no kernel of this call is in front
};
constexpr int JN_WARPS = 8;
template <int D, int WARPS, int PARTS>
__global__ void __launch_bounds__(JN_WARPS * 32, PARTS > 4 ? 4 : (D == 64 ? 8 : 5)) prefix_join_kernel(const __grid_constant__ JoinParams jp) {
  pdl_launch_dependents();
  constexpr unsigned ALL = 0xffffffffu;
  constexpr int LANES = D / 4, SUB = 32 / LANES, LOADS = PARTS / SUB;  // lanes per part, parts per load; PARTS at a time
  __shared__ float4 o_s[WARPS > 1 ? JN_WARPS : 1][32];
  __shared__ float2 ml_s[WARPS > 1 ? JN_WARPS : 1];
  const PrefixParams& p = jp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / WARPS, rank = warp % WARPS;
  const int row = static_cast<int>(blockIdx.x), h = static_cast<int>(blockIdx.y) * (JN_WARPS / WARPS) + team;
  if (jp.first) pdl_wait();
  const bool in = h < p.q_heads;
  int parts[2] = {0, 0}, s;
  int64_t i;
  if (row_sequence<true>(p.rows, row, s, i)) {
    const int prefix = prefix_keys(p, group_of(p, s)), own = own_keys(p, p.rows.lengths[s], i);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const Span& sp = jp.span[e];
      const int64_t keys = sp.kind == kSpanPrefix ? prefix : (sp.kind == kSpanOwn ? own : static_cast<int64_t>(align_keys(prefix)) + own);
      if (sp.chunks) parts[e] = static_cast<int>((keys + sp.chunk - 1) / sp.chunk);
    }
  }
  if (!jp.first) pdl_wait();
  // part n of the row: those of span 0, then those of span 1
  const int n_parts = in ? parts[0] + parts[1] : 0, slice = (n_parts + WARPS - 1) / WARPS;
  const int64_t at = static_cast<int64_t>(row) * p.q_heads + h, step = static_cast<int64_t>(p.rows.rows) * p.q_heads;
  auto place = [&](int n) { return at + (n < parts[0] ? jp.span[0].part0 + n : jp.span[1].part0 + n - parts[0]) * step; };
  const float NEG_INF = __int_as_float(0xff800000);
  float m = NEG_INF, sum = 0.0f;
  float4 acc = make_float4(0, 0, 0, 0);
  const int sub = lane / LANES, col = (lane % LANES) * 4, end = min(n_parts, (rank + 1) * slice);
  for (int n0 = rank * slice; n0 < end; n0 += PARTS) {
    float2 ml = make_float2(NEG_INF, 0.0f);
    if (lane < PARTS && n0 + lane < end) ml = p.part_ml[place(n0 + lane)];
    float4 x[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int n = n0 + k * SUB + sub;
      x[k] = make_float4(0, 0, 0, 0);
      if (n < end) x[k] = *reinterpret_cast<const float4*>(p.part_o + place(n) * D + col);
    }
    float mx = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(ALL, mx, o));
    const float m_new = fmaxf(m, mx), ref = m_new == NEG_INF ? 0.0f : m_new, alpha = ex2(m - ref), w = ex2(ml.x - ref);
    m = m_new;
    sum = sum * alpha + w * ml.y;
    acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const float wc = __shfl_sync(ALL, w, k * SUB + sub);  // (0 behind the end)
      acc.x += wc * x[k].x; acc.y += wc * x[k].y; acc.z += wc * x[k].z; acc.w += wc * x[k].w;
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(ALL, sum, x);
  if (SUB == 2) {
    acc.x += __shfl_xor_sync(ALL, acc.x, 16); acc.y += __shfl_xor_sync(ALL, acc.y, 16);
    acc.z += __shfl_xor_sync(ALL, acc.z, 16); acc.w += __shfl_xor_sync(ALL, acc.w, 16);
  }
  if (WARPS > 1) {
    o_s[warp][lane] = acc;
    if (lane == 0) ml_s[warp] = make_float2(m, sum);
    __syncthreads();
    if (rank != 0) return;
    float all = NEG_INF;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all = fmaxf(all, ml_s[warp + w].x);
    const float ref = all == NEG_INF ? 0.0f : all;
    sum = 0.0f;
    acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2(ml_s[warp + w].x - ref);
      const float4 x = o_s[warp + w][lane];
      sum += f * ml_s[warp + w].y;
      acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
  }
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  if (in && sub == 0)
    *reinterpret_cast<uint2*>(p.out + row * p.o_row + h * p.o_head + col) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// Where the tile kernel wrote the rows itself: zeros for those of no sequence, a warp per row.
template <int D>
__global__ void __launch_bounds__(JN_WARPS * 32) prefix_rest_kernel(const __grid_constant__ JoinParams jp) {
  pdl_launch_dependents();
  const PrefixParams& p = jp.p;
  const int row = static_cast<int>(blockIdx.x) * JN_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  int s;
  int64_t i;
  const bool rest = row < p.rows.rows && !row_sequence<true>(p.rows, row, s, i);
  pdl_wait();
  if (!rest) return;
  for (int n = lane; n < p.q_heads * (D / 8); n += 32) *reinterpret_cast<uint4*>(p.out + row * p.o_row + n / (D / 8) * p.o_head + n % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
}

template <int D>
cudaError_t launch_join(const JoinParams& jp, int parts, cudaStream_t st) {
  if (jp.span[0].part0 < 0)
    return launch_dependent(prefix_rest_kernel<D>, dim3(static_cast<unsigned>((jp.p.rows.rows + JN_WARPS - 1) / JN_WARPS)), dim3(JN_WARPS * 32), 0, st, jp);
  // warps per row and head: so many that each has its parts in one turn, while the SMs have room for them
  constexpr int AT_ONCE = D == 64 ? 16 : 8;
  const int64_t cells = static_cast<int64_t>(jp.p.rows.rows) * jp.p.q_heads;
  int warps = 1;
  while (warps < 8 && parts > warps * AT_ONCE && 2 * warps * cells <= 32 * static_cast<int64_t>(sm_count())) warps <<= 1;
  auto kernel = parts <= 4 && cells > 64 * static_cast<int64_t>(sm_count()) ? prefix_join_kernel<D, 1, 4>
                           : (warps == 8 ? prefix_join_kernel<D, 8, AT_ONCE>
                                         : (warps == 4 ? prefix_join_kernel<D, 4, AT_ONCE> : (warps == 2 ? prefix_join_kernel<D, 2, AT_ONCE> : prefix_join_kernel<D, 1, AT_ONCE>)));
  const int per_block = JN_WARPS / warps;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(jp.p.rows.rows), static_cast<unsigned>((jp.p.q_heads + per_block - 1) / per_block)), dim3(JN_WARPS * 32), 0, st, jp);
}

struct Plan {
  Span span[2];
  enum Kernel { kRows, kTiles, kPairs } kernel[2];  // that walks the span
  int blocks;                                       // of eight rows, of the kernel for few rows
  int parts;
  int64_t ml_bytes, bytes;

  Span part(Kernel k, int i) const { return kernel[i] == k ? span[i] : kNoSpan; }  // the span, where kernel k walks it
  bool walks(Kernel k) const { return part(k, 0).chunks > 0 || part(k, 1).chunks > 0; }
};

int64_t round_up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

// Keys per chunk for a span of `items` tiles times key heads.  Short runs are cut into shares of one round of CTAs (`resident`), rounded up to
// a unit, which can make a few more CTAs than the round has places (128 items over 3,584 keys: shares of 774, chunks of 832, 640 CTAs for 592 places); long
// ones into several rounds, since owners differ in length and the last round should cost little.  Each part costs its sums in
// scratch, so no chunk is below `least` keys there.  `capacity` is what the tables have place for, not what lengths (on the device) fill: wide
// tables and a long owner among short ones get chunks that are too long (64 rows over 8,191 keys, 32 heads on 8 of 128: 39 us, with
// a table for 131,072 144; 199 sequences of 100 tokens and one of 100,000: 1.5 ms, 120,000 tokens in equal runs 0.1).
int chunk_keys(int64_t capacity, int64_t items, int64_t resident, int64_t unit, int64_t least, int64_t rounds) {
  const int64_t one_round = (capacity * items + resident - 1) / resident;
  int64_t c = one_round;
  if (one_round > least) {
    const int64_t cuts = (rounds * resident + items - 1) / items;
    c = capacity / cuts > least ? (capacity + cuts - 1) / cuts : least;
  }
  c = round_up(c > unit ? c : unit, unit);
  const int64_t all = round_up(capacity, unit);
  return static_cast<int>(c < all ? c : all);
}

// The same for the tile kernel, whose items are long: the cut that an estimate finds fastest.  `streams` take items one after another, 128 keys
// in `us`, with 4 us for what an item costs besides; `cells` rows and heads leave sums per part, written and read at 4.5 TB/s, where there is
// more than one part (`joint`: or none).  Tried: for each number of turns that the streams take, as many cuts as fill them, and where the keys
// and the parts of a turn cost the same.
int tile_chunk_keys(int64_t capacity, int64_t items, int64_t streams, int64_t unit, double us, int head_dim, int64_t cells, bool joint) {
  const double part_us = static_cast<double>(cells * head_dim) * 8.0 / 4.5e6, walk_us = static_cast<double>(capacity) / 128 * us;
  const int64_t most = (capacity + unit - 1) / unit, turns0 = (items + streams - 1) / streams;
  int64_t best = round_up(capacity, unit);
  double best_us = 1e300;
  auto look_at = [&](int64_t cuts) {
    const int64_t c = cuts < 1 ? 1 : (cuts > most ? most : cuts), chunk = round_up((capacity + c - 1) / c, unit), n = (capacity + chunk - 1) / chunk;
    const double turns = static_cast<double>((items * n + streams - 1) / streams);
    const double all = turns * (static_cast<double>(chunk) / 128 * us + 4.0) + (joint && n == 1 ? 0.0 : static_cast<double>(n) * part_us);
    if (all < best_us) {
      best_us = all;
      best = chunk;
    }
  };
  look_at(1);
  for (int64_t turns = turns0; turns < turns0 + 8; ++turns) {
    const int64_t full = turns * streams / items, even = static_cast<int64_t>(sqrt(static_cast<double>(turns) * walk_us / part_us) + 0.5);
    look_at(full);
    if (even < full) look_at(even);
    if (full >= most) break;
  }
  return static_cast<int>(best);
}

int64_t rows_resident(int blocks, int head_dim) { return static_cast<int64_t>(rows_ctas(blocks, head_dim)) * sm_count(); }

int check_prefix(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d, PrefixParams& p, Plan& plan) {
  const int rc = check_paged(cache, rows, p.cache, p.rows);
  if (rc) return rc;
  if (!d || d->struct_size != static_cast<int32_t>(sizeof(vx_prefix_attention_desc))) return fail(-1, "vx_prefix_attention_desc: struct_size");
  if (d->reserved != 0) return fail(-1, "vx_prefix_attention_desc: reserved must be 0");
  if (cache->head_dim != 64 && cache->head_dim != 128) return fail(-1, "head_dim must be 64 or 128 (got %d)", cache->head_dim);
  if (d->q_heads < 1 || d->q_heads > 65535 || d->q_heads % cache->kv_heads != 0)
    return fail(-1, "q_heads (%d) must be a multiple of kv_heads (%d)", d->q_heads, cache->kv_heads);
  if (d->groups < 0 || d->groups > (1ll << 31) - 1) return fail(-1, "bad number of groups %lld", (long long)d->groups);
  if (rows->rows * d->q_heads + (rows->sequences + d->groups) * cache->kv_heads >= (1ll << 31)) return fail(-1, "rows * q_heads and (sequences + groups) * kv_heads must stay below 2^31 together");
  if (d->groups > 0) {
    if (!d->group_offsets && rows->sequences % d->groups != 0)
      return fail(-1, "without group_offsets the groups are of one size (sequences %lld, groups %lld)", (long long)rows->sequences, (long long)d->groups);
    if (d->prefix_pages < 0 || d->prefix_pages > ((1ll << 31) - 1) / cache->page_size) return fail(-1, "a prefix may have up to 2^31 - 1 tokens");
    if (!d->prefix_lengths || (d->prefix_pages > 0 && (!d->prefix_table || d->ld_prefix < d->prefix_pages)))
      return fail(-1, "prefix_lengths or prefix_table is NULL, or its rows are too short");
  }
  p.scale2 = d->scale * 1.4426950408889634f;
  if (!(d->scale > 0.0f) || !(p.scale2 < INFINITY)) return fail(-1, "scale must be positive and finite, scale log2(e) too");
  const int per = d->q_heads / cache->kv_heads;
  p.q_heads = d->q_heads;
  p.kv_heads = cache->kv_heads;
  p.per_kv = FastDiv(static_cast<uint32_t>(per));
  p.groups = static_cast<int32_t>(d->groups);
  p.group_offsets = d->group_offsets;
  p.group_size = p.groups > 0 && !p.group_offsets ? static_cast<int32_t>(rows->sequences / d->groups) : 0;
  p.prefix = {d->prefix_table, d->ld_prefix, static_cast<int32_t>(d->prefix_pages)};
  p.prefix_lengths = d->prefix_lengths;

  plan = Plan{};
  const int64_t R = rows->rows, S = rows->sequences, G = d->groups;
  plan.span[0] = plan.span[1] = kNoSpan;
  if (R == 0 || S == 0 || cache->pages == 0) return 0;  // no key anywhere
  const int64_t cap_p = G > 0 ? d->prefix_pages * cache->page_size : 0, cap_o = rows->table_pages * cache->page_size;
  if (cap_p + cap_o > (1ll << 31) - 1024) return fail(-1, "prefix and own tokens of a sequence may be 2^31 - 1024 together");  // (indexes of keys are 32 bits)
  // The kernel of a span goes by its rows per owner and key head, on the average, and its keys, as many as the tables have place for (which
  // kernel takes a row changes no result beyond rounding).
  const bool single = !rows->row_offsets;
  const int64_t rows_p = cap_p > 0 ? R * per / G : 0, rows_o = cap_o > 0 ? R * per / S : 0;
  auto cut = [&](Span& sp, SpanKind kind, Plan::Kernel kernel, int64_t owners, int64_t cap, int64_t equal_rows) {
    if (cap <= 0 || owners <= 0) return;
    const int tm = kernel == Plan::kPairs ? 2 * kSlotRows : (kernel == Plan::kTiles ? kSlotRows : 8 * plan.blocks);
    sp.kind = kind;
    sp.equal = equal_rows > 0 ? static_cast<int32_t>((equal_rows + tm - 1) / tm) : 0;
    sp.slots = static_cast<int32_t>(sp.equal ? owners * sp.equal : R * per / tm + owners);
    const int64_t items = static_cast<int64_t>(sp.slots) * p.kv_heads, sms = sm_count();
    if (kernel != Plan::kRows) {  // (slots are places for tiles; of tiles there are as many as owners of average size have)
      const int64_t tiles = owners * ((R * per / owners + tm - 1) / tm), n = (tiles < sp.slots ? tiles : sp.slots) * p.kv_heads;
      const bool paired = kernel == Plan::kPairs;
      sp.chunk = tile_chunk_keys(cap, n, paired ? sms : 2 * sms, paired ? 256 : 128, paired && cache->head_dim == 64 ? 1.4 : 2.0, cache->head_dim, R * d->q_heads, kind == kSpanJoint);
    }
    else sp.chunk = chunk_keys(cap, items, rows_resident(plan.blocks, cache->head_dim), 16 * PR_WARPS, cache->head_dim == 64 ? 1024 : 256, 3);
    sp.chunks = static_cast<int32_t>((cap + sp.chunk - 1) / sp.chunk);
  };
  if (rows_o > kSlotRows) {
    // Whole prompts or long chunks: prefix and own tokens in a row, no joining of the two, but a walk of the prefix per sequence.  8 key heads,
    // prompts without a history, the two apart (prefix by groups) against in a row, in us:
    //   head_dim 64    130 rows  4 sequences, one prefix of 1,000 keys 42 : 26   of 8,000 62 : 54     64 sequences, 1,000 133 : 120   8,000 349 : 514
    //                  256 rows                               49 : 32            77 : 60                            211 : 124         592 : 544
    //                  512 rows                               58 : 40           112 : 93                            393 : 214       1,130 : 945
    //   head_dim 128   132 rows                               46 : 30            69 : 59                            140 : 119         376 : 559
    //                  256 rows                               52 : 35            85 : 67                            239 : 122         664 : 576
    // (in a row loses where many sequences with few rows share a long prefix: their second slots are empty)
    plan.kernel[0] = plan.kernel[1] = Plan::kPairs;
    cut(plan.span[0], kSpanJoint, Plan::kPairs, S, round_up(cap_p, kSpanAlign) + cap_o, single ? per : 0);
    if (plan.span[0].chunks == 1) plan.span[0].part0 = -1;
  } else {
    // prefix_rows_kernel walks the keys once per 16 rows, without much to set up; the tile kernel starts slower and walks them once per 128.
    // One group, 8 key heads, single tokens, rows kernel against tiles, in us:
    //   head_dim 64    16 rows  4,000 keys 17 : 21   16,000 keys 20 : 28   40,000 keys 30 : 40     32 rows  4,000 keys 20 : 22   16,000 keys 26 : 30   40,000 keys 48 : 41
    //   head_dim 128    8 rows  4,000 keys 15 : 20   16,000 keys 28 : 32   40,000 keys 53 : 50     16 rows  4,000 keys 17 : 22   16,000 keys 30 : 32   40,000 keys 57 : 50
    //                  32 rows  4,000 keys 20 : 24    8,000 keys 26 : 26   16,000 keys 44 : 32     48 rows  4,000 keys 24 : 24    8,000 keys 38 : 28
    // A rule that meets these within 3 us: what the walks read together.
    const double bytes = 4.0 * static_cast<double>(G * cap_p) * cache->kv_heads * cache->head_dim;  // of the keys and values
    const bool few = rows_p <= (cache->head_dim == 64 ? 16 : 8) || (rows_p <= 64 && static_cast<double>((rows_p + 15) / 16) * bytes <= 64.0 * 1048576.0);
    // Pairs of slots share their keys, which counts where there are many; with an odd number of slots one of a pair idles, and a pair starts
    // slower.  8 key heads, slots by themselves against pairs, in us:
    //   head_dim 64, 6 MB of keys and values   256 rows 28 : 30   500 34 : 37      49 MB (8 groups)  256 rows 79 : 79   384 108 : 116   500 136 : 132
    //                61 MB (1 group)           256 rows 58 : 56   384 75 : 83   500 91 : 86
    //   head_dim 128, 12 MB  256 rows 28 : 32   512 36 : 38   600 36 : 38          34 MB  256 rows 39 : 42
    //                98 MB (8 groups)  200 rows 67 : 65   360 101 : 101   512 124 : 116   123 MB (1 group)  200 rows 67 : 63   256 67 : 65   360 85 : 89   512 108 : 95
    // (The rule below meets these within 4 us.)
    const bool pairs = rows_p > 4 * kSlotRows || (rows_p > 3 * kSlotRows && bytes > 32.0 * 1048576.0) || (rows_p > kSlotRows && bytes > 64.0 * 1048576.0);
    plan.kernel[0] = few ? Plan::kRows : (pairs ? Plan::kPairs : Plan::kTiles);
    // Own tokens of many sequences are many short walks, whose start counts for more.  160 sequences without a prefix, new tokens behind a
    // history, 8 key heads, rows kernel against tiles, in us:
    //   head_dim 64   12 rows  0 + 12 keys 22 : 38  500 + 12 62 : 79    24 rows  0 + 24 34 : 46  2,000 + 24 224 : 225    48 rows  100 + 48 75 : 75  500 + 48 139 : 110
    //   head_dim 128  16 rows  0 + 4 keys 36 : 44   500 + 4 106 : 99    32 rows  0 + 8 54 : 54   100 + 8 79 : 65  500 + 8 163 : 111    64 rows  0 + 16 91 : 79
    // (The rule below misses at head_dim 128, 16 rows with 500 tokens before them and 32 with 100.)
    const int64_t width = rows_o * cache->head_dim;
    plan.kernel[1] = width <= 32 * 64 || (width <= 64 * 64 && cap_o <= 256) ? Plan::kRows : Plan::kTiles;
    plan.blocks = (plan.kernel[0] == Plan::kRows && rows_p > 8) || (plan.kernel[1] == Plan::kRows && rows_o > 8) ? 2 : 1;
    cut(plan.span[0], kSpanPrefix, plan.kernel[0], G, cap_p, single && p.group_size > 0 ? static_cast<int64_t>(p.group_size) * per : 0);
    cut(plan.span[1], kSpanOwn, plan.kernel[1], S, cap_o, single ? per : 0);
    plan.span[1].part0 = plan.span[0].chunks;
  }
  plan.parts = plan.span[0].part0 < 0 ? 0 : plan.span[0].chunks + plan.span[1].chunks;
  const int64_t cells = R * d->q_heads;
  plan.ml_bytes = round_up(plan.parts * cells * 8, 32);
  plan.bytes = plan.ml_bytes + plan.parts * cells * cache->head_dim * 4;
  return 0;
}

}  // namespace
}  // namespace vx

extern "C" int64_t vx_prefix_attention_scratch(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d) {
  using namespace vx;
  PrefixParams p{};
  Plan plan;
  const int rc = check_prefix(cache, rows, d, p, plan);
  return rc ? rc : plan.bytes;
}

extern "C" int vx_prefix_attention_launches(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d) {
  using namespace vx;
  PrefixParams p{};
  Plan plan;
  const int rc = check_prefix(cache, rows, d, p, plan);
  if (rc) return rc;
  int n = p.rows.rows > 0 ? 1 : 0;  // the join
  for (const Plan::Kernel k : {Plan::kRows, Plan::kTiles, Plan::kPairs}) n += plan.walks(k) ? 1 : 0;
  return n;
}

extern "C" int vx_prefix_attention(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d, void* stream) {
  using namespace vx;
  PrefixParams p{};
  Plan plan;
  const int rc = check_prefix(cache, rows, d, p, plan);
  if (rc) return rc;
  if (p.rows.rows == 0) return 0;
  if (!d->q || !d->out) return fail(-1, "q and out must not be NULL");
  if (!pieces_ok(d->q, d->q_row, d->q_head, 2) || !pieces_ok(d->out, d->o_row, d->o_head, 2)) return fail(-1, "rows and heads of q and out must be 16-byte aligned");
  if (shares_places(p.rows.rows, d->o_row, d->q_heads, d->o_head, cache->head_dim)) return fail(-1, "two rows or heads of out in one place (stride below head_dim)");
  if (plan.bytes > 0 && (!d->scratch || (reinterpret_cast<uintptr_t>(d->scratch) & 31) != 0 || d->scratch_bytes < plan.bytes))
    return fail(-1, "scratch must be %lld bytes, 32-byte aligned", (long long)plan.bytes);
  p.q = static_cast<const __nv_bfloat16*>(d->q); p.q_row = d->q_row; p.q_head = d->q_head;
  p.out = static_cast<__nv_bfloat16*>(d->out); p.o_row = d->o_row; p.o_head = d->o_head;
  p.part_ml = static_cast<float2*>(d->scratch);
  p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(d->scratch) + plan.ml_bytes);
  const auto st = static_cast<cudaStream_t>(stream);
  const bool d64 = cache->head_dim == 64;
  p.status = device_status_ptr();
  for (const Plan::Kernel k : {Plan::kPairs, Plan::kTiles})
    if (plan.walks(k)) {
      const int e = launch_prefix_tiles(p, cache->head_dim, k == Plan::kPairs, plan.part(k, 0), plan.part(k, 1), stream);
      if (e) return e;
    }
  if (plan.walks(Plan::kRows)) {
    RowsParams rp{p, {plan.part(Plan::kRows, 0), plan.part(Plan::kRows, 1)}, {1, 1}, 0, plan.walks(Plan::kPairs) || plan.walks(Plan::kTiles) ? 1 : 0};
    int64_t blocks = 0;
    for (int i = 0; i < 2; ++i) {
      const Span& sp = rp.span[i];
      const int64_t items = static_cast<int64_t>(sp.slots) * sp.chunks * p.kv_heads;
      // All four warps of a CTA on an item while one round of CTAs takes them all, else so many that each has about 128 keys: twice as many take
      // 28 us for 27 (64 hypotheses of 102 to 198 tokens, four utterances of 1,005 to 1,792 frames) and 37 for 32 (124 of 30 to 60 tokens), half as many 29 and 32.
      rp.warps[i] = items <= rows_resident(plan.blocks, cache->head_dim) || sp.chunk > 256 ? 4 : (sp.chunk > 128 ? 2 : 1);
      blocks += (items * rp.warps[i] + PR_WARPS - 1) / PR_WARPS;
      if (i == 0) rp.first_blocks = static_cast<int32_t>(blocks);
    }
    if (blocks >= (1ll << 31)) return fail(-1, "too much work for one call (%lld blocks)", (long long)blocks);
    const int e = d64 ? (plan.blocks == 2 ? launch_rows<64, 2>(rp, blocks, st) : launch_rows<64, 1>(rp, blocks, st))
                      : (plan.blocks == 2 ? launch_rows<128, 2>(rp, blocks, st) : launch_rows<128, 1>(rp, blocks, st));
    if (e) return e;
  }
  JoinParams jp{p, {plan.span[0], plan.span[1]}, plan.parts == 0 && plan.span[0].part0 >= 0 ? 1 : 0};
  VX_CUDA_OK(d64 ? launch_join<64>(jp, plan.parts, st) : launch_join<128>(jp, plan.parts, st));
  return 0;
}
