// Attention over a cache in 4 bits, for few rows per owner and key head (the cut of the work: vx_prefix.cuh; what it is: vx_prefix_attn.cu, whose
// kernel for few rows this one follows: up to 16 rows against one chunk of keys, by one, two or four warps, keys and values on the m16 side of
// m16n8k16 products).  What is its own:
//
// A unit of 16 keys (vx_paged.cuh) is one bulk copy of 9 D bytes, for the keys and for the values; a warp has a ring of them.  Units whose page is not
// there are left out of the ring, so that a step has 16 keys or the end of a run.
//
// Products are fp16: a code is 0 to 6 in halves, a scale of 4 significant bits over 256 at most 1.875 and 2^-17 at least, so code times scale is exact.
// Queries are multiplied by a power of two of their row, which puts the largest in [1, 2): from 2^-17 of it on bf16 values stay exact, smaller
// ones are off by 2^-25 of it at most.  Whatever bytes a cache holds are finite values, so what a row does not see needs a probability of 0 only.
//
// Probabilities are 2^(x - reference).  fp16 goes from 2^-24 to 2^16, so the reference is a maximum less 7 and moves when exceeded by 15: the largest is between 2^7 and 2^15,
// and the others are off by 2^-11 or by 2^-32 of the largest (2^-25 of it with the maximum itself as reference: a key in front of 90,000 that are 2^25 times less likely took a
// part of their weight from the result, though not from the row's sum, which is fp32).
//
// Where the values come from, lane = 4 g + c:
//   S^T = K Q^T: a lane has D / 4 values of keys g and g + 8, those at (D / 4) c: their scales are its own.  Two values of a byte are one register of
//     a product; q is read in the same order.
//   O^T += V^T P^T: a lane has the D / 8 values at (D / 8) g of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9.  The halves of two keys' bytes are put together
//     (key 2 c low), so that a converted byte is one register: columns 2 t and 2 t + 1 of a word are rows g and g + 8 of product t.
// What bounds it: issue slots.  A unit takes a warp some 410 instructions at head_dim 128, 163 of them in the ALU pipe; 64 sequences of 4,000 to 8,000 tokens, 32 query heads on 8 key
// heads of 128 (269 MB), take 86 to 91 us, 3.1 TB/s, issue slots 63 % busy (bf16 pages: 171).  Few keys: round trips to memory; ten sequences of 400 tokens, 8 heads of 64, 6.5 us.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "vx_common.cuh"
#include "vx_prefix.cuh"
#include "vx_ptx.cuh"

namespace vx {
namespace {

// CTAs of four warps per SM; those of eight or sixteen, which take an item each, have as many warps together.  (Two blocks of rows at head_dim 128 spill 48 bytes, at 168
// registers, the others none.)
constexpr int rows4_ctas(int rb, int head_dim) { return head_dim == 64 ? 4 : (rb == 2 ? 3 : 4); }

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// 8 x 8 block of 16-bit values, lane 4 g + c holding (g, 2 c) and (g, 2 c + 1): the same of its transpose
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int BYTES>
__device__ __forceinline__ void ld_shared_words(uint32_t addr, uint32_t (&r)[BYTES / 4]) {
  if constexpr (BYTES == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else if constexpr (BYTES == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r[0]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_u8(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u16 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
  return r;
}
// scale bytes (lo, hi) of a word's two halves as fp16 over 256
__device__ __forceinline__ uint32_t scales_as_half(uint32_t two) { return (two << 7) & 0x3f803f80u; }

template <int D>
struct Rows4Shape {
  static constexpr int kUnit = kFp4Unit * D;
  static constexpr int kStages = D == 128 ? 4 : 6;
  static constexpr int kRing = kStages * 2 * kUnit;  // of a warp
};

// RB blocks of eight rows.  WHOLE: an item has all keys of its rows, those of the prefix and its own (one chunk of a joint span), and writes them to `out`.
template <int D, int RB, int WARPS, bool WHOLE>
__global__ void __launch_bounds__(WARPS * 32, rows4_ctas(RB, D) * PR_WARPS / WARPS) prefix_rows_fp4_kernel(const __grid_constant__ RowsParams rp) {
  using Shape = Rows4Shape<D>;
  constexpr int NS = Shape::kStages, UNIT = Shape::kUnit;
  constexpr int KW = D / 32;  // words of a key per lane
  constexpr int VW = D / 64;  // words of a value per lane
  constexpr int TM = 8 * RB;
  constexpr unsigned ALL = 0xffffffffu;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 ml_s[WARPS][TM];
  __shared__ uint64_t full_s[WARPS][NS];
  __shared__ int first_s[WARPS][NS];  // first key of a stage
  const PrefixParams& p = rp.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  if (lane < NS) mbar_init(&full_s[warp][lane], 1);
  if (lane == 0) mbar_fence_init();
  __syncwarp();
  // Beside the tile kernel of the same call: see prefix_rows_kernel.
  struct Behind {
    const bool last;
    __device__ ~Behind() {
      if (last) pdl_wait();
    }
  } behind{rp.beside != 0};
  if (!rp.beside) pdl_wait();
  pdl_launch_dependents();
  int n = static_cast<int>(blockIdx.x);
  const bool second = n >= rp.first_blocks;
  if (second) n -= rp.first_blocks;
  const Span& sp = rp.span[second];
  const int warps = rp.warps[second], team = warp / warps, rank = warp - team * warps;  // the warps of an item
  n = n * (WARPS / warps) + team;
  const int head = n % p.kv_heads;
  n /= p.kv_heads;
  const int chunk = n / sp.slots;
  if (chunk >= sp.chunks) return;
  const bool own = WHOLE || sp.kind == kSpanOwn;
  if (WHOLE && blockIdx.x == 0) {  // rows of no sequence: zeros
    const int head_pieces = D / 8, pieces = p.q_heads * head_pieces;
    const int before = owner_row0(p, true, 0), behind = owner_row0(p, true, p.rows.sequences);
    for (int row = 0; row < p.rows.rows; ++row) {
      if (row == before) row = max(behind, before);
      if (row >= p.rows.rows) break;
      for (int i = threadIdx.x; i < pieces; i += WARPS * 32)
        *reinterpret_cast<uint4*>(p.out + row * p.o_row + i / head_pieces * p.o_head + i % head_pieces * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  ItemRows it;
  if (!find_rows<TM>(p, sp, n - chunk * sp.slots, it)) return;
  const int length = own ? tokens_before(p, it.owner) : 0;
  // keys [key0, keys): those of the chunk that the tile's last row sees; in front of them, joint, `shared` units of the prefix
  int keys = own ? own_keys(p, length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(min(it.rho0 + TM, it.rows) - 1)))) : prefix_keys(p, it.owner);
  if (!WHOLE && static_cast<int64_t>(chunk) * sp.chunk >= keys) return;
  const int key0 = chunk * sp.chunk;
  keys = static_cast<int>(min(static_cast<int64_t>(keys), static_cast<int64_t>(key0) + sp.chunk));
  int group = -1, shared_keys = 0;
  if (WHOLE && length >= 0) {
    group = group_of(p, it.owner);
    shared_keys = prefix_keys(p, group);
  }
  const int shared = (shared_keys + 15) / 16;
  const PagedTable& table = own ? p.rows.table : p.prefix;
  const int blocks = it.rows - it.rho0 > 8 ? RB : 1;  // that have rows

  // The warp's units, in its turn: unit i of them begins with key key0 + 16 (rank + i warps).  They are looked up 32 at a time, a lane each, one
  // turn ahead; the lane that has a unit issues its copies.
  const int units = shared + (keys - key0 + 15) / 16, mine = units > rank ? (units - rank - 1) / warps + 1 : 0;
  const int64_t head_at = static_cast<int64_t>(head) * p.fp4.page_units.d * UNIT;
  const uint32_t ring = smem_u32(smem) + warp * Shape::kRing;
  auto look_up = [&](int i, uint32_t& rest) {
    rest = 0;
    if (i >= mine) return -1;
    uint32_t index;
    const int unit = rank + i * warps - shared;
    const bool in_prefix = WHOLE && unit < 0;
    p.fp4.page_units.divmod(static_cast<uint32_t>(in_prefix ? unit + shared : key0 / 16 + unit), index, rest);
    return page_of(in_prefix ? p.prefix : table, in_prefix ? group : it.owner, index, p.cache.pages);
  };
  uint32_t rest, rest_next;
  int page = look_up(lane, rest), page_next = look_up(32 + lane, rest_next);
  uint32_t present = __ballot_sync(ALL, page >= 0);
  int turn = 0, issued = 0, write = 0;
  auto fetch = [&] {  // the next unit that is there
    while (present == 0) {
      if ((turn += 32) >= mine) return;
      page = page_next;
      rest = rest_next;
      page_next = look_up(turn + 32 + lane, rest_next);
      present = __ballot_sync(ALL, page >= 0);
    }
    const int at = __ffs(present) - 1;
    present &= present - 1;
    if (lane == at) {
      uint64_t* const bar = &full_s[warp][write];
      uint8_t* const dst = smem + warp * Shape::kRing + write * 2 * UNIT;
      first_s[warp][write] = key0 + 16 * (rank + (turn + at) * warps - shared);  // (of the prefix: as far in front)
      mbar_expect_tx(bar, 2 * UNIT);
      const int64_t off = head_at + static_cast<int64_t>(rest) * UNIT;
      bulk_load(dst, p.fp4.k + page * p.fp4.k_page + off, UNIT, bar);
      bulk_load(dst + UNIT, p.fp4.v + page * p.fp4.v_page + off, UNIT, bar);
    }
    ++issued;
    if (++write == NS) write = 0;
  };
#pragma unroll 1
  for (int i = 0; i < NS; ++i) fetch();

  // queries: row 8 r + g, the values (D / 4) c + 8 i of this lane; the exponents of the rows' powers of two
  uint32_t q[RB][KW][4];
  float factor[RB][2];  // of the scores of rows 8 r + 2 c + e
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int rho = it.rho0 + 8 * r + g;
    uint32_t tok, hq;
    p.per_kv.divmod(static_cast<uint32_t>(rho), tok, hq);
    const __nv_bfloat16* src = p.q + static_cast<int64_t>(it.row0 + static_cast<int>(tok)) * p.q_row + (head * static_cast<int64_t>(p.per_kv.d) + hq) * p.q_head;
    uint32_t raw[KW][4], most = 0;
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (rho < it.rows) u = *reinterpret_cast<const uint4*>(src + (D / 4) * c + 8 * i);
      raw[i][0] = u.x; raw[i][1] = u.y; raw[i][2] = u.z; raw[i][3] = u.w;
#pragma unroll
      for (int j = 0; j < 4; ++j) most = max(most, max(raw[i][j] & 0x7fff0000u, (raw[i][j] & 0x7fffu) << 16));
    }
    most = max(most, __shfl_xor_sync(ALL, most, 1));
    most = max(most, __shfl_xor_sync(ALL, most, 2));
    const int e = min(max(static_cast<int>(most >> 23), 1), 227);  // (to 2^100; what is above, to 2^115, fp16 holds as it is)
    const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23), up = fminf(p.scale2 * __uint_as_float(static_cast<uint32_t>(e) << 23), 3.0e38f);
#pragma unroll
    for (int i = 0; i < KW; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[r][i][j] = pack_f16(__uint_as_float(raw[i][j] << 16) * down, __uint_as_float(raw[i][j] & 0xffff0000u) * down);
    factor[r][0] = __shfl_sync(ALL, up, 8 * c);
    factor[r][1] = __shfl_sync(ALL, up, 8 * c + 4);
  }
  // keys that row 8 r + 2 c + e sees; the first row of the tile sees fewest
  int limit[RB][2], min_limit = keys;
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      limit[r][e] = own ? min(own_keys(p, length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(it.rho0 + 8 * r + 2 * c + e)))), keys) : keys;
  if (own) min_limit = min(own_keys(p, length, static_cast<int>(p.per_kv.div(static_cast<uint32_t>(it.rho0)))), keys);

  const float NEG_INF = __int_as_float(0xff800000);
  float m_ref[RB][2], l[RB][2], o[RB][VW][4][4];  // of rows 8 r + 2 c + e
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    m_ref[r][0] = m_ref[r][1] = NEG_INF;
    l[r][0] = l[r][1] = 0.0f;
#pragma unroll
    for (int b = 0; b < VW; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[r][b][j][0] = o[r][b][j][1] = o[r][b][j][2] = o[r][b][j][3] = 0.0f;
  }

  // where this lane reads in a stage
  const uint32_t k_at = g * (D / 2) + c * (D / 8), ks_at = 8 * D + g * (D / 16) + c * (D / 64);          // keys g, g + 8
  const uint32_t v_at = UNIT + 2 * c * (D / 2) + g * (D / 16), vs_at = UNIT + 8 * D + 2 * c * (D / 16) + g * (D / 16) / 8;  // keys 2 c + e + 8 f
  auto step = [&](const uint32_t at, const int j0) {
    float s[RB][4];  // [2 b + e]: key 8 b + g, row 8 r + 2 c + e
#pragma unroll
    for (int r = 0; r < RB; ++r) s[r][0] = s[r][1] = s[r][2] = s[r][3] = 0.0f;
    {
      uint32_t kw[2][KW], ks[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        ld_shared_words<D / 8>(at + k_at + f * 8 * (D / 2), kw[f]);
        ks[f] = D == 128 ? ld_shared_u16(at + ks_at + f * 8 * (D / 16)) : ld_shared_u8(at + ks_at + f * 8 * (D / 16));
      }
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        uint32_t h[2][4];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          // the scale of the word's values in both halves: its byte, the low one of ks for the first two words
          const uint32_t sc = scales_as_half(__byte_perm(ks[f], 0, D == 128 && i >= KW / 2 ? 0x4141 : 0x4040));
          e2m1_as_half(kw[f][i], h[f]);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[f][j] = mul_f16x2(h[f][j], sc);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r)
          if (r < blocks) {
            mma_f16_16816(s[r], h[0][0], h[1][0], h[0][1], h[1][1], q[r][i][0], q[r][i][1]);
            mma_f16_16816(s[r], h[0][2], h[1][2], h[0][3], h[1][3], q[r][i][2], q[r][i][3]);
          }
      }
    }
    // scores in units of log2; keys that the row does not see count as -inf
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[r][e] *= factor[r][e & 1];
    if (WHOLE && j0 < 0) {  // of the prefix (key0 is 0): its last unit may end early
      const int end = shared_keys - 16 * shared;
      if (j0 + 16 > end) {
#pragma unroll
        for (int r = 0; r < RB; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j0 + 8 * (e >> 1) + g >= end) s[r][e] = NEG_INF;
      }
    } else if (j0 + 16 > min_limit) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j0 + 8 * (e >> 1) + g >= limit[r][e & 1]) s[r][e] = NEG_INF;
    }
    bool moves = false;
    float mx[RB][2];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[r][e] = fmaxf(s[r][e], s[r][2 + e]);
        moves = moves || mx[r][e] - m_ref[r][e] > kFp4Below + 8.0f;  // (the difference: a sum can be rounded up)
      }
    if (__any_sync(ALL, moves)) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mx[r][e] = fmaxf(mx[r][e], __shfl_xor_sync(ALL, mx[r][e], x));
          const float m_new = fmaxf(m_ref[r][e], mx[r][e] - kFp4Below);
          const float alpha = m_new == NEG_INF ? 1.0f : ex2(m_ref[r][e] - m_new);
          m_ref[r][e] = m_new;
          l[r][e] *= alpha;
#pragma unroll
          for (int b = 0; b < VW; ++b)
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
        pt[r][b] = transpose8x8(pack_f16(x0, x1));
      }
    }
    uint32_t vw[4][VW], sc[2];  // keys 2 c + (e & 1) + 8 (e >> 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) ld_shared_words<D / 16>(at + v_at + ((e & 1) + 8 * (e >> 1)) * (D / 2), vw[e]);
#pragma unroll
    for (int f = 0; f < 2; ++f) sc[f] = scales_as_half(ld_shared_u8(at + vs_at + 8 * f * (D / 16)) | ld_shared_u8(at + vs_at + (8 * f + 1) * (D / 16)) << 16);
#pragma unroll
    for (int b = 0; b < VW; ++b) {
      uint32_t even[2][4], odd[2][4];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const uint32_t x = vw[2 * f][b], y = vw[2 * f + 1][b];
        e2m1_as_half((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), even[f]);
        e2m1_as_half(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), odd[f]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          even[f][j] = mul_f16x2(even[f][j], sc[f]);
          odd[f][j] = mul_f16x2(odd[f][j], sc[f]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < RB; ++r)
          if (r < blocks) mma_f16_16816(o[r][b][j], even[0][j], odd[0][j], even[1][j], odd[1][j], pt[r][0], pt[r][1]);
    }
  };
  int stage = 0, done = 0;
  uint32_t phase = 0;
  auto next_stage = [&] {
    if (++stage == NS) {
      stage = 0;
      phase ^= 1;
    }
  };
#pragma unroll 1
  for (; done < issued; ++done) {
    if (!__all_sync(ALL, mbar_wait(&full_s[warp][stage], phase, p.status, 60))) break;
    step(ring + stage * 2 * UNIT, first_s[warp][stage]);
    __syncwarp();  // every lane has read the stage: it is filled again
    fetch();
    next_stage();
  }
  // Copies on their way after a limit ran out: each is waited for, with a limit, before its place is used for something else.
#pragma unroll 1
  for (; done < issued; ++done) {
    __all_sync(ALL, mbar_wait(&full_s[warp][stage], phase, p.status, 60));
    next_stage();
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
      for (int x = 4; x < 32; x <<= 1) l[r][e] += __shfl_xor_sync(ALL, l[r][e], x);
      const int lr = 8 * r + 2 * c + e;
      if (g == 0) ml_s[warp][lr] = make_float2(m_ref[r][e], l[r][e]);
#pragma unroll
      for (int b = 0; b < VW; ++b) {  // columns (D / 8) g + 8 b + 2 j + {0, 1}
        float* dst = o_s + warp * OWN + lr * PITCH + (D / 8) * g + 8 * b;
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
      const float a = ex2(ml_s[w][lr].x - ref), f = a * p.v_factor;
      const float4 x = *reinterpret_cast<const float4*>(o_s + w * OWN + lr * PITCH + col);
      sum += a * ml_s[w][lr].y;
      acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
    uint32_t tok, hq;
    p.per_kv.divmod(static_cast<uint32_t>(rho), tok, hq);
    const int64_t row = it.row0 + static_cast<int>(tok), qh = head * static_cast<int64_t>(p.per_kv.d) + hq;
    if (WHOLE) {
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(p.out + row * p.o_row + qh * p.o_head + col) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      continue;
    }
    const int64_t at = (static_cast<int64_t>(sp.part0 + chunk) * p.rows.rows + row) * p.q_heads + qh;
    if (col == 0) p.part_ml[at] = make_float2(m, sum);
    *reinterpret_cast<float4*>(p.part_o + at * D + col) = acc;
  }
}

template <int D, int RB, int WARPS, bool WHOLE>
int launch(const RowsParams& rp, int64_t blocks, cudaStream_t st) {
  constexpr int kSmem = WARPS * Rows4Shape<D>::kRing;
  int dev = 0;
  VX_CUDA_OK(cudaGetDevice(&dev));
  static std::atomic<uint64_t> attr_done{0};
  const bool cached = dev >= 0 && dev < 64;
  if (!cached || !(attr_done.load(std::memory_order_acquire) & (1ull << dev))) {
    VX_CUDA_OK(cudaFuncSetAttribute(prefix_rows_fp4_kernel<D, RB, WARPS, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (cached) attr_done.fetch_or(1ull << dev, std::memory_order_release);
  }
  VX_CUDA_OK(launch_dependent(prefix_rows_fp4_kernel<D, RB, WARPS, WHOLE>, dim3(static_cast<unsigned>(blocks)), dim3(WARPS * 32), kSmem, st, rp));
  return 0;
}
template <int D>
int launch(const RowsParams& rp, int rb, int64_t blocks, cudaStream_t st) {
  if (rp.span[0].part0 < 0)
    return rp.warps[0] == 16 ? launch<D, 1, 16, true>(rp, blocks, st) : rp.warps[0] == 8 ? launch<D, 1, 8, true>(rp, blocks, st) : launch<D, 1, PR_WARPS, true>(rp, blocks, st);
  return rb == 2 ? launch<D, 2, PR_WARPS, false>(rp, blocks, st) : launch<D, 1, PR_WARPS, false>(rp, blocks, st);
}

}  // namespace

int rows_fp4_ctas(int rb, int head_dim) { return rows4_ctas(rb, head_dim); }

int launch_rows_fp4(const RowsParams& rp, int head_dim, int rb, int64_t blocks, void* stream) {
  const auto st = static_cast<cudaStream_t>(stream);
  return head_dim == 64 ? launch<64>(rp, rb, blocks, st) : launch<128>(rp, rb, blocks, st);
}

}  // namespace vx
