// Attention of new tokens over a shared prefix and their own tokens in a paged cache:
//
//   out[r, h] = sum_j softmax_j(scale q[r, h] . k_j) v_j
//   keys: tokens [0, prefix_lengths[g]) of the group's pages, own tokens t <= lengths[s] + i of the sequence
//
// One warp per row and head.  32 keys a step: a lane takes the score of one key, the maximum and the sum of the softmax run along
// (m, l), and every lane sums its share of the 32 weighted values.
// What bounds it: L1 and L2; every row and head reads its keys and values for itself.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "vx_common.cuh"
#include "vx_paged.cuh"
#include "vx_ptx.cuh"

namespace vx {
namespace {

constexpr int PA_WARPS = 4;

struct PrefixParams {
  PagedCache cache;
  KvRows rows;
  const __nv_bfloat16* q;
  int64_t q_row, q_head;
  __nv_bfloat16* out;
  int64_t o_row, o_head;
  int32_t q_heads, per_kv;
  int32_t groups, group_size;
  const int32_t* group_offsets;
  PagedTable prefix;
  const int32_t* prefix_lengths;
  float scale;
};

// group of a sequence, -1: none
__device__ __forceinline__ int group_of(const PrefixParams& p, int s) {
  if (p.groups == 0) return -1;
  if (!p.group_offsets) return s / p.group_size;
  const int g = find_owner(p.group_offsets, p.groups, s);
  return s >= p.group_offsets[g] && s < p.group_offsets[g + 1] ? g : -1;
}

template <int D>
__global__ void __launch_bounds__(PA_WARPS * 32) prefix_attention_kernel(const PrefixParams p) {
  pdl_launch_dependents();
  __shared__ float q_s[PA_WARPS][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * PA_WARPS + warp;
  pdl_wait();
  if (item >= static_cast<int64_t>(p.rows.rows) * p.q_heads) return;
  const int row = static_cast<int>(item / p.q_heads), head = static_cast<int>(item % p.q_heads), kv = head / p.per_kv;
  constexpr int VL = D / 32;
  for (int c = 0; c < VL; ++c) {
    const int i = c * 32 + lane;
    q_s[warp][i] = __bfloat162float(p.q[row * p.q_row + head * p.q_head + i]) * p.scale;
  }
  __syncwarp();
  float m = -INFINITY, l = 0.0f, o[VL] = {};
  auto run = [&](const PagedTable& table, int owner, int64_t n) {
    n = min(n, static_cast<int64_t>(table.pages) * p.cache.page_size.d);
    for (int64_t j0 = 0; j0 < n; j0 += 32) {
      const int64_t j = j0 + lane;
      uint32_t index, slot;
      p.cache.page_size.divmod(static_cast<uint32_t>(j), index, slot);
      const int page = j < n ? page_of(table, owner, index, p.cache.pages) : -1;
      float s = -INFINITY;
      if (page >= 0) {
        const uint4* k = reinterpret_cast<const uint4*>(p.cache.k.p + page * p.cache.k.page + slot * p.cache.k.token + kv * p.cache.k.head);
        s = 0.0f;
        for (int c = 0; c < D / 8; ++c) {
          const uint4 u = k[c];
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s += __uint_as_float(w[e] << 16) * q_s[warp][c * 8 + 2 * e] + __uint_as_float(w[e] & 0xffff0000u) * q_s[warp][c * 8 + 2 * e + 1];
        }
      }
      float mx = s;
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float m_new = fmaxf(m, mx);
      const float ref = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = expf(m - ref), w = page >= 0 ? expf(s - ref) : 0.0f;
      float sum = w;
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l = l * alpha + sum;
      m = m_new;
#pragma unroll
      for (int c = 0; c < VL; ++c) o[c] *= alpha;
      for (int x = 0; x < 32; ++x) {
        const int pg = __shfl_sync(0xffffffffu, page, x);
        const uint32_t sl = __shfl_sync(0xffffffffu, slot, x);
        const float wx = __shfl_sync(0xffffffffu, w, x);
        if (pg < 0) continue;
        const __nv_bfloat16* v = p.cache.v.p + pg * p.cache.v.page + sl * p.cache.v.token + kv * p.cache.v.head;
#pragma unroll
        for (int c = 0; c < VL; ++c) o[c] += wx * __bfloat162float(v[c * 32 + lane]);
      }
    }
  };
  int s, i;
  if (row_sequence(p.rows, row, s, i)) {
    const int g = group_of(p, s);
    if (g >= 0) run(p.prefix, g, p.prefix_lengths[g]);
    run(p.rows.table, s, static_cast<int64_t>(p.rows.lengths[s]) + i + 1);
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  for (int c = 0; c < VL; ++c) p.out[row * p.o_row + head * p.o_head + c * 32 + lane] = __float2bfloat16_rn(o[c] * inv);
}

int check_prefix(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d, PrefixParams& p) {
  const int rc = check_paged(cache, rows, p.cache, p.rows);
  if (rc) return rc;
  if (!d || d->struct_size != static_cast<int32_t>(sizeof(vx_prefix_attention_desc))) return fail(-1, "vx_prefix_attention_desc: struct_size");
  if (d->reserved != 0) return fail(-1, "vx_prefix_attention_desc: reserved must be 0");
  if (cache->head_dim != 64 && cache->head_dim != 128) return fail(-1, "head_dim must be 64 or 128 (got %d)", cache->head_dim);
  if (d->q_heads < 1 || d->q_heads > 65535 || d->q_heads % cache->kv_heads != 0)
    return fail(-1, "q_heads (%d) must be a multiple of kv_heads (%d)", d->q_heads, cache->kv_heads);
  if (rows->rows * d->q_heads >= (1ll << 31)) return fail(-1, "rows * q_heads must stay below 2^31");
  if (d->groups < 0 || d->groups > (1ll << 31) - 1) return fail(-1, "bad number of groups %lld", (long long)d->groups);
  if (d->groups > 0) {
    if (!d->group_offsets && rows->sequences % d->groups != 0)
      return fail(-1, "without group_offsets the groups are of one size (sequences %lld, groups %lld)", (long long)rows->sequences, (long long)d->groups);
    if (d->prefix_pages < 0 || d->prefix_pages * cache->page_size > (1ll << 31) - 1) return fail(-1, "a prefix may have up to 2^31 - 1 tokens");
    if (!d->prefix_lengths || (d->prefix_pages > 0 && (!d->prefix_table || d->ld_prefix < d->prefix_pages)))
      return fail(-1, "prefix_lengths or prefix_table is NULL, or its rows are too short");
  }
  p.q_heads = d->q_heads;
  p.per_kv = d->q_heads / cache->kv_heads;
  p.groups = static_cast<int32_t>(d->groups);
  p.group_offsets = d->group_offsets;
  p.group_size = p.groups > 0 && !p.group_offsets ? static_cast<int32_t>(rows->sequences / d->groups) : 0;
  p.prefix = {d->prefix_table, d->ld_prefix, static_cast<int32_t>(d->prefix_pages)};
  p.prefix_lengths = d->prefix_lengths;
  p.scale = d->scale;
  return 0;
}

}  // namespace
}  // namespace vx

extern "C" int64_t vx_prefix_attention_scratch(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d) {
  using namespace vx;
  PrefixParams p{};
  const int rc = check_prefix(cache, rows, d, p);
  return rc ? rc : 0;
}

extern "C" int vx_prefix_attention(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_prefix_attention_desc* d, void* stream) {
  using namespace vx;
  PrefixParams p{};
  const int rc = check_prefix(cache, rows, d, p);
  if (rc) return rc;
  if (p.rows.rows == 0) return 0;
  if (!d->q || !d->out) return fail(-1, "q and out must not be NULL");
  if (!pieces_ok(d->q, d->q_row, d->q_head, 2) || !pieces_ok(d->out, d->o_row, d->o_head, 2)) return fail(-1, "rows and heads of q and out must be 16-byte aligned");
  p.q = static_cast<const __nv_bfloat16*>(d->q); p.q_row = d->q_row; p.q_head = d->q_head;
  p.out = static_cast<__nv_bfloat16*>(d->out); p.o_row = d->o_row; p.o_head = d->o_head;
  const int64_t items = static_cast<int64_t>(p.rows.rows) * p.q_heads;
  const dim3 grid(static_cast<unsigned>((items + PA_WARPS - 1) / PA_WARPS));
  const auto st = static_cast<cudaStream_t>(stream);
  if (cache->head_dim == 64) VX_CUDA_OK(launch_dependent(prefix_attention_kernel<64>, grid, dim3(PA_WARPS * 32), 0, st, p));
  else VX_CUDA_OK(launch_dependent(prefix_attention_kernel<128>, grid, dim3(PA_WARPS * 32), 0, st, p));
  return 0;
}
