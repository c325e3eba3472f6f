// New keys and values into the pages of a cache, rotated by position on the way, with the queries:
//
//   k page(s, t) = bf16(R(p) k[r])     v page(s, t) = bf16(v[r])     q_out[r] = bf16(R(p) q[r])
//   s, i: sequence of row r and its index there;  t = lengths[s] + i;  p = starts[s] + t
//   R(p): (a, b) -> (a cos - b sin, b cos + a sin) for every pair of the first rot_dim values, by the table's row p.
//
// A thread takes 16 values of one head of one row: the eight pairs of two 16-byte pieces (halves: pieces 8 u and rot_dim / 2 + 8 u,
// interleaved: 16 consecutive values), so cosines and sines are 64 consecutive bytes of the table and no value is read twice.  Where a
// row goes -- sequence, page, place -- is looked up once per row and block, not per thread.
// What bounds it: HBM (each input byte read once, each output byte written once; the table's rows come from L1 for all heads but the first):
// 89,978 tokens of 24 sequences, 32 query and 8 key heads of 128, half of each rotated, 2.2 GB in 354 us, 6.3 TB/s.  Small calls: the launch (2.8 us
// for 10 tokens).

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "vx_common.cuh"
#include "vx_paged.cuh"
#include "vx_ptx.cuh"

namespace vx {

int check_paged(const vx_kv_cache* cache, const vx_kv_rows* rows, PagedCache& c, KvRows& r) {
  if (!cache || cache->struct_size != static_cast<int32_t>(sizeof(vx_kv_cache))) return fail(-1, "vx_kv_cache: struct_size");
  if (!rows || rows->struct_size != static_cast<int32_t>(sizeof(vx_kv_rows))) return fail(-1, "vx_kv_rows: struct_size");
  if (rows->reserved != 0) return fail(-1, "vx_kv_rows: reserved must be 0");
  constexpr int64_t kMax = (1ll << 31) - 1;
  if (cache->page_size < 1 || cache->pages < 0 || cache->pages > kMax || cache->kv_heads < 1 || cache->kv_heads > 65535)
    return fail(-1, "vx_kv_cache: bad shape (pages %lld, page_size %d, kv_heads %d)", (long long)cache->pages, cache->page_size, cache->kv_heads);
  if (cache->pages > 0 && (!cache->k || !cache->v)) return fail(-1, "vx_kv_cache: k and v must not be NULL");
  const int64_t strides[] = {cache->k_page, cache->k_token, cache->k_head, cache->v_page, cache->v_token, cache->v_head};
  for (const int64_t s : strides)
    if (s < 0 || s % 8 != 0) return fail(-1, "vx_kv_cache: strides must be multiples of 8 elements");
  if (!aligned16(cache->k) || !aligned16(cache->v)) return fail(-1, "vx_kv_cache: k and v must be 16-byte aligned");
  if (rows->rows < 0 || rows->rows > kMax || rows->sequences < 0 || rows->sequences > kMax) return fail(-1, "vx_kv_rows: bad shape");
  if (!rows->row_offsets && rows->rows != rows->sequences)
    return fail(-1, "vx_kv_rows: without row_offsets every sequence has one row (rows %lld, sequences %lld)", (long long)rows->rows, (long long)rows->sequences);
  if (rows->table_pages < 0 || rows->table_pages > kMax / cache->page_size) return fail(-1, "vx_kv_rows: a sequence may have up to 2^31 - 1 tokens");
  if (rows->rows > 0 && rows->sequences > 0) {
    if (!rows->lengths) return fail(-1, "vx_kv_rows: lengths must not be NULL");
    if (rows->table_pages > 0 && (!rows->page_table || rows->ld_table < rows->table_pages)) return fail(-1, "vx_kv_rows: page_table NULL or its rows too short");
  }
  c.k = {static_cast<__nv_bfloat16*>(cache->k), cache->k_page, cache->k_token, cache->k_head};
  c.v = {static_cast<__nv_bfloat16*>(cache->v), cache->v_page, cache->v_token, cache->v_head};
  c.page_size = FastDiv(static_cast<uint32_t>(cache->page_size));
  c.pages = static_cast<int32_t>(cache->pages);
  r.rows = static_cast<int32_t>(rows->rows);
  r.sequences = static_cast<int32_t>(rows->sequences);
  r.lengths = rows->lengths;
  r.row_offsets = rows->row_offsets;
  r.table = {rows->page_table, rows->ld_table, static_cast<int32_t>(rows->table_pages)};
  return 0;
}

namespace {

constexpr int AP_THREADS = 256;
constexpr int AP_BLOCKS = 6;     // per SM, at 40 registers a thread: five of 46 take 375 us at the size above, seven or eight, which spill, 507
constexpr int AP_UNITS = 16;     // of a thread in large calls, since a block looks its rows up before it moves any: 4 take 422 us there, 8 391, 16 375 (of five blocks)
constexpr int AP_MAX_ROWS = 32;  // rows of a block at most

struct AppendParams {
  PagedCache cache;
  KvRows rows;
  const void *k, *v, *q;
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;
  __nv_bfloat16* q_out;
  int64_t qo_row, qo_head;
  const float* rotary;
  int64_t ld_rotary;
  int32_t positions;
  const int32_t* starts;
  int32_t q_heads, kv_heads, rot_units;  // rotated units of 16 values per head
  int32_t half;                          // rot_dim / 2; 0: interleaved (or no rotation)
  int32_t rows_per_block;
  FastDiv units_per_row, units_per_head;
};

// where the rows of a block go
struct RowPlace {
  int64_t k, v;      // offset of the token's place in the cache, -1: not stored
  int32_t position;  // -1: left out
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(w[j] << 16);
    x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&v);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__global__ void __launch_bounds__(AP_THREADS, AP_BLOCKS) kv_append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  __shared__ RowPlace place[AP_MAX_ROWS];
  const int row0 = static_cast<int>(blockIdx.x) * p.rows_per_block;
  const int n_rows = min(p.rows_per_block, p.rows.rows - row0);
  pdl_wait();
  if (static_cast<int>(threadIdx.x) < n_rows) {
    RowPlace pl{-1, -1, -1};
    int s;
    int64_t i;
    if (row_sequence(p.rows, row0 + threadIdx.x, s, i)) {
      const int64_t t = p.rows.lengths[s] + i;
      const int64_t pos = t + (p.starts ? p.starts[s] : 0);
      if (!p.rotary) pl.position = 0;
      else if (pos >= 0 && pos < p.positions) pl.position = static_cast<int32_t>(pos);
      if (pl.position >= 0 && t < (1ll << 31)) {
        uint32_t index, slot;
        p.cache.page_size.divmod(static_cast<uint32_t>(t), index, slot);
        const int page = page_of(p.rows.table, s, index, p.cache.pages);
        if (page >= 0) {
          pl.k = page * p.cache.k.page + slot * p.cache.k.token;
          pl.v = page * p.cache.v.page + slot * p.cache.v.token;
        }
      }
    }
    place[threadIdx.x] = pl;
  }
  __syncthreads();
  const uint32_t total = static_cast<uint32_t>(n_rows) * p.units_per_row.d;
  for (uint32_t n = threadIdx.x; n < total; n += AP_THREADS) {
    uint32_t lr, unit, head, u;
    p.units_per_row.divmod(n, lr, unit);
    p.units_per_head.divmod(unit, head, u);
    const RowPlace pl = place[lr];
    const int64_t row = row0 + static_cast<int>(lr);
    // which of the three, its input and its output
    const T* src;
    __nv_bfloat16* dst;
    bool rotates = static_cast<int>(u) < p.rot_units;
    if (static_cast<int>(head) < p.q_heads) {
      src = static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head;
      dst = p.q_out + row * p.qo_row + head * p.qo_head;
    } else if (static_cast<int>(head) < p.q_heads + p.kv_heads) {
      head -= p.q_heads;
      if (pl.k < 0) continue;
      src = static_cast<const T*>(p.k) + row * p.k_row + head * p.k_head;
      dst = p.cache.k.p + pl.k + head * p.cache.k.head;
    } else {
      head -= p.q_heads + p.kv_heads;
      if (pl.v < 0) continue;
      src = static_cast<const T*>(p.v) + row * p.v_row + head * p.v_head;
      dst = p.cache.v.p + pl.v + head * p.cache.v.head;
      rotates = false;
    }
    // the two pieces of eight
    int c0 = 16 * static_cast<int>(u), c1 = c0 + 8;
    if (rotates && p.half) {
      c0 = 8 * static_cast<int>(u);
      c1 = c0 + p.half;
    }
    float a[8] = {}, b[8] = {};
    if (pl.position >= 0) {
      load8(src + c0, a);
      load8(src + c1, b);
      if (rotates) {
        const float* cs = p.rotary + pl.position * p.ld_rotary + 8 * u;
        float c[8], s[8];
        load8(cs, c);
        load8(cs + 8 * p.rot_units, s);
        if (p.half) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = a[j], y = b[j];
            a[j] = x * c[j] - y * s[j];
            b[j] = y * c[j] + x * s[j];
          }
        } else {
          auto turn = [&](float (&x)[8], int j0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float e = x[2 * j], o = x[2 * j + 1];
              x[2 * j] = e * c[j0 + j] - o * s[j0 + j];
              x[2 * j + 1] = o * c[j0 + j] + e * s[j0 + j];
            }
          };
          turn(a, 0);
          turn(b, 4);
        }
      }
    }
    store8(dst + c0, a);
    store8(dst + c1, b);
  }
}

}  // namespace
}  // namespace vx

extern "C" int vx_kv_append(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_kv_append_desc* d, void* stream) {
  using namespace vx;
  AppendParams p{};
  const int rc = check_paged(cache, rows, p.cache, p.rows);
  if (rc) return rc;
  if (!d || d->struct_size != static_cast<int32_t>(sizeof(vx_kv_append_desc))) return fail(-1, "vx_kv_append_desc: struct_size");
  if (d->reserved != 0) return fail(-1, "vx_kv_append_desc: reserved must be 0");
  const int D = cache->head_dim;
  if (D < 16 || D > 256 || D % 16 != 0) return fail(-1, "head_dim must be a multiple of 16 up to 256 (got %d)", D);
  if (d->dtype != VX_F32 && d->dtype != VX_BF16) return fail(-1, "dtype must be VX_F32 or VX_BF16");
  const bool has_q = d->q != nullptr;
  if (has_q ? !d->q_out || d->q_heads < 1 : d->q_out != nullptr) return fail(-1, "q and q_out go together, with q_heads >= 1");
  if (has_q && d->q_heads > 65535) return fail(-1, "too many heads");
  if (d->rotary) {
    if (d->rot_dim < 16 || d->rot_dim > D || d->rot_dim % 16 != 0) return fail(-1, "rot_dim must be a multiple of 16 up to head_dim (got %d)", d->rot_dim);
    if (d->positions < 0 || d->ld_rotary < d->rot_dim || !pieces_ok(d->rotary, d->ld_rotary, 0, 4)) return fail(-1, "rotary must be 16-byte aligned rows of rot_dim floats");
  }
  if (p.rows.rows == 0) return 0;
  if (!d->k || !d->v) return fail(-1, "k and v must not be NULL");
  const int64_t extent[3] = {cache->pages, cache->page_size, cache->kv_heads};
  const int64_t k_step[3] = {cache->k_page, cache->k_token, cache->k_head}, v_step[3] = {cache->v_page, cache->v_token, cache->v_head};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (k_step[i] < D || v_step[i] < D)) return fail(-1, "two tokens or heads of the cache in one place (stride below head_dim)");
  const int es = d->dtype == VX_F32 ? 4 : 2;
  if (!pieces_ok(d->k, d->k_row, d->k_head, es) || !pieces_ok(d->v, d->v_row, d->v_head, es) ||
      (has_q && (!pieces_ok(d->q, d->q_row, d->q_head, es) || !pieces_ok(d->q_out, d->qo_row, d->qo_head, 2))))
    return fail(-1, "rows and heads of q, k, v and q_out must be 16-byte aligned");
  if (has_q && shares_places(p.rows.rows, d->qo_row, d->q_heads, d->qo_head, D)) return fail(-1, "two rows or heads of q_out in one place (stride below head_dim)");
  if (d->q == d->q_out && has_q && (d->dtype != VX_BF16 || d->q_row != d->qo_row || d->q_head != d->qo_head)) return fail(-1, "q_out may be q only as the same bf16 tensor");
  p.k = d->k; p.v = d->v; p.q = d->q;
  p.k_row = d->k_row; p.k_head = d->k_head; p.v_row = d->v_row; p.v_head = d->v_head; p.q_row = d->q_row; p.q_head = d->q_head;
  p.q_out = static_cast<__nv_bfloat16*>(d->q_out); p.qo_row = d->qo_row; p.qo_head = d->qo_head;
  p.rotary = d->rotary; p.ld_rotary = d->ld_rotary;
  p.positions = static_cast<int32_t>(d->positions < (1ll << 31) - 1 ? d->positions : (1ll << 31) - 1);
  p.starts = d->starts;
  p.q_heads = has_q ? d->q_heads : 0;
  p.kv_heads = cache->kv_heads;
  p.rot_units = d->rotary ? d->rot_dim / 16 : 0;
  p.half = d->rotary && !d->interleaved ? d->rot_dim / 2 : 0;
  p.units_per_head = FastDiv(static_cast<uint32_t>(D / 16));
  const int64_t upr = static_cast<int64_t>(p.q_heads + 2 * p.kv_heads) * (D / 16);
  p.units_per_row = FastDiv(static_cast<uint32_t>(upr));
  // Rows per block; fewer while that leaves SMs without a block.
  int64_t rpb = (AP_UNITS * AP_THREADS + upr - 1) / upr;
  const int64_t fill = p.rows.rows / (4 * sm_count());
  if (rpb > fill) rpb = fill;
  if (rpb > AP_MAX_ROWS) rpb = AP_MAX_ROWS;
  if (rpb < 1) rpb = 1;
  p.rows_per_block = static_cast<int32_t>(rpb);
  const dim3 grid(static_cast<unsigned>((p.rows.rows + rpb - 1) / rpb));
  const auto st = static_cast<cudaStream_t>(stream);
  if (d->dtype == VX_F32) VX_CUDA_OK(launch_dependent(kv_append_kernel<float>, grid, dim3(AP_THREADS), 0, st, p));
  else VX_CUDA_OK(launch_dependent(kv_append_kernel<__nv_bfloat16>, grid, dim3(AP_THREADS), 0, st, p));
  return 0;
}
