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

//
// Into a cache in 4 bits (FP4): a thread takes the 16 values of one scale of a key or value; for a rotated key it loads the partners of its values
// too, so that no thread waits for another's maximum (a second load of the same bytes, from L1).  The size above takes 384 us, 1.9 GB at 4.9 TB/s: issue slots 56 % busy,
// loads in flight of five blocks an SM (queries by a launch of their own, of six blocks: 410); 10 tokens 5 us, the call.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "vx_common.cuh"
#include "vx_paged.cuh"
#include "vx_ptx.cuh"
#include "vx_quant_math.cuh"

namespace vx {

namespace {
int check_rows(const vx_kv_rows* rows, int page_size, KvRows& r) {
  if (!rows || rows->struct_size != static_cast<int32_t>(sizeof(vx_kv_rows))) return fail(-1, "vx_kv_rows: struct_size");
  if (rows->reserved != 0) return fail(-1, "vx_kv_rows: reserved must be 0");
  constexpr int64_t kMax = (1ll << 31) - 1;
  if (rows->rows < 0 || rows->rows > kMax || rows->sequences < 0 || rows->sequences > kMax) return fail(-1, "vx_kv_rows: bad shape");
  if (!rows->row_offsets && rows->rows != rows->sequences)
    return fail(-1, "vx_kv_rows: without row_offsets every sequence has one row (rows %lld, sequences %lld)", (long long)rows->rows, (long long)rows->sequences);
  if (rows->table_pages < 0 || rows->table_pages > kMax / page_size) return fail(-1, "vx_kv_rows: a sequence may have up to 2^31 - 1 tokens");
  if (rows->rows > 0 && rows->sequences > 0) {
    if (!rows->lengths) return fail(-1, "vx_kv_rows: lengths must not be NULL");
    if (rows->table_pages > 0 && (!rows->page_table || rows->ld_table < rows->table_pages)) return fail(-1, "vx_kv_rows: page_table NULL or its rows too short");
  }
  r.rows = static_cast<int32_t>(rows->rows);
  r.sequences = static_cast<int32_t>(rows->sequences);
  r.lengths = rows->lengths;
  r.row_offsets = rows->row_offsets;
  r.table = {rows->page_table, rows->ld_table, static_cast<int32_t>(rows->table_pages)};
  return 0;
}
bool power_of_two(float x) {
  int e;
  return x >= 0x1p-32f && x <= 0x1p32f && frexpf(x, &e) == 0.5f;
}
}  // namespace

int check_paged(const vx_kv_cache* cache, const vx_kv_rows* rows, PagedCache& c, KvRows& r) {
  if (!cache || cache->struct_size != static_cast<int32_t>(sizeof(vx_kv_cache))) return fail(-1, "vx_kv_cache: struct_size");
  constexpr int64_t kMax = (1ll << 31) - 1;
  if (cache->page_size < 1 || cache->pages < 0 || cache->pages > kMax || cache->kv_heads < 1 || cache->kv_heads > 65535)
    return fail(-1, "vx_kv_cache: bad shape (pages %lld, page_size %d, kv_heads %d)", (long long)cache->pages, cache->page_size, cache->kv_heads);
  if (cache->pages > 0 && (!cache->k || !cache->v)) return fail(-1, "vx_kv_cache: k and v must not be NULL");
  const int64_t strides[] = {cache->k_page, cache->k_token, cache->k_head, cache->v_page, cache->v_token, cache->v_head};
  for (const int64_t s : strides)
    if (s < 0 || s % 8 != 0) return fail(-1, "vx_kv_cache: strides must be multiples of 8 elements");
  if (!aligned16(cache->k) || !aligned16(cache->v)) return fail(-1, "vx_kv_cache: k and v must be 16-byte aligned");
  if (const int rc = check_rows(rows, cache->page_size, r)) return rc;
  c.k = {static_cast<__nv_bfloat16*>(cache->k), cache->k_page, cache->k_token, cache->k_head};
  c.v = {static_cast<__nv_bfloat16*>(cache->v), cache->v_page, cache->v_token, cache->v_head};
  c.page_size = FastDiv(static_cast<uint32_t>(cache->page_size));
  c.pages = static_cast<int32_t>(cache->pages);
  return 0;
}

int check_paged(const vx_kv_cache_fp4* cache, const vx_kv_rows* rows, Fp4Cache& c, KvRows& r) {
  if (!cache || cache->struct_size != static_cast<int32_t>(sizeof(vx_kv_cache_fp4))) return fail(-1, "vx_kv_cache_fp4: struct_size");
  constexpr int64_t kMax = (1ll << 31) - 1;
  if (cache->page_size < 16 || cache->page_size % 16 != 0) return fail(-1, "vx_kv_cache_fp4: page_size must be a multiple of 16 (got %d)", cache->page_size);
  if (cache->pages < 0 || cache->pages > kMax || cache->kv_heads < 1 || cache->kv_heads > 65535)
    return fail(-1, "vx_kv_cache_fp4: bad shape (pages %lld, kv_heads %d)", (long long)cache->pages, cache->kv_heads);
  const int D = cache->head_dim;
  if (D < 16 || D > 256 || D % 16 != 0) return fail(-1, "head_dim must be a multiple of 16 up to 256 (got %d)", D);
  if (cache->pages > 0 && (!cache->k || !cache->v)) return fail(-1, "vx_kv_cache_fp4: k and v must not be NULL");
  if (!aligned16(cache->k) || !aligned16(cache->v)) return fail(-1, "vx_kv_cache_fp4: k and v must be 16-byte aligned");
  const int64_t page = static_cast<int64_t>(cache->kv_heads) * (cache->page_size / kFp4Tokens) * kFp4Unit * D;
  for (const int64_t s : {cache->k_page, cache->v_page})
    if (s % 16 != 0 || s < 0 || (cache->pages > 1 && s < page)) return fail(-1, "vx_kv_cache_fp4: pages must be a multiple of 16 bytes apart, %lld or more", (long long)page);
  if (!power_of_two(cache->k_scale) || !power_of_two(cache->v_scale)) return fail(-1, "k_scale and v_scale must be powers of two from 2^-32 to 2^32");
  if (const int rc = check_rows(rows, cache->page_size, r)) return rc;
  c = {static_cast<uint8_t*>(cache->k), static_cast<uint8_t*>(cache->v), cache->k_page, cache->v_page, cache->k_scale, cache->v_scale,
       FastDiv(static_cast<uint32_t>(cache->page_size / kFp4Tokens)), static_cast<int32_t>(cache->pages)};
  return 0;
}

namespace {

constexpr int AP_THREADS = 256;
constexpr int AP_BLOCKS = 6;     // per SM, at 40 registers a thread: five of 46 take 375 us at the size above, seven or eight, which spill, 507
constexpr int AP_BLOCKS_FP4 = 5;  // at 48 registers (bf16 rows spill 28 bytes, fp32 rows 8): 384 us for four of 62 389, six 399 (and with 17 divisions for 16 values, four of them, 418)
constexpr int AP_UNITS = 16;     // of a thread in large calls, since a block looks its rows up before it moves any: 4 take 422 us there, 8 391, 16 375 (of five blocks)
constexpr int AP_MAX_ROWS = 32;  // rows of a block at most

struct AppendParams {
  PagedCache cache;
  Fp4Cache fp4;
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
  int32_t head_dim;
};

// where the rows of a block go
struct RowPlace {
  int64_t k, v;      // offset of the token's place in the cache, -1: not stored; FP4: of its unit of head 0, in bytes
  int32_t position;  // -1: left out
  int32_t token;     // FP4: of the unit
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

// Pieces of eight: the rotated values from c0 on of a key, every product and sum rounded (the bytes of a cache in 4 bits are then a function of the inputs
// and not of how a compiler contracts them).
template <typename T>
__device__ __forceinline__ void rotated8(const AppendParams& p, const T* src, const float* cs, int c0, float (&x)[8]) {
  load8(src + c0, x);
  const int rot = 16 * p.rot_units;
  if (c0 >= rot) return;
  if (p.half) {
    const bool second = c0 >= p.half;
    float y[8], c[8], s[8];
    load8(src + (second ? c0 - p.half : c0 + p.half), y);
    load8(cs + (second ? c0 - p.half : c0), c);
    load8(cs + (second ? c0 : c0 + p.half), s);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = __fmul_rn(x[j], c[j]), b = __fmul_rn(y[j], s[j]);
      x[j] = second ? __fadd_rn(a, b) : __fsub_rn(a, b);
    }
  } else {
    const float4 c = *reinterpret_cast<const float4*>(cs + c0 / 2), s = *reinterpret_cast<const float4*>(cs + rot / 2 + c0 / 2);
    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = x[2 * j], o = x[2 * j + 1];
      x[2 * j] = __fsub_rn(__fmul_rn(e, cc[j]), __fmul_rn(o, ss[j]));
      x[2 * j + 1] = __fadd_rn(__fmul_rn(o, cc[j]), __fmul_rn(e, ss[j]));
    }
  }
}

// Sixteen values to codes and their scale.  The quotient by the scale is rounded to fp32 first: a value whose significand has 24 bits at most, over a scale whose
// significand has 4, is a border between two codes exactly or is off it by more than half a unit, so the code is that of the exact quotient.  A
// quotient is formed from the correctly rounded reciprocal and one remainder step (Markstein, IBM J. Res. Dev. 34(1), 1990, see Nv16Tensor); below fp32's
// normal range it is far below the first border.  (17 divisions instead: see AP_BLOCKS_FP4.)
__device__ __forceinline__ uint2 quantize16(const float (&a)[8], const float (&b)[8], float inv_g, uint32_t& byte) {
  const float most = __fmul_rn(fmaxf(amax8(a), amax8(b)), inv_g);
  constexpr float kSixth = 1.0f / 6.0f;  // correctly rounded
  const float sixth = __fmul_rn(most, kSixth);
  byte = __nv_cvt_float_to_fp8(most < 1e30f ? __fmaf_rn(__fmaf_rn(-sixth, 6.0f, most), kSixth, sixth) : most, __NV_SATFINITE, __NV_E4M3) & 0x7fu;
  const float s = e4m3_to_float(byte);
  if (byte == 0) return make_uint2(0, 0);
  const float r = __frcp_rn(s);
  const uint64_t g2 = pack_f32x2(inv_g, inv_g), r2 = pack_f32x2(r, r), s2 = pack_f32x2(-s, -s);
  uint32_t w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint64_t x = mul_f32x2(e ? pack_f32x2(b[j], b[j + 1]) : pack_f32x2(a[j], a[j + 1]), g2), q0 = mul_f32x2(x, r2);
      unpack_f32x2(fma_f32x2(fma_f32x2(q0, s2, x), r2, q0), q[j], q[j + 1]);
    }
    if (!(most < INFINITY)) {  // (infinities, which have no remainder: to the largest codes of their signs)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = __fmul_rn(e ? b[j] : a[j], inv_g);
        if (!(fabsf(x) < INFINITY)) q[j] = x;
      }
    }
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w[e])
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  }
  return make_uint2(w[0], w[1]);
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(AP_THREADS, FP4 ? AP_BLOCKS_FP4 : AP_BLOCKS) kv_append_kernel(const __grid_constant__ AppendParams p) {
  pdl_launch_dependents();
  __shared__ RowPlace place[AP_MAX_ROWS];
  const int row0 = static_cast<int>(blockIdx.x) * p.rows_per_block;
  const int n_rows = min(p.rows_per_block, p.rows.rows - row0);
  pdl_wait();
  if (static_cast<int>(threadIdx.x) < n_rows) {
    RowPlace pl{-1, -1, -1, 0};
    int s;
    int64_t i;
    if (row_sequence(p.rows, row0 + threadIdx.x, s, i)) {
      const int64_t t = p.rows.lengths[s] + i;
      const int64_t pos = t + (p.starts ? p.starts[s] : 0);
      if (!p.rotary) pl.position = 0;
      else if (pos >= 0 && pos < p.positions) pl.position = static_cast<int32_t>(pos);
      if (pl.position >= 0 && t < (1ll << 31)) {
        uint32_t index, slot;
        if (FP4) p.fp4.page_units.divmod(static_cast<uint32_t>(t) / kFp4Tokens, index, slot);
        else p.cache.page_size.divmod(static_cast<uint32_t>(t), index, slot);
        const int page = page_of(p.rows.table, s, index, FP4 ? p.fp4.pages : p.cache.pages);
        if (page >= 0) {
          pl.k = FP4 ? page * p.fp4.k_page + static_cast<int64_t>(slot) * (kFp4Unit * p.head_dim) : page * p.cache.k.page + slot * p.cache.k.token;
          pl.v = FP4 ? page * p.fp4.v_page + static_cast<int64_t>(slot) * (kFp4Unit * p.head_dim) : page * p.cache.v.page + slot * p.cache.v.token;
          pl.token = static_cast<int32_t>(t % kFp4Tokens);
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
    if (FP4 && static_cast<int>(head) >= p.q_heads) {  // 16 values of a scale
      head -= p.q_heads;
      const bool key = static_cast<int>(head) < p.kv_heads;
      if (!key) head -= p.kv_heads;
      if ((key ? pl.k : pl.v) < 0) continue;
      const int c = 16 * static_cast<int>(u), D = p.head_dim;
      uint8_t* const at = (key ? p.fp4.k + pl.k : p.fp4.v + pl.v) + static_cast<int64_t>(head) * p.fp4.page_units.d * (kFp4Unit * D);
      float a[8], b[8];
      if (key) {
        const T* const x = static_cast<const T*>(p.k) + row * p.k_row + head * p.k_head;
        const float* const cs = p.rotary + pl.position * p.ld_rotary;
        rotated8(p, x, cs, c, a);
        rotated8(p, x, cs, c + 8, b);
      } else {
        const T* const x = static_cast<const T*>(p.v) + row * p.v_row + head * p.v_head + c;
        load8(x, a);
        load8(x + 8, b);
      }
      uint32_t byte;
      *reinterpret_cast<uint2*>(at + pl.token * (D / 2) + c / 2) = quantize16(a, b, key ? 1.0f / p.fp4.k_scale : 1.0f / p.fp4.v_scale, byte);
      at[8 * D + pl.token * (D / 16) + u] = static_cast<uint8_t>(byte);
      continue;
    }
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

// What the entry points share: the rest of the parameters, the launch.  `cache` has been checked; D, kv_heads: its own.
template <bool FP4>
int append(AppendParams& p, const vx_kv_append_desc* d, int D, int kv_heads, void* stream) {
  if (!d || d->struct_size != static_cast<int32_t>(sizeof(vx_kv_append_desc))) return fail(-1, "vx_kv_append_desc: struct_size");
  if (d->reserved != 0) return fail(-1, "vx_kv_append_desc: reserved must be 0");
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
  if (!FP4) {
    const int64_t extent[3] = {p.cache.pages, static_cast<int64_t>(p.cache.page_size.d), kv_heads};
    const int64_t k_step[3] = {p.cache.k.page, p.cache.k.token, p.cache.k.head}, v_step[3] = {p.cache.v.page, p.cache.v.token, p.cache.v.head};
    for (int i = 0; i < 3; ++i)
      if (extent[i] > 1 && (k_step[i] < D || v_step[i] < D)) return fail(-1, "two tokens or heads of the cache in one place (stride below head_dim)");
  }
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
  p.kv_heads = kv_heads;
  p.head_dim = D;
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
  if (d->dtype == VX_F32) VX_CUDA_OK(launch_dependent(kv_append_kernel<float, FP4>, grid, dim3(AP_THREADS), 0, st, p));
  else VX_CUDA_OK(launch_dependent(kv_append_kernel<__nv_bfloat16, FP4>, grid, dim3(AP_THREADS), 0, st, p));
  return 0;
}

// Values of a cache in 4 bits: a thread takes the 16 values of a scale, 32 bytes of the result; neighbours follow each other in a head of a token.
struct ValuesParams {
  const uint8_t* pages;
  int64_t page_bytes, total;  // total: scales
  float scale;
  int32_t head_dim;
  FastDiv per_head, per_token, tokens;
  __nv_bfloat16* out;
};
// WIDE: more than 2^31 scales, with divisions of 64 bits.
template <bool WIDE>
__global__ void __launch_bounds__(256) kv_values_kernel(const __grid_constant__ ValuesParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int D = p.head_dim;
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; n < p.total; n += static_cast<int64_t>(gridDim.x) * 256) {
    // page, token, head, scale of the head
    const uint32_t per_token = p.per_token.d;
    int64_t page;
    uint32_t head, u, token, in_token;
    if (WIDE) {
      const int64_t place = n / per_token;
      in_token = static_cast<uint32_t>(n - place * per_token);
      page = place / p.tokens.d;
      token = static_cast<uint32_t>(place - page * p.tokens.d);
    } else {
      uint32_t place, page32;
      p.per_token.divmod(static_cast<uint32_t>(n), place, in_token);
      p.tokens.divmod(place, page32, token);
      page = page32;
    }
    p.per_head.divmod(in_token, head, u);
    const uint8_t* const unit = p.pages + page * p.page_bytes + (static_cast<int64_t>(head) * (p.tokens.d / kFp4Tokens) + token / kFp4Tokens) * (kFp4Unit * D);
    token %= kFp4Tokens;
    const uint2 codes = *reinterpret_cast<const uint2*>(unit + token * (D / 2) + u * 8);
    const float s = __half2float(__ushort_as_half(static_cast<unsigned short>(e4m3_as_half(unit[8 * D + token * (D / 16) + u])))) * 256.0f * p.scale;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t h[4];
      e2m1_as_half(j ? codes.y : codes.x, h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
        const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * s, f.y * s);
        w[4 * j + e] = *reinterpret_cast<const uint32_t*>(&b);
      }
    }
    uint4* const dst = reinterpret_cast<uint4*>(p.out + n * 16);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

}  // namespace
}  // namespace vx

extern "C" int vx_kv_append(const vx_kv_cache* cache, const vx_kv_rows* rows, const vx_kv_append_desc* d, void* stream) {
  using namespace vx;
  AppendParams p{};
  const int rc = check_paged(cache, rows, p.cache, p.rows);
  return rc ? rc : append<false>(p, d, cache->head_dim, cache->kv_heads, stream);
}

extern "C" int vx_kv_append_fp4(const vx_kv_cache_fp4* cache, const vx_kv_rows* rows, const vx_kv_append_desc* d, void* stream) {
  using namespace vx;
  AppendParams p{};
  const int rc = check_paged(cache, rows, p.fp4, p.rows);
  return rc ? rc : append<true>(p, d, cache->head_dim, cache->kv_heads, stream);
}

extern "C" int vx_kv_values_fp4(const void* pages, int64_t n_pages, int64_t page_bytes, int page_size, int kv_heads, int head_dim, float scale, void* out,
                                void* stream) {
  using namespace vx;
  vx_kv_cache_fp4 cache{};
  cache.struct_size = sizeof(cache);
  cache.page_size = page_size;
  cache.pages = n_pages;
  cache.kv_heads = kv_heads;
  cache.head_dim = head_dim;
  cache.k = cache.v = const_cast<void*>(pages);
  cache.k_page = cache.v_page = page_bytes;
  cache.k_scale = cache.v_scale = scale;
  vx_kv_rows rows{};
  rows.struct_size = sizeof(rows);
  Fp4Cache c;
  KvRows r;
  if (const int rc = check_paged(&cache, &rows, c, r)) return rc;
  if (n_pages == 0) return 0;
  if (!out || !aligned16(out)) return fail(-1, "out must be 16-byte aligned");
  ValuesParams p{c.k, page_bytes, n_pages * page_size * kv_heads * (head_dim / 16), scale, head_dim, FastDiv(static_cast<uint32_t>(head_dim / 16)),
                 FastDiv(static_cast<uint32_t>(kv_heads * (head_dim / 16))), FastDiv(static_cast<uint32_t>(page_size)), static_cast<__nv_bfloat16*>(out)};
  const int64_t blocks = (p.total + 255) / 256, most = 64 * static_cast<int64_t>(sm_count());
  VX_CUDA_OK(launch_dependent(p.total < (1ll << 31) ? kv_values_kernel<false> : kv_values_kernel<true>, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, static_cast<cudaStream_t>(stream), p));
  return 0;
}
