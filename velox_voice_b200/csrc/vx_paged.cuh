// Paged cache of keys and values: what the kernels that write it (vx_kv_append.cu) and read it (vx_prefix_attn.cu) share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "vx_common.cuh"

namespace vx {

// n / d and n % d for 0 <= n < 2^31 and a divisor known on the host.  With s = ceil(log2 d) and m = floor(2^(31 + s) / d) + 1,
// n / d = floor(n m / 2^(31 + s)): m d exceeds 2^(31 + s) by at most d <= 2^s, an error of n m / 2^(31 + s) below n 2^s / (d 2^(31 + s)) < 1 / d.
struct FastDiv {
  uint32_t d, mul, shift;  // mul 0: d = 1
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), mul(0), shift(0) {
    if (d <= 1) return;
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    mul = static_cast<uint32_t>((1ull << (31 + s)) / d) + 1;
    shift = s - 1;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return mul == 0 ? n : __umulhi(n, mul) >> shift; }
  __device__ __forceinline__ void divmod(uint32_t n, uint32_t& q, uint32_t& r) const {
    q = div(n);
    r = n - q * d;
  }
};

// One run of tokens per owner (sequence or group) through a table of pages.
struct PagedTable {
  const int32_t* table;
  int64_t ld;
  int32_t pages;  // entries per owner
};

// One of the two tensors of a cache.
struct PagedTensor {
  __nv_bfloat16* p;
  int64_t page, token, head;  // strides in elements
};

struct PagedCache {
  PagedTensor k, v;
  FastDiv page_size;
  int32_t pages;
};

// Rows and sequences of a call.  Whatever the device memory behind it holds, indexes formed from it stay in range.
struct KvRows {
  int32_t rows, sequences;
  const int32_t* lengths;
  const int32_t* row_offsets;
  PagedTable table;
};

// Largest s in [0, n) with offsets[s] <= x, and 0 if there is none.
__device__ __forceinline__ int find_owner(const int32_t* offsets, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Largest o in [0, n) with first(o) <= x (first ascending), and 0 if there is none, by a whole warp: 32 places a turn instead of one, each
// turn one round trip to memory (120 sequences: 2 instead of 7, 3 us of a CTA that lives for 8).
template <class First>
__device__ __forceinline__ int find_by_warp(int n, int x, First first) {
  const unsigned lane = threadIdx.x & 31;
  unsigned lo = 0, hi = n;  // (unsigned: lo + 31 step can pass 2^31)
  while (hi - lo > 1) {
    const unsigned step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, lane == 0 || (at < hi && first(static_cast<int>(at)) <= x));
    lo += (31 - __clz(below)) * step;
    hi = min(hi, lo + step);
  }
  return static_cast<int>(lo);
}

// Sequence of a row and the row's index among the new tokens of that sequence, from its offset, which may lie in front of the call's rows; false:
// no sequence, or one that takes no part.
// WARP: all lanes of the warp ask for the same row.
template <bool WARP = false>
__device__ __forceinline__ bool row_sequence(const KvRows& kr, int row, int& s, int64_t& i) {
  s = row;
  i = 0;
  if (kr.sequences == 0) return false;
  if (kr.row_offsets) {
    if (WARP) s = find_by_warp(kr.sequences, row, [&](int o) { return kr.row_offsets[o]; });
    else s = find_owner(kr.row_offsets, kr.sequences, row);
    i = static_cast<int64_t>(row) - kr.row_offsets[s];
    if (i < 0 || row >= kr.row_offsets[s + 1]) return false;
  }
  return kr.lengths[s] >= 0;
}

// Page of an owner's token t, or -1: not there.
__device__ __forceinline__ int page_of(const PagedTable& t, int owner, uint32_t index, int32_t pages) {
  if (index >= static_cast<uint32_t>(t.pages)) return -1;
  const int page = t.table[static_cast<int64_t>(owner) * t.ld + index];
  return page >= 0 && page < pages ? page : -1;
}

// Checks of the descriptors that both entry points make; 0 or an error code.
int check_paged(const vx_kv_cache* cache, const vx_kv_rows* rows, PagedCache& c, KvRows& r);
// Element strides and address of a bf16 / fp32 operand whose 16-byte pieces are read whole.
inline bool pieces_ok(const void* p, int64_t a, int64_t b, int elem) { return aligned16(p) && a * elem % 16 == 0 && b * elem % 16 == 0; }
// A result [rows, heads, head_dim] whose rows or heads lie in one place.
inline bool shares_places(int64_t rows, int64_t row, int64_t heads, int64_t head, int head_dim) {
  return (rows > 1 && row < head_dim && row > -head_dim) || (heads > 1 && head < head_dim && head > -head_dim);
}

}  // namespace vx
