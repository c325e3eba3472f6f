// Drafted tokens against the target's probabilities (vx_verify_drafts), in two launches:
//
//   verify_rows_kernel   a cluster per row: the row's largest logit and the sum of 2^((x - max) c), c = log2(e) / T, of the target and of the drafter, in
//                        one pass in fp32; from them whether the row's draft stands.  The exponentials come out within 2^-16 (a difference, c and a product, 2^-24 each of an
//                        exponent up to 128), their sums, 16 or more of a thread at a time, each time rounded and, where the maximum moves, multiplied by an exponential (2^-22),
//                        within 2^-16 + vocab 1.25 2^-33 more at worst, so where u q(d) and p(d) are 2^-12 + vocab 2^-31 of each other apart the comparison is settled; the
//                        others, some 1 of 4,000, are left open.
//   verify_next_kernel   a cluster per sequence: the first row whose draft falls (open rows settled in fp64), and the token drawn from what is left there:
//                        sums of both rows, then of max(p - q, 0) in ascending order -- CTA, warp, group of 32, lane -- in fp64, since a token stands or falls
//                        with one comparison of a sum over the vocabulary: with 131,071 tokens and fp32 sums one draw of ten would be near a border.
//
// What bounds them: the first, HBM (384 rows of 131,071 in fp32 and 320 of the drafter's, 369 MB in 71 us by ncu, 5.2 TB/s); the second, 66 us there (127 both, in a call), latency: two walks in
// fp64, nine operations a logit, that keep half of the issue slots busy, and the clusters' barriers between them; small calls the round trips to memory: 50 rows of
// 5,538 take 11.5 us in both together.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "vx_common.cuh"
#include "vx_paged.cuh"
#include "vx_ptx.cuh"

namespace vx {
namespace {

constexpr int VR_THREADS = 128;  // rows of 5,538 have three pieces of 16 bytes a thread: 256 threads, of which an SM holds half as many rows, take 27.8 us for 26.5 with 1,038 rows
constexpr int VN_THREADS = 512;
constexpr int VR_CTAS = 8;     // per SM at least, of rows, at 64 registers: eight loads of 16 bytes a thread are on their way.  Ten and twelve, at 48 and 40, where bf16 rows spill, take 131 and 136 us for the
                               // 127 of a call with 64 sequences of six rows of 131,071 in fp32, 30.2 and 33.9 for 26.6 with 1,038 rows of 5,538 in bf16
constexpr int VR_LEAST = 4096, VN_LEAST = 4096;  // values of a CTA, where a row is cut
constexpr unsigned ALL = 0xffffffffu;

enum Draft : int32_t { kFalls = 0, kStands = 1, kOpen = 2 };

// What the first launch leaves of a row.
struct RowFinding {
  float most, draft_most;  // largest logits; most NaN: nothing is drawn from the row
  int32_t draft;           // Draft
  int32_t best;            // temperature 0: its first largest token, -1: none
};

struct VerifyParams {
  const void *logits, *draft_logits;
  int64_t ld, ld_draft;
  const void* ids;
  int32_t ids64;
  int32_t rows, vocab, sequences;
  const float2* uniforms;
  const int32_t* row_offsets;
  double log2e_t;  // log2(e) / temperature
  int32_t greedy;
  int32_t *accepted, *next;
  RowFinding* found;
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ int64_t id_at(const VerifyParams& p, int row) {
  return p.ids64 ? static_cast<const int64_t*>(p.ids)[row] : static_cast<const int32_t*>(p.ids)[row];
}
__device__ __forceinline__ int first_row_of(const VerifyParams& p, int s) { return p.row_offsets ? min(max(p.row_offsets[s], 0), p.rows) : s; }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename V>
__device__ __forceinline__ V ld_cluster(const V* p, uint32_t rank) {  // of the same variable of another CTA
  static_assert(sizeof(V) == 8 || sizeof(V) == 4, "");
  const uint32_t a = map_to_cta(smem_u32(p), rank);
  V v;
  if constexpr (sizeof(V) == 8) {
    uint64_t x;
    asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(x) : "r"(a) : "memory");
    memcpy(&v, &x, 8);
  } else {
    uint32_t x;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
    memcpy(&v, &x, 4);
  }
  return v;
}

// ---------------------------------------------------------------- rows

// Maximum and sum of a part of a row, of this thread; and, for temperature 0, the first place of the maximum.
struct Running {
  float m = -INFINITY, sum = 0.0f;
  float ref = 0.0f;  // m, 0 for -infinity
  int at = 0x7fffffff;
};

// N values, in ascending order; `at`: place of the first, the next PIECE follow it, those behind are `step` further
template <bool GREEDY, int PIECE, int N>
__device__ __forceinline__ void take(Running& r, const float (&x)[N], int at, int step, float c) {
  float m = x[0];
#pragma unroll
  for (int j = 1; j < N; ++j) m = fmaxf(m, x[j]);
  if (GREEDY) {
    // (NaN: the sum tells)
#pragma unroll
    for (int j = 0; j < N; ++j) r.sum += x[j] != x[j] ? 1.0f : 0.0f;
    if (m > r.m || (m == r.m && at < r.at)) {  // (the values around the pieces come last)
      r.m = m;
#pragma unroll
      for (int j = N - 1; j >= 0; --j)
        if (x[j] == m) r.at = at + j / PIECE * step + j % PIECE;
    }
  } else {
    if (m > r.m) {
      r.sum *= ex2((r.m - m) * c);
      r.m = m;
      r.ref = m;
    }
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j & 1] += ex2((x[j] - r.ref) * c);  // (x c - m c in one operation is off by 2^-24 of m c, and m c is not bounded)
    r.sum += sum[0] + sum[1];
  }
}
template <bool GREEDY>
__device__ __forceinline__ void join(Running& a, float m, float sum, int at, float c) {
  if (GREEDY) {
    a.sum += sum;
    if (m > a.m || (m == a.m && at < a.at)) a.at = at;
    a.m = fmaxf(a.m, m);
  } else {
    const float top = fmaxf(a.m, m), ref = top == -INFINITY ? 0.0f : top;
    a.sum = a.sum * ex2((a.m - ref) * c) + sum * ex2((m - ref) * c);
    a.m = top;
  }
}

// 16-byte pieces of a row from the first aligned one on, values in front and behind one by one; pieces first, first + step, ...
template <typename T>
struct RowPieces {
  static constexpr int N = 16 / sizeof(T);
  const T* row;
  int head, pieces, rest;  // values in front of the pieces, pieces, values around them
  __device__ __forceinline__ RowPieces(const T* r, int n) : row(r) {
    head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / static_cast<int>(sizeof(T)), n);
    pieces = (n - head) / N;
    rest = n - pieces * N;
  }
  __device__ __forceinline__ uint4 load(int i) const {  // behind the end: -infinity
    constexpr uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
    return i < pieces ? reinterpret_cast<const uint4*>(row + head)[i] : make_uint4(none, none, none, none);
  }
  __device__ __forceinline__ static void convert(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      } else {
        x[j] = __uint_as_float(w[j]);
      }
    }
  }
  __device__ __forceinline__ int rest_at(int i) const { return i < head ? i : pieces * N + i; }  // where the i-th value around the pieces is
};

// One or two rows (SIDES) together: all that is loaded of a turn is on its way before any of it is used.
template <typename T, bool GREEDY, int SIDES>
__device__ __forceinline__ void walk(Running (&r)[2], const T* const (&rows)[2], int n, int first, int step, float c) {
  using Pieces = RowPieces<T>;
  constexpr int AHEAD = 4;
  const Pieces p[2] = {Pieces(rows[0], n), Pieces(rows[SIDES - 1], n)};
  const int most = SIDES == 2 ? max(p[0].pieces, p[1].pieces) : p[0].pieces;
  float edge[2];
  bool has[2] = {};
#pragma unroll
  for (int e = 0; e < SIDES; ++e) {  // (fewer than 2 N values)
    has[e] = first < p[e].rest;
    edge[e] = has[e] ? to_float(rows[e][p[e].rest_at(first)]) : -INFINITY;
  }
#pragma unroll 1
  for (int i = first; i < most; i += AHEAD * step) {
    uint4 u[SIDES][AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a)
#pragma unroll
      for (int e = 0; e < SIDES; ++e) u[e][a] = p[e].load(i + a * step);
#pragma unroll
    for (int e = 0; e < SIDES; ++e) {
      float x[AHEAD * Pieces::N];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) Pieces::convert(u[e][a], x + a * Pieces::N);
      take<GREEDY, Pieces::N>(r[e], x, p[e].head + i * Pieces::N, step * Pieces::N, c);
    }
  }
#pragma unroll
  for (int e = 0; e < SIDES; ++e)
    if (has[e]) {
      const float x[1] = {edge[e]};
      take<GREEDY, 1>(r[e], x, p[e].rest_at(first), 0, c);
    }
}

template <typename T, bool GREEDY>
__global__ void __launch_bounds__(VR_THREADS, VR_CTAS) verify_rows_kernel(const __grid_constant__ VerifyParams p, int ctas) {
  pdl_launch_dependents();
  __shared__ float m_s[2][VR_THREADS / 32], sum_s[2][VR_THREADS / 32];
  __shared__ int at_s[VR_THREADS / 32];
  __shared__ float out_m[2], out_sum[2];
  __shared__ int out_at;
  const int row = static_cast<int>(blockIdx.x) / ctas, rank = static_cast<int>(blockIdx.x) - row * ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  // the row's sequence: its last row has no draft
  int s = row;
  bool last = true, there = p.sequences > 0;
  if (p.row_offsets && there) {
    s = find_by_warp(p.sequences, row, [&](int o) { return p.row_offsets[o]; });
    const int end = first_row_of(p, s + 1);
    there = row >= first_row_of(p, s) && row < end;
    last = row == end - 1;
  }
  if (!there) return;  // (all CTAs of the cluster)
  const float c = GREEDY ? 1.0f : static_cast<float>(p.log2e_t);
  const T* const row_t = static_cast<const T*>(p.logits) + row * p.ld;
  const bool drafter = !GREEDY && p.draft_logits && !last;
  const T* const row_d = drafter ? static_cast<const T*>(p.draft_logits) + row * p.ld_draft : row_t;
  // (of the draft, for the end: on its way with the rows)
  const int64_t draft = last ? -1 : id_at(p, row + 1);
  const bool known = draft >= 0 && draft < p.vocab;
  const float u = p.uniforms[row].x, draft_t = known ? to_float(row_t[draft]) : 0.0f, draft_d = known ? to_float(row_d[draft]) : 0.0f;
  Running r[2];
  const T* const rows[2] = {row_t, row_d};
  if (drafter) walk<T, GREEDY, 2>(r, rows, p.vocab, rank * VR_THREADS + threadIdx.x, ctas * VR_THREADS, c);
  else walk<T, GREEDY, 1>(r, rows, p.vocab, rank * VR_THREADS + threadIdx.x, ctas * VR_THREADS, c);
#pragma unroll
  for (int e = 0; e < (GREEDY ? 1 : 2); ++e) {
    if (e == 1 && !drafter) break;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m = __shfl_xor_sync(ALL, r[e].m, o), sum = __shfl_xor_sync(ALL, r[e].sum, o);
      join<GREEDY>(r[e], m, sum, GREEDY ? __shfl_xor_sync(ALL, r[e].at, o) : 0, c);
    }
    if (lane == 0) {
      m_s[e][warp] = r[e].m;
      sum_s[e][warp] = r[e].sum;
      if (GREEDY) at_s[warp] = r[e].at;
    }
  }
  __syncthreads();
  const int sides = drafter ? 2 : 1;
  if (threadIdx.x < sides) {
    Running a;
    for (int w = 0; w < VR_THREADS / 32; ++w) join<GREEDY>(a, m_s[threadIdx.x][w], sum_s[threadIdx.x][w], GREEDY ? at_s[w] : 0, c);
    out_m[threadIdx.x] = a.m;
    out_sum[threadIdx.x] = a.sum;
    if (GREEDY) out_at = a.at;
  }
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  if (rank == 0 && threadIdx.x == 0) {
    Running a[2];
    for (int e = 0; e < sides; ++e) {
      if (ctas == 1) {
        a[e].m = out_m[e];
        a[e].sum = out_sum[e];
        a[e].at = GREEDY ? out_at : 0;
      } else {
        for (int k = 0; k < ctas; ++k) join<GREEDY>(a[e], ld_cluster(&out_m[e], k), ld_cluster(&out_sum[e], k), GREEDY ? ld_cluster(&out_at, k) : 0, c);
      }
    }
    RowFinding f{a[0].m, a[1].m, kFalls, -1};
    auto sound = [](const Running& r) { return r.sum > 0.0f && r.sum < INFINITY && fabsf(r.m) < INFINITY; };  // (NaN among the logits: the sum is)
    if (!GREEDY && !(sound(a[0]) && (!drafter || sound(a[1])))) f.most = NAN;  // nothing is drawn from this row
    if (GREEDY) {
      // (a maximum that is not finite, or NaN among the logits: none)
      f.best = a[0].sum == 0.0f && fabsf(a[0].m) < INFINITY ? a[0].at : -1;
      if (known && f.best == draft) f.draft = kStands;
    } else if (known && f.most == f.most) {
      const float pt = ex2((draft_t - a[0].m) * c), qd = drafter ? ex2((draft_d - a[1].m) * c) : 1.0f;
      const float left = u * qd * a[0].sum, right = pt * (drafter ? a[1].sum : 1.0f), gap = fmaxf(left, right) * (0x1p-12f + 0x1p-31f * static_cast<float>(p.vocab));
      // (anything near the end of the range is open)
      if (!(left > 1e-30f && right > 1e-30f && left < 1e30f && right < 1e30f) || fabsf(left - right) <= gap) f.draft = kOpen;
      else f.draft = left < right ? kStands : kFalls;
    }
    p.found[row] = f;
  }
  if (ctas > 1) cluster_sync_all();  // (a CTA's shared memory is read by the first)
}

// ---------------------------------------------------------------- the token behind

// 2^y = 2^floor(n / 1024) 2^(n mod 1024 / 1024) 2^r with n = 1024 y rounded, |r| <= 1 / 2048: the second factor from a table, which a block makes of two of
// 32, the third by its Taylor series to r^3 (the next term is below 2^-50).  (A table of 64 and a series to r^5: three of eleven fp64 operations more.)
constexpr int kExpTable = 1024;
__device__ const double kCoarse[32] = {  // 2^(k / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
__device__ const double kFine[32] = {  // 2^(k / 1024)
    1.0, 1.0006771306930664, 1.0013547198921082, 1.002032767907594, 1.0027112750502025, 1.0033902416308227, 1.004069667960554, 1.0047495543507072,
    1.0054299011128027, 1.006110708558573, 1.0067919769999607, 1.0074737067491204, 1.0081558981184175, 1.0088385514204294, 1.0095216669679448, 1.0102052450739643,
    1.0108892860517005, 1.011573790214578, 1.0122587578762337, 1.0129441893505169, 1.0136300849514894, 1.0143164449934257, 1.0150032697908125, 1.0156905596583505,
    1.016378314910953, 1.0170665358637463, 1.0177552228320703, 1.0184443761314785, 1.019133996077738, 1.0198240829868295, 1.0205146371749483, 1.0212056589585028};

// 2^((x - at) c) for x <= at; 0 below 2^-1000.  (The difference first: it is exact, or as near as its own size asks for; x c and at c are not bounded.)
struct Weight {
  double c, at;
  float c32, at32;
  __device__ __forceinline__ double operator()(const double* tab, float x) const {
    constexpr double big = 6755399441055744.0 / kExpTable;  // 1.5 2^52 / 1024: the last bit of a sum is 1 / 1024
    const double y = static_cast<double>(x) - at, t = fma(y, c, big), r = fma(y, c, -(t - big));
    const int n = __double2loint(t);
    constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3;
    const double s = tab[n & (kExpTable - 1)], v = fma(s, fma(fma(c3, r, c2), r, c1) * r, s);
    const int high = __double2hiint(v) + ((n >> 10) << 20);
    return (x - at32) * c32 >= -1000.0f ? __hiloint2double(high, __double2loint(v)) : 0.0;
  }
};

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}
__device__ __forceinline__ double warp_scan(double x) {  // the sum up to this lane, its own included
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(ALL, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// The tokens of a CTA are a run of the vocabulary, those of its warps runs of that, and a warp takes 32 neighbours at a time: sums by warps are sums in
// ascending order, whose first to pass a number tells the warp that has the token.  (That warp's run, 2,048 of 131,071 tokens in a cluster of four, walked by the
// warp alone took some 10 us.)
template <typename T>
__global__ void __launch_bounds__(VN_THREADS, 2) verify_next_kernel(const __grid_constant__ VerifyParams p, int ctas) {
  pdl_launch_dependents();
  constexpr int WARPS = VN_THREADS / 32, AHEAD = 4;
  __shared__ double tab[kExpTable];
  __shared__ double warp_s[2][2][WARPS], cta_s[2][2];  // each in turn, so that one barrier per exchange is enough
  const int s = static_cast<int>(blockIdx.x) / ctas, rank = static_cast<int>(blockIdx.x) - s * ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kExpTable; i += VN_THREADS) tab[i] = kCoarse[i >> 5] * kFine[i & 31];
  pdl_wait();
  const int row0 = first_row_of(p, s), row1 = first_row_of(p, s + 1), drafts = row1 - row0 - 1;
  const bool writer = rank == 0 && threadIdx.x == 0;
  if (drafts < 0) {
    if (writer) {
      p.accepted[s] = 0;
      p.next[s] = -1;
    }
    return;
  }
  // The first draft from one on that does not stand for certain, and what was found of its row: 32 rows at a time, a lane each.
  RowFinding found;
  auto first_doubt = [&](int from) {
    while (true) {
      const int n = min(drafts - from + 1, 32);  // (with the row behind the last draft)
      const RowFinding f = p.found[row0 + from + min(lane, n - 1)];
      const unsigned doubt = __ballot_sync(ALL, lane < n && (f.draft != kStands || from + lane == drafts));
      if (doubt) {
        const int at = __ffs(doubt) - 1;
        found.most = __shfl_sync(ALL, f.most, at);
        found.draft_most = __shfl_sync(ALL, f.draft_most, at);
        found.draft = __shfl_sync(ALL, f.draft, at);
        found.best = __shfl_sync(ALL, f.best, at);
        return from + at;
      }
      from += n;
    }
  };
  if (p.greedy) {
    if (warp == 0 && rank == 0) {
      const int i = first_doubt(0);
      if (lane == 0) {
        p.accepted[s] = i;
        p.next[s] = found.best;
      }
    }
    return;
  }
  // this warp's tokens
  const int each = ((p.vocab + ctas * WARPS - 1) / (ctas * WARPS) + 31) / 32 * 32;
  const int v0 = min((rank * WARPS + warp) * each, p.vocab), v1 = min(v0 + each, p.vocab);
  int turn = 0;
  // a and b, the warps' own, summed over the cluster; what lane w keeps: a of warp w and of those up to it, in this CTA; lane k: of CTA k and of those up to it
  double warp_own, warp_up, cta_own, cta_up;
  auto sums_of_warps = [&](double a) {
    turn ^= 1;
    if (lane == 0) warp_s[turn][0][warp] = a;
    __syncthreads();
    warp_own = lane < WARPS ? warp_s[turn][0][lane] : 0.0;
    warp_up = warp_scan(warp_own);
  };
  auto sum_all = [&](double& a, double& b) {
    if (lane == 0) warp_s[turn ^ 1][1][warp] = b;
    sums_of_warps(a);
    a = __shfl_sync(ALL, warp_up, 31);
    b = warp_sum(lane < WARPS ? warp_s[turn][1][lane] : 0.0);
    cta_own = cta_up = a;
    if (ctas > 1) {
      if (threadIdx.x == 0) {
        cta_s[turn][0] = a;
        cta_s[turn][1] = b;
      }
      cluster_sync_all();
      cta_own = lane < ctas ? ld_cluster(&cta_s[turn][0], lane) : 0.0;
      b = warp_sum(lane < ctas ? ld_cluster(&cta_s[turn][1], lane) : 0.0);
      cta_up = warp_scan(cta_own);
      a = __shfl_sync(ALL, cta_up, 31);
    } else if (lane > 0) {
      cta_own = 0.0;
    }
  };
  // The row that is looked at: weights of its tokens, times 2^(largest logit c); the drafter's
  const double c = p.log2e_t;
  const T *t, *d;   // d: NULL without a drafter
  Weight wt, wd;
  int sure;         // the draft, where the drafter was sure of it; -1: none
  auto begin_row = [&](int i) {
    const int row = row0 + i;
    t = static_cast<const T*>(p.logits) + row * p.ld;
    d = i < drafts && p.draft_logits ? static_cast<const T*>(p.draft_logits) + row * p.ld_draft : nullptr;
    wt = {c, found.most, static_cast<float>(c), found.most};
    wd = {c, found.draft_most, static_cast<float>(c), found.draft_most};
    sure = -1;
    if (i < drafts && !p.draft_logits) {
      const int64_t id = id_at(p, row + 1);
      if (id >= 0 && id < p.vocab) sure = static_cast<int>(id);
    }
  };
  // What is left of a token's weight: the target's less `ratio` of the drafter's, where that is above 0, nothing for the token `out`.  One body for the sums
  // (ratio 0) and for what is drawn from: what is fetched for the first time costs here.  BOTH: there is a drafter.
  double ratio = 0.0;
  int out = -1;
  auto left_of = [&](auto both, int v, float x, float y, double& drafter) {
    double w = wt(tab, x);
    if (decltype(both)::value) {
      drafter = wd(tab, y);
      w = fma(drafter, -ratio, w);
      if (__double2hiint(w) < 0) w = 0.0;
    }
    return v == out ? 0.0 : w;
  };
  // sums over this warp's tokens, 32 at a time in ascending order, the next AHEAD groups on their way
  auto walk_row = [&](auto both, double& a, double& b) {
    constexpr bool BOTH = decltype(both)::value;
    float x[AHEAD], y[AHEAD];
    auto load = [&](int v) {
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {  // (behind the end: of no weight)
        x[e] = v + 32 * e < v1 ? to_float(t[v + 32 * e]) : -INFINITY;
        y[e] = BOTH && v + 32 * e < v1 ? to_float(d[v + 32 * e]) : -INFINITY;
      }
    };
    double sum[2] = {0.0, 0.0}, other[2] = {0.0, 0.0};
    load(v0 + lane);
#pragma unroll 1
    for (int v = v0 + lane; v - lane < v1; v += 32 * AHEAD) {
      float x0[AHEAD], y0[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        x0[e] = x[e];
        y0[e] = y[e];
      }
      load(v + 32 * AHEAD);
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        double drafter = 0.0;
        sum[e & 1] += left_of(both, v + 32 * e, x0[e], y0[e], drafter);
        other[e & 1] += drafter;
      }
    }
    a = warp_sum(sum[0] + sum[1]);
    b = BOTH ? warp_sum(other[0] + other[1]) : 0.0;
  };
  __syncthreads();  // (the table)
  int i = first_doubt(0), chosen = -1;
  enum { kSums, kRest, kAll } what = kSums;     // what is summed up
  if (found.most == found.most) begin_row(i);
#pragma unroll 1
  while (found.most == found.most) {            // (uniform over the cluster; NaN: nothing is drawn from the row)
    double all, others;
    if (d) walk_row(std::true_type{}, all, others);
    else walk_row(std::false_type{}, all, others);
    sum_all(all, others);
    if (what == kSums) {
      if (i < drafts && found.draft == kOpen) {
        const int64_t id = id_at(p, row0 + i + 1);
        if (id >= 0 && id < p.vocab) {
          const double left = static_cast<double>(p.uniforms[row0 + i].x) * (d ? wd(tab, to_float(d[id])) / others : 1.0);
          if (left < wt(tab, to_float(t[id])) / all) {
            i = first_doubt(i + 1);
            begin_row(i);
            continue;
          }
        }
      }
      what = kAll;
      if (d || sure >= 0) {
        what = kRest;
        ratio = d ? all / others : 0.0;
        out = sure;
        continue;
      }
    } else if (what == kRest && !(all > 0.0)) {  // nothing is left: p
      what = kAll;
      ratio = 0.0;
      out = -1;
      continue;
    }
    const double target = static_cast<double>(p.uniforms[row0 + i].y) * all;
    // The first part whose sum passes the target has the token; a number that is not below 1 (or rounding) can leave none: then the last with a weight.
    double before = 0.0;
    bool exact = true;
    auto holder_of = [&](double part, double up) {  // of a lane's part and those up to it; `before` moves on to what is in front of it
      const unsigned has = __ballot_sync(ALL, part > 0.0), over = exact ? __ballot_sync(ALL, before + up > target) & has : 0;
      exact = over != 0;
      const int at = over ? __ffs(over) - 1 : 31 - __clz(has);
      const double front = __shfl_sync(ALL, up, max(at - 1, 0));
      if (at > 0) before += front;
      return at;
    };
    if (holder_of(cta_own, cta_up) != rank) break;
    // The run of the CTA's warp that has it, walked again by all of the CTA's, and of that the warp's that has it, until a warp's part is what it holds.
    int holder = holder_of(warp_own, warp_up), run0 = min((rank * WARPS + max(holder, 0)) * each, p.vocab), run1 = min(run0 + each, p.vocab);
    while (true) {
      const int part = ((run1 - run0 + WARPS - 1) / WARPS + 31) / 32 * 32, w0 = min(run0 + warp * part, run1), w1 = min(w0 + part, run1);
      double x[AHEAD] = {}, sum = 0.0;
#pragma unroll 1
      for (int v = w0; v < w1; v += 32 * AHEAD) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
          const int at = v + 32 * e + lane;
          double drafter;
          const float l = at < w1 ? to_float(t[at]) : -INFINITY;
          x[e] = d ? left_of(std::true_type{}, at, l, at < w1 ? to_float(d[at]) : -INFINITY, drafter) : left_of(std::false_type{}, at, l, 0.0f, drafter);
        }
        sum += (x[0] + x[1]) + (x[2] + x[3]);
      }
      sums_of_warps(warp_sum(sum));
      holder = max(holder_of(warp_own, warp_up), 0);
      if (part <= 32 * AHEAD) {
        if (warp == holder) {
#pragma unroll
          for (int e = 0; e < AHEAD; ++e) {  // groups of 32 neighbours
            const double up = warp_scan(x[e]);
            const unsigned has = __ballot_sync(ALL, x[e] > 0.0), over = exact ? __ballot_sync(ALL, before + up > target) & has : 0;
            if (over) {
              chosen = w0 + 32 * e + __ffs(over) - 1;
              break;
            }
            if (has) chosen = w0 + 32 * e + 31 - __clz(has);
            before += __shfl_sync(ALL, up, 31);
          }
        }
        break;
      }
      run0 = min(run0 + holder * part, run1);
      run1 = min(run0 + part, run1);
    }
    break;
  }
  if (chosen < 0 ? writer && found.most != found.most : lane == 0) {
    p.accepted[s] = i;
    p.next[s] = chosen;
  }
  if (ctas > 1) cluster_sync_all();  // (shared memory of a CTA that ended is not read)
}

// Launch in clusters of `ctas`.
template <typename K>
cudaError_t launch_clusters(K kernel, int64_t owners, int ctas, int threads, cudaStream_t st, const VerifyParams& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(owners * ctas));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (ctas > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim = {static_cast<unsigned>(ctas), 1, 1};
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(n);
  return cudaLaunchKernelEx(&cfg, kernel, p, ctas);
}
// CTAs per owner: as many as leave no more than `most` in all and each `least` values or more
int cluster_size(int64_t owners, int64_t most, int64_t values, int64_t least) {
  int c = 1;
  while (c < 8 && 2 * c * owners <= most && values >= 2 * c * least) c *= 2;
  return c;
}

}  // namespace
}  // namespace vx

extern "C" int64_t vx_verify_drafts_scratch(int64_t rows) { return rows < 0 ? -1 : rows * static_cast<int64_t>(sizeof(vx::RowFinding)); }

extern "C" int vx_verify_drafts(const vx_verify_desc* d, void* stream) {
  using namespace vx;
  if (!d || d->struct_size != static_cast<int32_t>(sizeof(vx_verify_desc))) return fail(-1, "vx_verify_desc: struct_size");
  if (d->reserved != 0) return fail(-1, "vx_verify_desc: reserved must be 0");
  if (d->dtype != VX_F32 && d->dtype != VX_BF16) return fail(-1, "dtype must be VX_F32 or VX_BF16");
  if (d->ids_bytes != 4 && d->ids_bytes != 8) return fail(-1, "ids must be i32 or i64 (ids_bytes %d)", d->ids_bytes);
  constexpr int64_t kMax = (1ll << 27);
  if (d->rows < 0 || d->rows > kMax || d->sequences < 0 || d->sequences > kMax || d->vocab < 1 || d->vocab > (1 << 24))
    return fail(-1, "bad shape (rows %lld, sequences %lld, vocab %lld)", (long long)d->rows, (long long)d->sequences, (long long)d->vocab);
  if (!d->row_offsets && d->rows != d->sequences)
    return fail(-1, "without row_offsets every sequence has one row (rows %lld, sequences %lld)", (long long)d->rows, (long long)d->sequences);
  if (!(d->temperature == 0.0 || (d->temperature >= 0x1p-20 && d->temperature <= 0x1p20))) return fail(-1, "temperature must be 0 or from 2^-20 to 2^20");
  if (d->sequences == 0) return 0;
  if (!d->accepted || !d->next) return fail(-1, "accepted and next must not be NULL");
  const int es = d->dtype == VX_F32 ? 4 : 2;
  if (d->rows > 0) {
    if (!d->logits || !d->ids || !d->uniforms) return fail(-1, "logits, ids and uniforms must not be NULL");
    if (reinterpret_cast<uintptr_t>(d->logits) % es || reinterpret_cast<uintptr_t>(d->draft_logits) % es || reinterpret_cast<uintptr_t>(d->uniforms) % 8 ||
        reinterpret_cast<uintptr_t>(d->ids) % d->ids_bytes)
      return fail(-1, "logits, ids and uniforms must be aligned to their elements (uniforms to a pair)");
    if (d->ld_logits < d->vocab || (d->draft_logits && d->ld_draft < d->vocab)) return fail(-1, "rows of logits are shorter than the vocabulary");
    if (!d->scratch || !aligned16(d->scratch) || d->scratch_bytes < vx_verify_drafts_scratch(d->rows))
      return fail(-1, "scratch must be %lld bytes, 16-byte aligned", (long long)vx_verify_drafts_scratch(d->rows));
  }
  VerifyParams p{};
  p.logits = d->logits; p.ld = d->ld_logits;
  p.draft_logits = d->draft_logits; p.ld_draft = d->ld_draft;
  p.ids = d->ids; p.ids64 = d->ids_bytes == 8;
  p.rows = static_cast<int32_t>(d->rows); p.vocab = static_cast<int32_t>(d->vocab); p.sequences = static_cast<int32_t>(d->sequences);
  p.uniforms = reinterpret_cast<const float2*>(d->uniforms);
  p.row_offsets = d->row_offsets;
  p.greedy = d->temperature == 0.0;
  p.log2e_t = p.greedy ? 1.0 : 1.4426950408889634074 / d->temperature;
  p.accepted = d->accepted; p.next = d->next;
  p.found = static_cast<RowFinding*>(d->scratch);
  const auto st = static_cast<cudaStream_t>(stream);
  const bool f32 = d->dtype == VX_F32;
  if (d->rows > 0) {
    const int ctas = cluster_size(d->rows, 24 * static_cast<int64_t>(sm_count()), d->vocab, VR_LEAST);
    auto kernel = p.greedy ? (f32 ? verify_rows_kernel<float, true> : verify_rows_kernel<__nv_bfloat16, true>)
                           : (f32 ? verify_rows_kernel<float, false> : verify_rows_kernel<__nv_bfloat16, false>);
    VX_CUDA_OK(launch_clusters(kernel, d->rows, ctas, VR_THREADS, st, p));
  }
  const int ctas = p.greedy ? 1 : cluster_size(d->sequences, 2 * static_cast<int64_t>(sm_count()), d->vocab, VN_LEAST);
  VX_CUDA_OK(launch_clusters(f32 ? verify_next_kernel<float> : verify_next_kernel<__nv_bfloat16>, d->sequences, ctas, VN_THREADS, st, p));
  return 0;
}
