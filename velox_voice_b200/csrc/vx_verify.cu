// Drafted tokens against the target's probabilities (vx_verify_drafts), in two launches:
//
//   verify_rows_kernel   a cluster per row: the row's largest logit and the sum of 2^((x - max) c), c = log2(e) / T, of the target and of the drafter, in
//                        one pass in fp32; from them whether the row's draft stands.  p(d) and q(d) come out within 2^-17 (2^-24 of the exponent, up to 128,
//                        in each of the two exponentials; sums of positive terms, the exponents of those that count small), so where u q(d) and
//                        p(d) are 2^-12 of each other apart the comparison is settled; the others, some 1 of 4,000, are left open.
//   verify_next_kernel   a cluster per sequence: the first row whose draft falls (open rows settled in fp64), and the token drawn from what is left there:
//                        sums of both rows, then of max(p - q, 0) in ascending order -- CTA, thread, token -- in fp64, since a token stands or falls with
//                        one comparison of a sum over the vocabulary: with 131,071 tokens and fp32 sums one draw of ten would be near a border.
//
// 2^y in fp64: y = n / 64 + r, |r| <= 1 / 128, 2^(n mod 64 / 64) from a table, 2^r by its Taylor series to r^5 (the next term is below 2^-54).

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "vx_common.cuh"
#include "vx_paged.cuh"
#include "vx_ptx.cuh"

namespace vx {
namespace {

constexpr int VR_THREADS = 256;
constexpr int VN_THREADS = 512;
constexpr unsigned ALL = 0xffffffffu;

enum Draft : int32_t { kFalls = 0, kStands = 1, kOpen = 2 };

// What the first launch leaves of a row.
struct RowFinding {
  float most, draft_most;  // largest logits
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
  int at = 0x7fffffff;
};

template <bool GREEDY, int N>
__device__ __forceinline__ void take(Running& r, const float (&x)[N], int at, float c) {
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
        if (x[j] == m) r.at = at + j;
    }
  } else {
    if (m > r.m) {
      r.sum *= ex2((r.m - m) * c);
      r.m = m;
    }
    const float ref = r.m == -INFINITY ? 0.0f : r.m;
#pragma unroll
    for (int j = 0; j < N; ++j) r.sum += ex2((x[j] - ref) * c);
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
template <typename T, bool GREEDY>
__device__ __forceinline__ void walk(Running& r, const T* row, int n, int first, int step, float c) {
  constexpr int N = 16 / sizeof(T), AHEAD = 4;
  const int head = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int>(sizeof(T)), n);
  const int pieces = (n - head) / N;
  auto convert = [](const uint4& u, float (&x)[N]) {
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
  };
  const uint4* const src = reinterpret_cast<const uint4*>(row + head);
  int i = first;
  for (; i + (AHEAD - 1) * step < pieces; i += AHEAD * step) {
    uint4 u[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) u[a] = src[i + a * step];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      float x[N];
      convert(u[a], x);
      take<GREEDY>(r, x, head + (i + a * step) * N, c);
    }
  }
  for (; i < pieces; i += step) {
    float x[N];
    convert(src[i], x);
    take<GREEDY>(r, x, head + i * N, c);
  }
  // the values around the pieces, of which there are fewer than 2 N
  const int rest = head + (n - head - pieces * N);
  if (first < rest) {
    const int at = first < head ? first : head + pieces * N + first - head;
    const float x[1] = {to_float(row[at])};
    take<GREEDY>(r, x, at, c);
  }
}

template <typename T, bool GREEDY>
__global__ void __launch_bounds__(VR_THREADS) verify_rows_kernel(const __grid_constant__ VerifyParams p, int ctas) {
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
  Running r[2];
#pragma unroll
  for (int e = 0; e < (GREEDY ? 1 : 2); ++e) {
    if (e == 1 && !drafter) break;
    walk<T, GREEDY>(r[e], e ? row_d : row_t, p.vocab, rank * VR_THREADS + threadIdx.x, ctas * VR_THREADS, c);
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
    const int64_t d = last ? -1 : id_at(p, row + 1);
    const bool known = d >= 0 && d < p.vocab;
    if (GREEDY) {
      // (a maximum that is not finite, or NaN among the logits: none)
      f.best = a[0].sum == 0.0f && fabsf(a[0].m) < INFINITY ? a[0].at : -1;
      if (known && f.best == d) f.draft = kStands;
    } else if (known) {
      const float pt = ex2((to_float(row_t[d]) - a[0].m) * c), qd = drafter ? ex2((to_float(row_d[d]) - a[1].m) * c) : 1.0f;
      const float left = p.uniforms[row].x * qd * a[0].sum, right = pt * (drafter ? a[1].sum : 1.0f), gap = fmaxf(left, right) * 0x1p-12f;
      // (anything that is NaN, infinite or near the end of the range is open)
      if (!(left > 1e-30f && right > 1e-30f && left < 1e30f && right < 1e30f) || fabsf(left - right) <= gap) f.draft = kOpen;
      else f.draft = left < right ? kStands : kFalls;
    }
    p.found[row] = f;
  }
  if (ctas > 1) cluster_sync_all();  // (a CTA's shared memory is read by the first)
}

// ---------------------------------------------------------------- the token behind

struct Exp2Table {
  double t[64];
};
// 2^y for y <= 0
__device__ __forceinline__ double exp2_fp64(const Exp2Table& tab, double y) {
  if (!(y >= -1020.0)) return y != y ? y : 0.0;
  const double big = 6755399441055744.0 / 64.0;  // 1.5 2^52 / 64: the last bit of a sum is 1 / 64
  const double t = y + big, r = y - (t - big);
  const int n = __double2loint(t);
  constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4, c5 = c4 * c1 / 5;
  const double s = tab.t[n & 63], q = fma(fma(fma(fma(c5, r, c4), r, c3), r, c2), r, c1) * r, v = fma(s, q, s);
  return __hiloint2double(__double2hiint(v) + ((n >> 6) << 20), __double2loint(v));
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}

template <typename T>
__global__ void __launch_bounds__(VN_THREADS) verify_next_kernel(const __grid_constant__ VerifyParams p, int ctas) {
  pdl_launch_dependents();
  __shared__ Exp2Table tab;
  __shared__ double warp_s[2][VN_THREADS / 32], cta_s[2][2];  // cta_s: in turn, so that one cluster barrier per exchange is enough
  const int s = static_cast<int>(blockIdx.x) / ctas, rank = static_cast<int>(blockIdx.x) - s * ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < 64) tab.t[threadIdx.x] = exp2(threadIdx.x / 64.0);
  __syncthreads();
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
  if (p.greedy) {
    if (writer) {
      int i = 0;
      while (i < drafts && p.found[row0 + i].draft == kStands) ++i;
      p.accepted[s] = i;
      p.next[s] = p.found[row0 + i].best;
    }
    return;
  }
  // this thread's tokens, in a row
  const int each = (p.vocab + ctas * VN_THREADS - 1) / (ctas * VN_THREADS);
  const int v0 = min((rank * VN_THREADS + static_cast<int>(threadIdx.x)) * each, p.vocab), v1 = min(v0 + each, p.vocab);
  int turn = 0;
  // a and b summed over the cluster, the CTAs' a in front of this one in `before`
  auto sum_all = [&](double& a, double& b, double& before) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane == 0) {
      warp_s[0][warp] = a;
      warp_s[1][warp] = b;
    }
    __syncthreads();
    a = b = before = 0.0;
    for (int w = 0; w < VN_THREADS / 32; ++w) {
      a += warp_s[0][w];
      b += warp_s[1][w];
    }
    if (ctas > 1) {
      turn ^= 1;
      if (threadIdx.x == 0) {
        cta_s[turn][0] = a;
        cta_s[turn][1] = b;
      }
      cluster_sync_all();
      a = b = 0.0;
      for (int k = 0; k < ctas; ++k) {
        if (k == rank) before = a;
        a += ld_cluster(&cta_s[turn][0], k);
        b += ld_cluster(&cta_s[turn][1], k);
      }
    }
    __syncthreads();
  };
  struct Row {
    const T *t, *d;
    double mt, md, zt, zd;
    int64_t draft;  // the token, where the drafter was sure; -1: none
  };
  auto weight_t = [&](const Row& r, int v) { return exp2_fp64(tab, (static_cast<double>(to_float(r.t[v])) - r.mt) * p.log2e_t); };
  auto weight_d = [&](const Row& r, int v) { return exp2_fp64(tab, (static_cast<double>(to_float(r.d[v])) - r.md) * p.log2e_t); };
  auto open_row = [&](int row, bool last) {  // with the sums of both sides
    Row r{static_cast<const T*>(p.logits) + row * p.ld, nullptr, p.found[row].most, 0.0, 0.0, 0.0, -1};
    if (!last && p.draft_logits) {
      r.d = static_cast<const T*>(p.draft_logits) + row * p.ld_draft;
      r.md = p.found[row].draft_most;
    } else if (!last) {
      r.draft = id_at(p, row + 1);
    }
    double a = 0.0, b = 0.0, before;
#pragma unroll 4
    for (int v = v0; v < v1; ++v) {
      a += weight_t(r, v);
      if (r.d) b += weight_d(r, v);
    }
    sum_all(a, b, before);
    r.zt = a;
    r.zd = b;
    return r;
  };
  int i = 0;
  Row r;
  bool opened = false;
  for (; i < drafts; ++i) {
    const int found = p.found[row0 + i].draft;
    opened = false;
    if (found == kStands) continue;
    if (found == kFalls) break;
    r = open_row(row0 + i, false);
    opened = true;
    const int64_t d = id_at(p, row0 + i + 1);
    if (d < 0 || d >= p.vocab) break;
    const double left = static_cast<double>(p.uniforms[row0 + i].x) * (r.d ? weight_d(r, static_cast<int>(d)) / r.zd : 1.0);
    if (!(left < weight_t(r, static_cast<int>(d)) / r.zt)) break;
  }
  const int row = row0 + i;
  if (!(opened && i < drafts)) r = open_row(row, i == drafts);
  // what is drawn from
  const bool rest = r.d != nullptr || r.draft >= 0;
  const double inv_t = 1.0 / r.zt, inv_d = r.d ? 1.0 / r.zd : 0.0;
  auto left_at = [&](int v, bool rest) {
    double x = weight_t(r, v) * inv_t;
    if (rest && r.d) x = fmax(x - weight_d(r, v) * inv_d, 0.0);
    else if (rest && v == r.draft) x = 0.0;
    return x;
  };
  int chosen = -1;
  const bool sound = r.zt > 0.0 && r.zt < INFINITY && (!r.d || (r.zd > 0.0 && r.zd < INFINITY));
  for (int pass = rest ? 0 : 1; sound && pass < 2; ++pass) {  // (uniform over the cluster)
    double mine = 0.0, unused = 0.0, before;
#pragma unroll 4
    for (int v = v0; v < v1; ++v) mine += left_at(v, pass == 0);
    // sums in front of this thread
    double up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(ALL, up, o);
      if (lane >= o) up += y;
    }
    double all = mine;
    sum_all(all, unused, before);
    if (!(all > 0.0)) continue;
    for (int w = 0; w < warp; ++w) before += warp_s[0][w];
    const double target = static_cast<double>(p.uniforms[row].y) * all;
    // The first thread whose sum passes the target has the token; rounding, or a number that is not below 1, can leave none: then the last with a weight.
    const bool passes = before + up > target, weighs = mine > 0.0;
    __shared__ int first_s[2], seen_s[2][2];
    if (threadIdx.x == 0) first_s[0] = 0x7fffffff, first_s[1] = -1;
    __syncthreads();
    const unsigned who = __ballot_sync(ALL, passes && weighs), weigh = __ballot_sync(ALL, weighs);
    if (lane == 0) {
      if (who) atomicMin(&first_s[0], warp * 32 + __ffs(who) - 1);
      if (weigh) atomicMax(&first_s[1], warp * 32 + 31 - __clz(weigh));
    }
    __syncthreads();
    int from = first_s[0], lastly = first_s[1], owner = from != 0x7fffffff ? rank : -1;
    bool exact = from != 0x7fffffff;
    if (ctas > 1) {
      if (threadIdx.x == 0) seen_s[pass][0] = from, seen_s[pass][1] = lastly;
      cluster_sync_all();
      owner = -1;
      int fallback = -1;
      for (int k = ctas - 1; k >= 0; --k) {
        if (ld_cluster(&seen_s[pass][0], k) != 0x7fffffff) owner = k;
        if (fallback < 0 && ld_cluster(&seen_s[pass][1], k) >= 0) fallback = k;
      }
      exact = owner >= 0;
      if (!exact) owner = fallback;
    } else if (!exact) {
      owner = 0;
    }
    if (owner == rank) {
      const int thread = exact ? from : lastly;
      if (warp == thread >> 5) {  // its tokens by the lanes of the warp
        const double base = __shfl_sync(ALL, before + up - mine, thread & 31);
        const int a0 = __shfl_sync(ALL, v0, thread & 31), a1 = __shfl_sync(ALL, v1, thread & 31);
        double sum = base;
        int pick = -1, heavy = -1;
        for (int v = a0; v < a1 && pick < 0; v += 32) {
          double x = v + lane < a1 ? left_at(v + lane, pass == 0) : 0.0;
          const unsigned has = __ballot_sync(ALL, x > 0.0);
          if (has) heavy = v + 31 - __clz(has);
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(ALL, x, o);
            if (lane >= o) x += y;
          }
          const unsigned over = __ballot_sync(ALL, sum + x > target) & has;
          if (over && exact) pick = v + __ffs(over) - 1;
          sum += __shfl_sync(ALL, x, 31);
        }
        chosen = pick >= 0 ? pick : heavy;
        if (lane == 0) {
          p.accepted[s] = i;
          p.next[s] = chosen;
        }
      }
    }
    if (ctas > 1) cluster_sync_all();
    return;
  }
  if (writer) {
    p.accepted[s] = i;
    p.next[s] = -1;
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
// CTAs per owner: while SMs would be left without one and each has `least` values
int cluster_size(int64_t owners, int64_t values, int64_t least) {
  int c = 1;
  while (c < 8 && 2 * c * owners <= 2 * static_cast<int64_t>(sm_count()) && values >= 2 * c * least) c *= 2;
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
    const int ctas = cluster_size(d->rows, d->vocab, 2048);
    auto kernel = p.greedy ? (f32 ? verify_rows_kernel<float, true> : verify_rows_kernel<__nv_bfloat16, true>)
                           : (f32 ? verify_rows_kernel<float, false> : verify_rows_kernel<__nv_bfloat16, false>);
    VX_CUDA_OK(launch_clusters(kernel, d->rows, ctas, VR_THREADS, st, p));
  }
  const int ctas = p.greedy ? 1 : cluster_size(d->sequences, d->vocab, VN_THREADS);
  VX_CUDA_OK(launch_clusters(f32 ? verify_next_kernel<float> : verify_next_kernel<__nv_bfloat16>, d->sequences, ctas, VN_THREADS, st, p));
  return 0;
}
