// Token-routed experts: the router, the order of the routed rows, and the copies into and out of that order.
//
//   eri_expert_route_fwd / _bwd   the k largest scores of a row (ties: the lower index) with softmax weights, and the gradient
//   eri_expert_plan               stable counting sort of the chosen experts: offsets and the row of every choice
//   eri_expert_scatter            xs[rows[t, j]] = x[t]                      (into expert order)
//   eri_expert_gather             out[t] = sum_j w[t, j] y[rows[t, j]]       (back; w == nullptr: all ones, the scatter's gradient)
//   eri_expert_gather_bwd         dy[rows[t, j]] = w[t, j] dout[t], dw[t, j] = <dout[t], y[rows[t, j]]>
//
// A choice outside [0, E) (padding) has row -1: it is neither copied nor added, whatever its neighbours hold. Rows from offsets[E]
// on belong to nobody and are written as zeros. Nothing is added with atomics: every result has one writer and one order of sums.
#include <limits.h>

#include "ptx.cuh"

using namespace eri;
typedef __nv_bfloat16 bf16;

namespace {

ERI_DEBUG_BOUNDS_DEFINE(expert_route)

constexpr int kMaxExperts = 1024, kMaxTop = 32;

// e^x for x <= 0 with a relative error near 2^-23: x = n ln2 + r with |r| <= ln2 / 2 (ln2 as the sum of a value of 12 bits,
// whose product with n is exact, and a rest), Taylor's series of e^r to r^7 (remainder below 2^-27). The special-function unit's
// 2^x would leave |x| 2^-24 of its argument's rounding in weights that are returned in 32 bits. Below -87: 0.
__device__ __forceinline__ float exp_nonpos(float x) {
  if (!(x >= -87.f)) return x != x ? x : 0.f;
  const float n = rintf(x * 1.4426950408889634f);
  float r = fmaf(n, -0.693115234375f, x);
  r = fmaf(n, -3.1946184945309e-05f, r);
  float p = 1.f / 5040.f;
  p = fmaf(p, r, 1.f / 720.f);
  p = fmaf(p, r, 1.f / 120.f);
  p = fmaf(p, r, 1.f / 24.f);
  p = fmaf(p, r, 1.f / 6.f);
  p = fmaf(p, r, 0.5f);
  p = fmaf(p, r, 1.f);
  p = fmaf(p, r, 1.f);
  return __int_as_float(__float_as_int(p) + ((int)n << 23));
}

// Order of the scores as unsigned integers: -0 equals +0, every NaN is the largest, 0 is no score at all.
__device__ __forceinline__ uint32_t score_key(float s) {
  const uint32_t b = __float_as_uint(s);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) return 0x80000000u;
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_score(uint32_t k) {
  if (k == 0xffffffffu) return __int_as_float(0x7fffffff);
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ float load_score(const float* s) { return *s; }
__device__ __forceinline__ float load_score(const bf16* s) { return __bfloat162float(*s); }
__device__ __forceinline__ void store_score(float* d, float v) { *d = v; }
__device__ __forceinline__ void store_score(bf16* d, float v) { *d = __float2bfloat16(v); }

constexpr float kNegInf = -__builtin_huge_valf();

// Softmax denominator of a row relative to its largest score m (not -inf): NaN when the row holds a NaN or +inf.
template <int VPL>
__device__ __forceinline__ float row_sum(const float (&v)[VPL], float m) {
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) z += exp_nonpos(v[i] - m);
  return warp_sum(z);
}

// One warp per token; lane l holds the scores of experts l, l + 32, ... in registers. Each of the k rounds is a maximum over the
// lanes' best keys and a minimum over the indices that reach it (two warp reductions), so equal scores come out in
// ascending order. Bound by instruction issue for k rounds of VPL + 2 reductions; the scores are read once.
template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_fwd_kernel(const T* __restrict__ scores, long long ld, const uint8_t* __restrict__ allowed,
                                                        long long* __restrict__ idx, float* __restrict__ w, int tokens, int E, int k,
                                                        int normalize) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= tokens) return;
  const T* s = scores + (long long)t * ld;
  float v[VPL];
  uint32_t key[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    const bool there = e < E;
    v[i] = there && (!allowed || allowed[e]) ? load_score(s + e) : kNegInf;
    key[i] = there ? score_key(v[i]) : 0u;
  }
  uint32_t my_key = 0u;
  int my_idx = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < VPL; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == top ? (uint32_t)(lane + 32 * at) : 0xffffffffu);
    if (lane == j) {
      my_key = top;
      my_idx = (int)e;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (e == (uint32_t)(lane + 32 * i)) key[i] = 0u;
  }
  const float val = key_score(my_key), m = __shfl_sync(0xffffffffu, val, 0);
  float z = lane < k ? exp_nonpos(val - m) : 0.f, sum;
  if (m == kNegInf) {              // a row that may choose nothing: no weight
    z = 0.f;
    sum = 1.f;
  } else {
    sum = normalize ? warp_sum(z) : row_sum<VPL>(v, m);
  }
  if (lane < k) {
    idx[(long long)t * k + lane] = my_idx;
    w[(long long)t * k + lane] = __fdiv_rn(z, sum);
  }
}

// normalize: ds = w_j (dw_j - <w, dw>) at the chosen, zero elsewhere. Otherwise ds = p (g - <w, dw>) with g = dw_j at the chosen.
template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_bwd_kernel(const T* __restrict__ scores, long long ld, const uint8_t* __restrict__ allowed,
                                                        const long long* __restrict__ idx, const float* __restrict__ w,
                                                        const float* __restrict__ dw, T* __restrict__ ds, int tokens, int E, int k,
                                                        int normalize) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t >= tokens) return;
  int my_idx = -1;
  float wj = 0.f, dj = 0.f;
  if (lane < k) {
    my_idx = (int)idx[(long long)t * k + lane];
    wj = w[(long long)t * k + lane];
    dj = dw[(long long)t * k + lane];
  }
  const float dot = warp_sum(wj * dj);
  float g[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) g[i] = 0.f;
  const float mine = normalize ? wj * (dj - dot) : dj;
  for (int j = 0; j < k; ++j) {
    const int e = __shfl_sync(0xffffffffu, my_idx, j);
    const float x = __shfl_sync(0xffffffffu, mine, j);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (e == lane + 32 * i) g[i] = x;
  }
  if (!normalize) {
    const T* s = scores + (long long)t * ld;
    float v[VPL], m = kNegInf;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      v[i] = e < E && (!allowed || allowed[e]) ? load_score(s + e) : kNegInf;
      nan |= v[i] != v[i];
      m = fmaxf(m, v[i]);
    }
    m = warp_max(m);
    if (__any_sync(0xffffffffu, nan)) m = __int_as_float(0x7fffffff);
    const float sum = m == kNegInf ? 1.f : row_sum<VPL>(v, m);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float p = m == kNegInf ? 0.f : __fdiv_rn(exp_nonpos(v[i] - m), sum);
      g[i] = p * (g[i] - dot);
    }
  }
  T* out = ds + (long long)t * E;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (lane + 32 * i < E) store_score(out + lane + 32 * i, !allowed || allowed[lane + 32 * i] ? g[i] : 0.f);
}

// ------------------------------------------------------------------------------------------- plan
// Stable counting sort by one cluster (one to eight CTAs of 32 warps). Every warp owns a consecutive piece of the choices and a
// private row of counters in shared memory: (1) it counts its piece, (2) the counters become prefix sums over the warps of a
// CTA, (3) the CTAs' totals are added over distributed shared memory, (4) the warp walks its piece again and hands out
// positions. Equal experts inside one group of 32 are found by ballots and ranked by the lanes below, so the order is that of the
// choices. A piece of at most kHold groups stays in registers between the two walks.
// Bound by instruction issue on its eight SMs (a ballot per bit and group of 32) and, for few choices, by its barriers: 49152
// choices of 64 experts take 11 us, 14 choices 2.5.
constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32, kHold = 8, kMaxCtas = 8;

__device__ __forceinline__ int load_choice(const void* idx, int wide, unsigned i, int E) {
  const long long e = wide ? reinterpret_cast<const long long*>(idx)[i] : (long long)reinterpret_cast<const int*>(idx)[i];
  return e >= 0 && e < E ? (int)e : -1;
}
__device__ __forceinline__ void load_group(int (&c)[kHold], const void* idx, int wide, unsigned i0, unsigned hi, int lane, int E) {
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const unsigned i = i0 + 32 * u + lane;         // (below 2^32: hi < 2^31)
    c[u] = i < hi ? load_choice(idx, wide, i, E) : -1;
  }
}
// Lanes of the warp whose choice is c's (one ballot per bit of an expert's number; lanes without a choice are nobody's).
__device__ __forceinline__ unsigned same_choice(int c, int bits) {
  unsigned m = __ballot_sync(0xffffffffu, c >= 0);
#pragma unroll 2
  for (int b = 0; b < bits; ++b) {
    const bool on = (c >> b) & 1;
    const unsigned v = __ballot_sync(0xffffffffu, on);
    m &= on ? v : ~v;
  }
  return m;
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {      // not ordered against other loads: all of a thread's are in flight
  int v;
  asm("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

__global__ void __launch_bounds__(kPlanThreads) expert_plan_kernel(const void* __restrict__ idx, int wide, int n, int E, int ctas,
                                                                   int* __restrict__ offsets, int* __restrict__ rows) {
  extern __shared__ int plan_smem[];
  int* total = plan_smem;                 // [E] this CTA's choices of every expert
  int* base = total + E;                  // [E] rows of lower CTAs of the expert
  int* first = base + E;                  // [E] first row of the expert
  int* cnt = first + E;                   // [kPlanWarps][E]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = ctas > 1 ? (int)cluster_ctarank() : 0;
  const int warps = ctas * kPlanWarps;
  const unsigned piece = (((unsigned)n + warps - 1) / warps + 31) / 32 * 32;
  const unsigned lo = (unsigned)min((unsigned long long)(rank * kPlanWarps + warp) * piece, (unsigned long long)n), hi = min(lo + piece, (unsigned)n);
  int* mine = cnt + (size_t)warp * E;
  const int bits = 32 - __clz(E - 1);
  int c[kHold];
  unsigned same[kHold];
  load_group(c, idx, wide, lo, hi, lane, E);
  for (int e = lane; e < E; e += 32) mine[e] = 0;
  __syncwarp();
  for (unsigned i0 = lo; i0 < hi; i0 += 32 * kHold) {
    if (i0 != lo) load_group(c, idx, wide, i0, hi, lane, E);
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      if (i0 + 32 * u < hi) {
        same[u] = same_choice(c[u], bits);
        if (c[u] >= 0 && lane == __ffs(same[u]) - 1) mine[c[u]] += __popc(same[u]);
        __syncwarp();
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kPlanThreads) {
    int sum = 0;
#pragma unroll 8
    for (int q = 0; q < kPlanWarps; ++q) {
      const int here = cnt[(size_t)q * E + e];
      cnt[(size_t)q * E + e] = sum;
      sum += here;
    }
    total[e] = sum;
  }
  if (ctas > 1) cluster_sync_all(); else __syncthreads();
  // every CTA adds up all totals itself
  for (int e = threadIdx.x; e < E; e += kPlanThreads) {
    int before = 0, all = 0;
    if (ctas > 1) {
      int x[kMaxCtas];
#pragma unroll
      for (int q = 0; q < kMaxCtas; ++q) x[q] = q < ctas ? ld_cluster(map_to_cta(smem_u32(total + e), (uint32_t)q)) : 0;
#pragma unroll
      for (int q = 0; q < kMaxCtas; ++q) {
        all += x[q];
        before += q < rank ? x[q] : 0;
      }
    } else {
      all = total[e];
    }
    first[e] = all;
    base[e] = before;
  }
  // no CTA leaves while another may read its totals: the wait is at the end
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane, all = e < E ? first[e] : 0;
      int scan = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += up;
      }
      if (e < E) {
        first[e] = run + scan - all;
        if (rank == 0) offsets[e] = run + scan - all;
      }
      run += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (lane == 0 && rank == 0) offsets[E] = run;
  }
  __syncthreads();
  const bool held = piece <= 32 * kHold;
  for (unsigned i0 = lo; i0 < hi; i0 += 32 * kHold) {
    if (!held) load_group(c, idx, wide, i0, hi, lane, E);
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
      if (i0 + 32 * u < hi) {
        const unsigned i = i0 + 32 * u + lane;
        if (!held) same[u] = same_choice(c[u], bits);
        int pos = -1;
        if (c[u] >= 0) pos = first[c[u]] + base[c[u]] + mine[c[u]] + __popc(same[u] & ((1u << lane) - 1u));
        __syncwarp();
        if (c[u] >= 0 && lane == __ffs(same[u]) - 1) mine[c[u]] += __popc(same[u]);
        __syncwarp();
        if (i < hi) {
          if (pos < 0 || ERI_DBG_INDEX(pos, n, 71)) rows[i] = pos;
        }
      }
    }
  }
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------------------------------------- copies
// A thread owns eight columns of one token. Rows come from the plan; one that is not in [0, n_rows) is skipped. 294 MB in 45 us, a copy's
// rate.
__global__ void __launch_bounds__(256) expert_scatter_kernel(const bf16* __restrict__ x, long long ldx, const int* __restrict__ rows,
                                                             const int* __restrict__ live, bf16* __restrict__ xs, long long items,
                                                             int vecs, int k, int n_rows, int D) {
  const long long stride = (long long)gridDim.x * blockDim.x;
  for (long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x; it < items; it += stride) {
    const long long t = it / vecs;
    const int c = (int)(it - t * vecs) * 8;
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(x + t * ldx + c);
    for (int j = 0; j < k; ++j) {
      const int r = rows[t * k + j];
      if (r >= 0 && r < n_rows) *reinterpret_cast<bf16x8*>(xs + (long long)r * D + c) = v;
    }
  }
  const int from = max(0, min(*live, n_rows));
  const long long rest = (long long)(n_rows - from) * vecs;
  bf16x8 z;
  z.u = make_uint4(0, 0, 0, 0);
  for (long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x; it < rest; it += stride)
    *reinterpret_cast<bf16x8*>(xs + (long long)from * D + it * 8) = z;
}

// out[t] = sum_j w[t, j] y[rows[t, j]] in 32 bits and ascending j, rounded once. A warp owns 512 columns of one token, a lane twice
// eight of them: the token's rows and weights are loaded once per warp and handed round, and eight loads of y are in flight per lane. 294 MB in
// 50 us (57 with one vector per thread).
constexpr int kFly = 4, kGatherCols = 512;
__global__ void __launch_bounds__(256) expert_gather_kernel(const bf16* __restrict__ y, long long ldy, const int* __restrict__ rows,
                                                            const float* __restrict__ w, bf16* __restrict__ out, long long items,
                                                            int chunks, int k, int n_rows, int D) {
  const int lane = threadIdx.x & 31;
  const long long stride = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long it = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += stride) {
    const long long t = it / chunks;
    const int c = (int)(it - t * chunks) * kGatherCols + lane * 8;
    const bool on0 = c < D, on1 = c + 256 < D;
    float acc[2][8];
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[0][q] = acc[1][q] = 0.f;
    for (int j0 = 0; j0 < k; j0 += 32) {
      int r = -1;
      float f = 1.f;
      if (j0 + lane < k) {
        r = rows[t * k + j0 + lane];
        if (w) f = w[t * k + j0 + lane];
        if (r >= n_rows) r = -1;
      }
      const int here = min(32, k - j0);
      for (int j = 0; j < here; j += kFly) {
        bf16x8 v[kFly][2];
        int ru[kFly];
#pragma unroll
        for (int u = 0; u < kFly; ++u) {
          ru[u] = j + u < here ? __shfl_sync(0xffffffffu, r, j + u) : -1;
          const bf16* src = y + (long long)ru[u] * ldy + c;
          if (ru[u] >= 0 && on0) v[u][0] = *reinterpret_cast<const bf16x8*>(src);
          if (ru[u] >= 0 && on1) v[u][1] = *reinterpret_cast<const bf16x8*>(src + 256);
        }
#pragma unroll
        for (int u = 0; u < kFly; ++u)
          if (ru[u] >= 0) {
            const float fu = __shfl_sync(0xffffffffu, f, j + u);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float a[8];
              unpack8(v[u][h], a);
#pragma unroll
              for (int q = 0; q < 8; ++q) acc[h][q] = fmaf(fu, a[q], acc[h][q]);
            }
          }
      }
    }
    if (on0) *reinterpret_cast<bf16x8*>(out + t * D + c) = pack8(acc[0]);
    if (on1) *reinterpret_cast<bf16x8*>(out + t * D + c + 256) = pack8(acc[1]);
  }
}

// dy[rows[t, j]] = w[t, j] dout[t] and dw[t, j] = <dout[t], y[rows[t, j]]>. `split` warps share a token, each 256 columns at a time: dout[t] and up to
// TOP of its rows come through a ring that the warp fills a piece ahead with asynchronous copies, across its tokens, so that reads do not
// wait for the stores of the piece before. The dot products are added in lane and warp order. Bound by DRAM with several rows per token, by
// issue with one. us, tokens x columns, rows per token: 8192 x 2560, 6: 89 to 98 (5.6 to 6.1 TB/s of reads and writes in equal parts; a CTA per
// token that loads into registers 105), 16384 x 2560, 2: 76 (139), 30000 x 1280, 1: 77 (159), 512 x 2560, 6: 7.5 (8.8). Three pieces:
// 4096 x 4096, 8: 94 instead of 100, but 512 x 2560 8.5; 16 warps per SM instead of 24: 16384 x 2560 84.
constexpr int kGbWarps = 8, kGbDepth = 2, kGbCols = 256, kGbRow = kGbCols * 2;
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Sums of TOP values over the warp, TOP - 1 + log2(32 / TOP) shuffles: lane l is left with the sum of value l / (32 / TOP).
template <int TOP>
__device__ __forceinline__ float warp_sums(float (&v)[TOP], int lane) {
#pragma unroll
  for (int n = TOP / 2, o = 16; n >= 1; n /= 2, o /= 2) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (int o = 16 / TOP; o >= 1; o /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}
template <int TOP>
__global__ void __launch_bounds__(kGbWarps * 32, 3) expert_gather_bwd_kernel(const bf16* __restrict__ dout, long long ldo,
                                                                             const bf16* __restrict__ y, long long ldy,
                                                                             const int* __restrict__ rows, const float* __restrict__ w,
                                                                             const int* __restrict__ live, bf16* __restrict__ dy,
                                                                             float* __restrict__ dw, int tokens, int k, int n_rows, int D,
                                                                             int split) {
  extern __shared__ __align__(16) uint8_t gb_ring[];
  __shared__ float part[2][kGbWarps][TOP];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, groups = (blockDim.x >> 5) / split, group = warp / split, wk = warp % split;
  const int piece = (min(k, TOP) + 1) * kGbRow, ring_bytes = kGbDepth * piece;
  const uint8_t* ring = gb_ring + warp * ring_bytes + lane * 16;
  const uint32_t dst = smem_u32(ring);
  const int c0 = wk * kGbCols, c_step = split * kGbCols;
  const long long first = blockIdx.x + (long long)group * gridDim.x, stride = (long long)gridDim.x * groups;
  // Row and weight of choice j0 + u in lane u; absent ones are -1.
  auto row_of = [&](long long t, int j0) {
    int r = -1;
    if (t < tokens && lane < TOP && j0 + lane < k) r = rows[t * k + j0 + lane];
    return r < n_rows ? r : -1;
  };
  auto weight_of = [&](long long t, int j0) { return t < tokens && lane < TOP && j0 + lane < k ? w[t * k + j0 + lane] : 0.f; };
  // the piece to fetch next: token, first of its TOP choices, columns
  long long ft = first;
  int fj = 0, fc = c0, fr = row_of(ft, 0), put = 0, get = 0;
  auto fetch = [&] {
    if (ft < tokens) {
      const int c = fc + lane * 8;
      const bool on = c < D;
      if (on) copy16(dst + put, dout + ft * ldo + c);
      if (dw) {
#pragma unroll
        for (int u = 0; u < TOP; ++u) {
          const int r = __shfl_sync(0xffffffffu, fr, u);
          if (on && r >= 0) copy16(dst + put + (u + 1) * kGbRow, y + r * ldy + c);
        }
      }
      fc += c_step;
      if (fc >= D) {
        fc = c0;
        fj += TOP;
        if (fj >= k) { fj = 0; ft += stride; }
        fr = row_of(ft, fj);
      }
    }
    put = put + piece == ring_bytes ? 0 : put + piece;
    asm volatile("cp.async.commit_group;" ::: "memory");      // also an empty group, so that groups count pieces
  };
#pragma unroll
  for (int i = 0; i < kGbDepth - 1; ++i) fetch();
  int buf = 0, next_r = row_of(first, 0);
  float next_f = weight_of(first, 0);
  for (long long t = first; t < tokens; t += stride) {
    for (int j0 = 0; j0 < k; j0 += TOP) {
      const int mr = next_r;
      const float mf = next_f;
      const bool last = j0 + TOP >= k;
      next_r = row_of(last ? t + stride : t, last ? 0 : j0 + TOP);          // a round ahead
      next_f = weight_of(last ? t + stride : t, last ? 0 : j0 + TOP);
      float dot[TOP];
#pragma unroll
      for (int u = 0; u < TOP; ++u) dot[u] = 0.f;
      for (int c = c0 + lane * 8; c - lane * 8 < D; c += c_step) {
        fetch();                          // into the piece read last; a lane reads what it copied itself
        asm volatile("cp.async.wait_group %0;" ::"n"(kGbDepth - 1) : "memory");
        const uint8_t* p = ring + get;
        get = get + piece == ring_bytes ? 0 : get + piece;
        float g[8];
        unpack8(*reinterpret_cast<const bf16x8*>(p), g);                    // whatever there is behind the last column: not used
#pragma unroll
        for (int u = 0; u < TOP; ++u) {
          const int r = __shfl_sync(0xffffffffu, mr, u);
          const float f = __shfl_sync(0xffffffffu, mf, u);
          if (r >= 0 && c < D) {
            if (dw) {
              float a[8];
              unpack8(*reinterpret_cast<const bf16x8*>(p + (u + 1) * kGbRow), a);
#pragma unroll
              for (int q = 0; q < 8; ++q) dot[u] = fmaf(g[q], a[q], dot[u]);
            }
            if (dy) {
              float o[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) o[q] = f * g[q];
              *reinterpret_cast<bf16x8*>(dy + (long long)r * D + c) = pack8(o);
            }
          }
        }
      }
      if (dw) {
        const int u = lane / (32 / TOP);
        float sum = warp_sums<TOP>(dot, lane);
        const bool mine = lane % (32 / TOP) == 0;
        if (split > 1) {
          if (mine) part[buf][warp][u] = sum;
          asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(split * 32) : "memory");
          sum = 0.f;
          if (wk == 0 && mine)
            for (int q = 0; q < split; ++q) sum += part[buf][warp + q][u];
          buf ^= 1;       // the next round writes the other half; the barrier there is behind these reads
        }
        if (wk == 0 && mine && j0 + u < k) dw[t * k + j0 + u] = sum;
      }
    }
  }
  if (dy) {
    const int from = max(0, min(*live, n_rows));
    const long long rest = (long long)(n_rows - from) * (D >> 3);
    bf16x8 z;
    z.u = make_uint4(0, 0, 0, 0);
    for (long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x; it < rest; it += (long long)gridDim.x * blockDim.x)
      *reinterpret_cast<bf16x8*>(dy + (long long)from * D + it * 8) = z;
  }
}
template <int TOP>
int gather_bwd(const bf16* dout, long long ldo, const bf16* y, long long ldy, const int* rows, const float* w, const int* live, bf16* dy,
               float* dw, int tokens, int k, int n_rows, int D, cudaStream_t st) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  static int sms[64] = {};
  if (!sms[dev]) {
    int n = 0;
    if (cudaFuncSetAttribute(expert_gather_bwd_kernel<TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGbWarps * kGbDepth * (TOP + 1) * kGbRow) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return -3;
    sms[dev] = n;
  }
  // as many warps per token as it has pieces of 256 columns, or pieces per warp alike
  const int chunks = (D + kGbCols - 1) / kGbCols, turns = (chunks + kGbWarps - 1) / kGbWarps, split = (chunks + turns - 1) / turns;
  const int groups = kGbWarps / split, warps = groups * split, smem = warps * kGbDepth * ((k < TOP ? k : TOP) + 1) * kGbRow;
  const int by_smem = 225 * 1024 / (smem + 2048), by_regs = 3 * kGbWarps / warps, per_sm = by_smem < by_regs ? by_smem : by_regs;
  const long long most = ((long long)tokens + groups - 1) / groups, ctas = (long long)per_sm * sms[dev];
  expert_gather_bwd_kernel<TOP><<<(unsigned)(most < ctas ? most : ctas), warps * 32, smem, st>>>(dout, ldo, y, ldy, rows, w, live, dy, dw, tokens,
                                                                                                  k, n_rows, D, split);
  return (int)cudaGetLastError();
}

template <typename T>
int route_fwd(const void* s, long long ld, const void* allowed, long long* idx, float* w, int tokens, int E, int k, int normalize,
              cudaStream_t st) {
  const unsigned grid = ((unsigned)tokens + 7) / 8;
#define ERI_ROUTE(V)                                                                                                       \
  route_fwd_kernel<T, V><<<grid, 256, 0, st>>>((const T*)s, ld, (const uint8_t*)allowed, idx, w, tokens, E, k, normalize)
  if (E <= 32) ERI_ROUTE(1);
  else if (E <= 64) ERI_ROUTE(2);
  else if (E <= 128) ERI_ROUTE(4);
  else if (E <= 256) ERI_ROUTE(8);
  else if (E <= 512) ERI_ROUTE(16);
  else ERI_ROUTE(32);
#undef ERI_ROUTE
  return (int)cudaGetLastError();
}

template <typename T>
int route_bwd(const void* s, long long ld, const void* allowed, const long long* idx, const float* w, const float* dw, void* ds,
              int tokens, int E, int k, int normalize, cudaStream_t st) {
  const unsigned grid = ((unsigned)tokens + 7) / 8;
#define ERI_ROUTE(V)                                                                                                            \
  route_bwd_kernel<T, V><<<grid, 256, 0, st>>>((const T*)s, ld, (const uint8_t*)allowed, idx, w, dw, (T*)ds, tokens, E, k, normalize)
  if (E <= 32) ERI_ROUTE(1);
  else if (E <= 64) ERI_ROUTE(2);
  else if (E <= 128) ERI_ROUTE(4);
  else if (E <= 256) ERI_ROUTE(8);
  else if (E <= 512) ERI_ROUTE(16);
  else ERI_ROUTE(32);
#undef ERI_ROUTE
  return (int)cudaGetLastError();
}

unsigned copy_grid(long long items) {       // a thread per item; the kernels loop beyond what a grid holds
  const long long g = (items + 255) / 256;
  return (unsigned)(g > 0x7fffffff ? 0x7fffffff : g);
}

bool dims_ok(int tokens, int k, int n_rows, int D) { return tokens >= 1 && k >= 1 && n_rows >= 0 && D >= 8 && D % 8 == 0; }

}  // namespace

extern "C" {

// scores [tokens, E] (row stride ld elements) fp32 (is_bf16 0) or bf16; allowed [E] bytes or null; idx [tokens, k] int64, w fp32.
int eri_expert_route_fwd(const void* scores, long long ld, const void* allowed, void* idx, float* w, int tokens, int E, int k,
                         int normalize, int is_bf16, void* stream) {
  if (tokens < 1 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxTop || ld < E) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  return is_bf16 ? route_fwd<bf16>(scores, ld, allowed, (long long*)idx, w, tokens, E, k, normalize, st)
                 : route_fwd<float>(scores, ld, allowed, (long long*)idx, w, tokens, E, k, normalize, st);
}

// ds [tokens, E] contiguous, of the scores' type.
int eri_expert_route_bwd(const void* scores, long long ld, const void* allowed, const void* idx, const float* w, const float* dw,
                         void* ds, int tokens, int E, int k, int normalize, int is_bf16, void* stream) {
  if (tokens < 1 || E < 1 || E > kMaxExperts || k < 1 || k > E || k > kMaxTop || ld < E) return -1;
  cudaStream_t st = (cudaStream_t)stream;
  return is_bf16 ? route_bwd<bf16>(scores, ld, allowed, (const long long*)idx, w, dw, ds, tokens, E, k, normalize, st)
                 : route_bwd<float>(scores, ld, allowed, (const long long*)idx, w, dw, ds, tokens, E, k, normalize, st);
}

// idx: n choices (int64 when wide, else int32). offsets [E + 1], rows [n] int32.
int eri_expert_plan(const void* idx, int wide, int n, int E, int* offsets, int* rows, void* stream) {
  if (n < 0 || E < 1 || E > kMaxExperts) return -1;
  const int smem = (kPlanWarps + 3) * E * (int)sizeof(int);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  static bool configured[64] = {};
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(expert_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (kPlanWarps + 3) * kMaxExperts * (int)sizeof(int)) != cudaSuccess)
      return -3;
    configured[dev] = true;
  }
  const int ctas = n <= 4096 ? 1 : n <= 8192 ? 2 : n <= 16384 ? 4 : kMaxCtas;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, expert_plan_kernel, idx, wide, n, E, ctas, offsets, rows);
}

// x [tokens, D] (row stride ldx) -> xs [n_rows, D]; live: offsets + E.
int eri_expert_scatter(const void* x, long long ldx, const int* rows, const int* live, void* xs, int tokens, int k, int n_rows, int D,
                       void* stream) {
  if (!dims_ok(tokens, k, n_rows, D) || ldx % 8 || (((uintptr_t)x | (uintptr_t)xs) & 15)) return -1;
  const long long items = (long long)tokens * (D / 8);
  expert_scatter_kernel<<<copy_grid(items), 256, 0, (cudaStream_t)stream>>>((const bf16*)x, ldx, rows, live, (bf16*)xs, items, D / 8, k,
                                                                            n_rows, D);
  return (int)cudaGetLastError();
}

int eri_expert_gather(const void* y, long long ldy, const int* rows, const float* w, void* out, int tokens, int k, int n_rows, int D,
                      void* stream) {
  if (!dims_ok(tokens, k, n_rows, D) || ldy % 8 || (((uintptr_t)y | (uintptr_t)out) & 15)) return -1;
  const int chunks = (D + kGatherCols - 1) / kGatherCols;
  const long long items = (long long)tokens * chunks;
  expert_gather_kernel<<<copy_grid(items * 32), 256, 0, (cudaStream_t)stream>>>((const bf16*)y, ldy, rows, w, (bf16*)out, items, chunks,
                                                                                k, n_rows, D);
  return (int)cudaGetLastError();
}

// dy [n_rows, D] or null, dw [tokens, k] or null.
int eri_expert_gather_bwd(const void* dout, long long ldo, const void* y, long long ldy, const int* rows, const float* w, const int* live,
                          void* dy, float* dw, int tokens, int k, int n_rows, int D, void* stream) {
  if (!dims_ok(tokens, k, n_rows, D) || ldo % 8 || ldy % 8 || (((uintptr_t)dout | (uintptr_t)y | (uintptr_t)dy) & 15)) return -1;
#define ERI_GATHER_BWD(TOP) \
  gather_bwd<TOP>((const bf16*)dout, ldo, (const bf16*)y, ldy, rows, w, live, (bf16*)dy, dw, tokens, k, n_rows, D, (cudaStream_t)stream)
  return k == 1 ? ERI_GATHER_BWD(1) : k == 2 ? ERI_GATHER_BWD(2) : k <= 4 ? ERI_GATHER_BWD(4) : ERI_GATHER_BWD(8);
#undef ERI_GATHER_BWD
}

}  // extern "C"

ERI_DEBUG_BOUNDS_EXPORT(expert_route)
