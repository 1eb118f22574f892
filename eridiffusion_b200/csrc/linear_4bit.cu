// Products of a few rows with a weight stored in 4 bits (int4 or NF4 codes, two to a byte with the even element in the low half, one
// fp32 scale per `block` consecutive elements of a weight row): the codes are read once and never expanded in memory.
//
//   eri_linear_4bit        y[r, n]  = sum_k x[r, k] level(q[e, n, k]) scale[e, n, k / block] (+ bias[n])
//   eri_linear_4bit_dgrad  dx[r, k] = sum_n dy[r, n] level(q[e, n, k]) scale[e, n, k / block]
//
// e: the expert of row r, offsets[e] <= r < offsets[e + 1] (offsets null: one weight for all rows). Rows of no expert are zeros. Up to
// eight rows of one expert share a pass over its codes.
#include <cuda_fp16.h>
#include <limits.h>

#include "ptx.cuh"

using namespace eri;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kRows = 8, kMaxExperts = 1024;

__constant__ float c_nf4[16] = {-1.0f, -0.6961928009986877f, -0.5250730514526367f, -0.39491748809814453f, -0.28444138169288635f,
                                -0.18477343022823334f, -0.09105003625154495f, 0.0f, 0.07958029955625534f, 0.16093020141124725f,
                                0.24611230194568634f, 0.33791524171829224f, 0.44070982933044434f, 0.5626170039176941f, 0.7229568362236023f,
                                1.0f};

struct Segment {
  int e, rows;        // rows of this CTA from row r on: 0 = another CTA's, -1 = row r belongs to no expert
};
// The bounds are the running maximum of the offsets inside [0, R], whatever they hold (expert_table, too): row r belongs to the
// expert before the first offset above r, from the largest offset before that one on. By a whole warp.
__device__ __forceinline__ Segment segment_of(const int* offsets, int E, int R, int r, int most, int lane) {
  if (!offsets) return Segment{0, r % most == 0 ? min(most, R - r) : 0};
  int first = 0;
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int o = e0 + lane <= E ? offsets[e0 + lane] : INT_MIN;
    const unsigned above = __ballot_sync(0xffffffffu, o > r);
    const int at = above ? __ffs(above) - 1 : 32;
    first = max(first, __reduce_max_sync(0xffffffffu, lane < at ? o : INT_MIN));
    if (above) {
      const int end = min(R, __shfl_sync(0xffffffffu, o, at)), e = e0 + at - 1;
      if (e < 0) break;
      return Segment{e, (r - first) % most == 0 ? min(most, end - r) : 0};
    }
  }
  return Segment{0, -1};
}

// ------------------------------------------------------------------------------------------- y = x W^T
// Sixteen weight rows are the rows of A in mma.m16n8k16, up to eight rows of x its columns. A lane decodes a quarter of a step of one
// weight row and of the row eight below it (8 or 16 codes each; the order of the reduction inside a step is free, so x is laid
// out in the order in which the codes come out of a word). The products of a step have one scale per weight row, which
// multiplies their fp32 sum; nothing is expanded in memory.
//   int4   code - 8 as bf16 (exact), x as it is: the products are exact; the seventh of the level multiplies the finished sum.
//   NF4    levels as fp16 (2^-12), fetched two at a time from a table of all 256 bytes in shared memory that every lane has for itself
//          (a bank of its own, so no conflicts). x as fp16 times a power of two that brings its largest magnitude in the step to
//          [2^14, 2^15): values down to 2^-32 of that are exact, the rest is off by 2^-39 of it.
// The reduction is split over the `kw` warps of a group, `nw` groups take 16 weight rows each. A warp copies the pieces of codes that
// it alone reads (four steps of 16 rows) asynchronously into a ring of its own, across the tiles of a persistent CTA, so that no
// warp waits for another but for the sum of a tile: partial sums meet in shared memory and are added in warp order.
// Bound by instruction issue (about 115 per warp and 1024 codes: decoding 48, ring copies 15, sums, barriers and x the rest), not by the
// 23 bytes per cycle and SM that memory delivers. us in a row of launches: one row 15360 x 2560 NF4 12.2 (22 MB, 5 of them before and
// behind the loop), 75776 x 2560 36.4 (3.0 TB/s; 34.8 with the codes in L2), eight rows 13824 x 5120 int4 20. Twelve rows of 9 experts of 5120 x 2560 24.6.
constexpr int kU = 4;                       // steps of a piece
constexpr int kMaxWarps = 20, kMaxSplit = 10;     // warps of an SM, warps that share a tile
constexpr int kTable = 256 * 32 * 4;        // bytes of the NF4 table
constexpr int kRedRow = 20;                 // partial sums: [warp][8 columns][16 rows + 4], so that a warp's stores hit 32 banks

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// d += A B
template <bool NF4>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (NF4)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Eight codes of a word as four pairs: int4 (0,4) (1,5) (2,6) (3,7), NF4 (0,1) (2,3) (4,5) (6,7).
template <bool NF4>
__device__ __forceinline__ void decode8(uint32_t c, const uint8_t (&table)[NF4 ? kTable : 16], uint32_t lane4, uint32_t (&h)[4]) {
  if constexpr (NF4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = *reinterpret_cast<const uint32_t*>(table + (((i == 0 ? c << 7 : c >> (8 * i - 7)) & 0x7f80u) | lane4));
  } else {
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);       // 128 + code - 136, exact
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t v = ((c >> (4 * i)) & 0x000f000fu) | 0x43004300u;
      const __nv_bfloat162 w = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), off);
      h[i] = *reinterpret_cast<const uint32_t*>(&w);
    }
  }
}

// What a ring knows of the weight; a kernel parameter, so that it costs no registers.
struct Weight {
  const uint8_t* codes;
  const float* scale;
  int N, K, k_bytes, spr, ratio;        // bytes and scales of a row, steps of a scale
};

// A warp's ring of pieces: kU steps (128 or 64 bytes) of 16 weight rows, and the steps' scales, [row][step], copied asynchronously DEPTH - 1
// pieces ahead of the one being read, one commit group per piece. 16-byte chunks are permuted by their row so that the rows that
// one read touches lie in different banks. Codes of rows behind the weight's last one stay what the ring holds (their products
// are not stored, or meet zeros), their scales are the last row's.
// STEP: 64 (the scale's block is a multiple of 64) or 32. WHOLE: K is whole pieces. (TMA copies of the same pieces, one
// instruction each, cost 1.3 us more before the first piece arrives and nothing less afterwards.)
template <int STEP, bool WHOLE, int DEPTH>
struct PieceRing {
  static constexpr int kRow = kU * STEP / 2;                  // bytes of a weight row in a piece
  static constexpr int kChunks = kRow / 16, kCopies = 16 * kChunks / 32;
  static constexpr int kPiece = 16 * kRow + 16 * kU * 4;
  static constexpr int kBytes = DEPTH * kPiece;
  const uint8_t* src;         // this lane's chunk of the next piece
  const float* s_src;
  long long tile_bytes, tile_scales;
  uint32_t dst, s_dst, put = 0, get = 0;
  int tile, piece, tile_end, tile_step, p_lo, p_hi;

  __device__ __forceinline__ PieceRing(uint32_t smem, int lane) {
    const int row = lane / kChunks, c = lane % kChunks;
    dst = smem + row * kRow + (chunk(row, c) << 4);
    s_dst = smem + 16 * kRow + lane * 4;
  }
  // place of a row's 16-byte chunk (rows 32 / kChunks apart are permuted alike)
  static __device__ __forceinline__ int chunk(int row, int c) { return STEP == 64 ? c ^ ((row << 1) & 7) : c ^ ((row >> 1) & 3); }
  // pieces lo .. hi - 1 of the 16-row tiles first, first + step, ... below end; everything fetched before has been read by every lane
  __device__ __forceinline__ void start(const Weight& w, int e, int lane, int first, int end, int step, int lo, int hi) {
    tile = first; tile_end = end; tile_step = step; p_lo = piece = lo; p_hi = hi;
    put = get = 0;
    const long long row = (long long)e * w.N + 16ll * first;
    tile_bytes = 16ll * step * w.k_bytes - (long long)(hi - lo) * kRow;
    tile_scales = 16ll * step * w.spr;
    src = w.codes + (row + lane / kChunks) * w.k_bytes + lo * kRow + lane % kChunks * 16;
    s_src = w.scale + (row + (lane >> 2)) * w.spr;
  }
  // The stage must have been read by every lane (a __syncwarp() before).
  __device__ __forceinline__ void fetch(const Weight& w, int lane) {
    if (tile < tile_end) {
      const int row = lane / kChunks, g = lane >> 2, t = lane & 3;
      const int s0 = piece * kU, si = w.ratio == 1 ? s0 + t : (s0 + t) / w.ratio;
      const int left = w.N - tile * 16;                          // weight rows from here on
      const uint8_t* q = src;
      if (WHOLE && left >= 16) {                                // nothing to leave out
#pragma unroll
        for (int i = 0; i < kCopies; ++i, q += (32 / kChunks) * w.k_bytes) copy16(dst + put + i * 512, q);
        const float* s = s_src + si;
        copy4(s_dst + put, s);
        copy4(s_dst + put + 128, s + 8 * w.spr);
      } else {
#pragma unroll
        for (int i = 0; i < kCopies; ++i, q += (32 / kChunks) * w.k_bytes)
          if ((WHOLE || piece * kRow + lane % kChunks * 16 < w.k_bytes) && (left >= 16 || i * (32 / kChunks) + row < left)) copy16(dst + put + i * 512, q);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (WHOLE || s0 + t < w.K / STEP)
            copy4(s_dst + put + 128 * h, s_src + (left >= 16 || g + 8 * h < left ? 8 * h : left - 1 - g) * w.spr + si);
      }
      src += kRow;
      if (++piece == p_hi) {
        piece = p_lo;
        tile += tile_step;
        src += tile_bytes;
        s_src += tile_scales;
      }
    }
    put = put + kPiece == kBytes ? 0u : put + kPiece;
    copy_commit();                                            // also an empty group, so that groups count pieces
  }
  // The next piece has landed, this lane's copies of it; a __syncwarp() makes it all lanes'.
  __device__ __forceinline__ void wait() { copy_wait<DEPTH - 2>(); }
  __device__ __forceinline__ void next() { get = get + kPiece == kBytes ? 0u : get + kPiece; }
};

struct Args4 {
  const bf16* x;
  long long ldx;
  Weight w;
  const int* offsets;
  const bf16* bias;
  bf16* y;
  int R, E, N, K;
  int kw, nw, rows;       // warps per group, groups, most rows of a pass
};

// Expert bounds that ascend inside [0, R] whatever the offsets hold, and the passes (of up to `rows` rows) of lower experts.
__device__ __forceinline__ void expert_table(const int* offsets, int E, int R, int rows, int* bound, int* passes, int lane) {
  int run = 0, total = 0;
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int e = e0 + lane;
    int b = e <= E ? max(0, min(offsets[e], R)) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, b, o);
      if (lane >= o) b = max(b, up);
    }
    b = max(b, run);
    if (e <= E) bound[e] = b;
    run = __shfl_sync(0xffffffffu, b, 31);
  }
  __syncwarp();
  for (int e0 = 0; e0 <= E; e0 += 32) {
    const int e = e0 + lane, mine = e < E ? (bound[e + 1] - bound[e] + rows - 1) / rows : 0;
    int scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    if (e <= E) passes[e] = total + scan - mine;
    total += __shfl_sync(0xffffffffu, scan, 31);
  }
}
// Rows [first, first + count) of pass i and their expert.
struct Pass {
  int e, first, count;
};
__device__ __forceinline__ Pass pass_of(int i, const int* bound, const int* passes, int E, int R, int rows) {
  if (!bound) return Pass{0, i * rows, min(rows, R - i * rows)};
  int lo = 0, hi = E;            // passes[lo] <= i < passes[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (passes[mid] <= i) lo = mid; else hi = mid;
  }
  const int first = bound[lo] + (i - passes[lo]) * rows;
  return Pass{lo, first, min(rows, bound[lo + 1] - first)};
}
__device__ __forceinline__ void build_table(uint8_t* table) {       // four lanes' copies of a pair at a time
  for (int i = threadIdx.x; i < 256 * 8; i += blockDim.x) {
    const uint32_t v = half2_bits(c_nf4[(i >> 3) & 15], c_nf4[i >> 7]);
    reinterpret_cast<uint4*>(table)[i] = make_uint4(v, v, v, v);
  }
}

__device__ __forceinline__ void group_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The work, passes x groups of nw tiles, is cut into equal consecutive shares, one per CTA: how many passes there are is known on the
// device only. WHOLE: the steps are whole pieces. DEPTH: pieces of a ring.
template <bool NF4, int STEP, bool WHOLE, int DEPTH>
__global__ void __launch_bounds__(kMaxWarps * 32, 1) linear_4bit_kernel(const Args4 p) {
  using Ring = PieceRing<STEP, WHOLE, DEPTH>;
  constexpr int kWords = STEP / 32;           // 32-bit words of codes per lane, weight row and step
  constexpr int kRow = Ring::kRow;
  extern __shared__ __align__(16) uint8_t sm4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int steps = p.K / STEP, warps = p.kw * p.nw;
  // The table and the zeros are static so that their addresses are constants of the loads.
  __shared__ __align__(128) uint8_t table[NF4 ? kTable : 16];
  __shared__ uint4 zero16;
  uint8_t* ring = sm4 + warp * Ring::kBytes;
  float* red = reinterpret_cast<float*>(sm4 + warps * Ring::kBytes);          // [2][warps][8][kRedRow]
  uint8_t* xs = reinterpret_cast<uint8_t*>(red + 2 * warps * 8 * kRedRow);    // [step][kWords][M][4 lanes] 16 bytes
  float* xscale = reinterpret_cast<float*>(xs + (size_t)p.rows * 2 * p.K);    // [step][8] (NF4)
  int* bound = p.offsets ? reinterpret_cast<int*>(xscale + (NF4 ? steps * 8 : 0)) : nullptr;
  int* passes = bound + p.E + 1;

  Ring feed(smem_u32(ring), lane);
  if (threadIdx.x == 0) zero16 = make_uint4(0, 0, 0, 0);
  if (bound) {
    if (warp == 0) expert_table(p.offsets, p.E, p.R, p.rows, bound, passes, lane);
    __syncthreads();
  }
  const int wg = warp / p.kw, wk = warp % p.kw;
  const int pieces = (steps + kU - 1) / kU, p_lo = pieces * wk / p.kw, p_hi = pieces * (wk + 1) / p.kw;
  const int tiles = (p.N + 15) / 16, groups = (tiles + p.nw - 1) / p.nw;
  // shares of one more or less unit, the larger ones first
  const int work = (bound ? passes[p.E] : (p.R + p.rows - 1) / p.rows) * groups;
  const int share = work / (int)gridDim.x, more = work - share * (int)gridDim.x, b = blockIdx.x;
  const int u_end = share * (b + 1) + min(b + 1, more);
  if (bound) {                                           // rows of no expert
    const long long head = (long long)bound[0] * p.N, tail = (long long)bound[p.E] * p.N, n = head + (long long)p.R * p.N - tail;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x)
      p.y[i < head ? i : tail + (i - head)] = __float2bfloat16(0.f);
  }
  // this lane's codes of step u in weight row g of a piece; row g + 8 is permuted alike
  uint32_t q_off[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u)
    q_off[u] = g * kRow + (STEP == 64 ? (Ring::chunk(g, 2 * u + (t >> 1)) << 4) + (t & 1) * 8 : (Ring::chunk(g, u) << 4) + t * 4);
  const uint32_t lane4 = lane * 4;
  int buf = 0, turn = 0;                                 // turn: the group's warp that adds up this round, another one every time
  bool built = false;

  for (int unit = share * b + min(b, more); unit < u_end;) {
    const int i_pass = unit / groups, g0 = unit - i_pass * groups, g1 = min(groups, g0 + (u_end - unit));
    unit += g1 - g0;
    const Pass ps = pass_of(i_pass, bound, passes, p.E, p.R, p.rows);
    const int M = ps.count, r0 = ps.first;
    feed.start(p.w, ps.e, lane, g0 * p.nw + wg, min(tiles, g1 * p.nw), p.nw, p_lo, p_hi);
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) feed.fetch(p.w, lane);
    if (NF4 && !built) build_table(table);               // under the first copies
    if (built) __syncthreads();                          // every group has read the x before
    built = true;
    // x in the order of the codes: a quad of lanes per row and step
    for (int i = threadIdx.x; i < steps * M * 4; i += blockDim.x) {
      const int st = i / (4 * M), m = (i >> 2) % M, q = i & 3;      // a warp's 32 items keep whole quads
      const bf16* src = p.x + (long long)(r0 + m) * p.ldx + st * STEP + q * (STEP / 4);
      float v[kWords][8], f = 1.f;
#pragma unroll
      for (int w = 0; w < kWords; ++w) unpack8(*reinterpret_cast<const bf16x8*>(src + w * 8), v[w]);
      if (NF4) {
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < kWords; ++w)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t b = __float_as_uint(v[w][j]) & 0x7fffffffu;
            if (b < 0x7f800000u) top = max(top, b);
          }
        const unsigned quad = 0xfu << (lane & ~3);
        top = max(top, __shfl_xor_sync(quad, top, 1));
        top = max(top, __shfl_xor_sync(quad, top, 2));
        const int e = max((int)(top >> 23) - 127, -112);
        f = __uint_as_float((uint32_t)(14 - e + 127) << 23);
        if (q == 0) xscale[st * 8 + m] = __uint_as_float((uint32_t)(e - 14 + 127) << 23);
      }
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint4 o;
        if (NF4)
          o = make_uint4(half2_bits(v[w][0] * f, v[w][1] * f), half2_bits(v[w][2] * f, v[w][3] * f), half2_bits(v[w][4] * f, v[w][5] * f),
                         half2_bits(v[w][6] * f, v[w][7] * f));
        else
          o = make_uint4(pack_bf162(v[w][0], v[w][4]), pack_bf162(v[w][1], v[w][5]), pack_bf162(v[w][2], v[w][6]), pack_bf162(v[w][3], v[w][7]));
        *reinterpret_cast<uint4*>(xs + ((size_t)(st * kWords + w) * M * 4 + m * 4 + q) * 16) = o;
      }
    }
    __syncthreads();

    // this lane's x of a step; lanes of absent columns read zeros
    const bool col = g < M;
    const uint32_t x_step = col ? (uint32_t)(kWords * M * 64) : 0u, x_word = col ? (uint32_t)(M * 64) : 0u;
    const uint8_t* x_lane = col ? xs + (size_t)p_lo * kU * kWords * M * 64 + g * 64 + t * 16 : reinterpret_cast<const uint8_t*>(&zero16);
    for (int grp = g0; grp < g1; ++grp) {
      const int tile = grp * p.nw + wg;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      if (tile < tiles) {
        const uint8_t* xp = x_lane;
        const float* xc_lane = xscale + p_lo * kU * 8 + 2 * t;
#pragma unroll 1
        for (int pc = p_lo; pc < p_hi; ++pc) {
          feed.wait();
          __syncwarp();                                  // every lane's copies of this piece have landed, the piece before has been read
          feed.fetch(p.w, lane);
          const uint8_t* codes = ring + feed.get;
          const float4 sa = *reinterpret_cast<const float4*>(codes + 16 * kRow + g * 16);
          const float4 sb = *reinterpret_cast<const float4*>(codes + 16 * kRow + g * 16 + 128);
          const float fa[kU] = {sa.x, sa.y, sa.z, sa.w}, fb[kU] = {sb.x, sb.y, sb.z, sb.w};
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            if (WHOLE || pc * kU + u < steps) {
              float part[4] = {0.f, 0.f, 0.f, 0.f};
              uint32_t c0[kWords], c1[kWords];
              const uint8_t* q = codes + q_off[u];
              if constexpr (kWords == 2) {
                const uint2 a = *reinterpret_cast<const uint2*>(q), b = *reinterpret_cast<const uint2*>(q + 8 * kRow);
                c0[0] = a.x; c0[kWords - 1] = a.y;
                c1[0] = b.x; c1[kWords - 1] = b.y;
              } else {
                c0[0] = *reinterpret_cast<const uint32_t*>(q);
                c1[0] = *reinterpret_cast<const uint32_t*>(q + 8 * kRow);
              }
#pragma unroll
              for (int w = 0; w < kWords; ++w) {
                const uint4 b = *reinterpret_cast<const uint4*>(xp + w * x_word);
                uint32_t h0[4], h1[4];
                decode8<NF4>(c0[w], table, lane4, h0);
                decode8<NF4>(c1[w], table, lane4, h1);
                mma16816<NF4>(part, h0[0], h1[0], h0[1], h1[1], b.x, b.y);
                mma16816<NF4>(part, h0[2], h1[2], h0[3], h1[3], b.z, b.w);
              }
              xp += x_step;
              if (NF4) {
                const float2 xc = *reinterpret_cast<const float2*>(xc_lane + u * 8);
                part[0] *= xc.x; part[1] *= xc.y; part[2] *= xc.x; part[3] *= xc.y;
              }
              acc[0] = fmaf(part[0], fa[u], acc[0]);
              acc[1] = fmaf(part[1], fa[u], acc[1]);
              acc[2] = fmaf(part[2], fb[u], acc[2]);
              acc[3] = fmaf(part[3], fb[u], acc[3]);
            }
          }
          xc_lane += kU * 8;
          feed.next();
        }
      }
      float* mine = red + (buf * warps + warp) * 8 * kRedRow + 2 * t * kRedRow + g;
      mine[0] = acc[0];
      mine[kRedRow] = acc[1];
      mine[8] = acc[2];
      mine[kRedRow + 8] = acc[3];
      // the warps of one group only: the others are at tiles of their own
      if (p.kw == 1) __syncwarp();
      else group_barrier(1 + wg, p.kw * 32);
      if (wk == turn) {
        const int row = lane & 15, n = tile * 16 + row;
        if (n < p.N)
          for (int m = lane >> 4; m < M; m += 2) {
            const float* src = red + ((buf * p.nw + wg) * p.kw * 8 + m) * kRedRow + row;
            float v = 0.f;
#pragma unroll 4
            for (int q = 0; q < p.kw; ++q) v += src[q * 8 * kRedRow];
            if (!NF4) v *= 1.f / 7.f;
            if (p.bias) v += __bfloat162float(p.bias[n]);
            p.y[(long long)(r0 + m) * p.N + n] = __float2bfloat16(v);
          }
      }
      turn = turn + 1 == p.kw ? 0 : turn + 1;
      buf ^= 1;       // the next round writes the other half; the barrier there is behind these reads
    }
  }
}

// ------------------------------------------------------------------------------------------- dx = dy W
// The reduction runs over the weight rows n, and every block of a row has a scale of its own: dy[m, n] scale[n, block] is formed in 32 bits
// for each block and becomes the B operand (16 weight rows x 8 rows of dy) of the block's products; A are the levels of 16 columns of
// W, one register holding two weight rows of one column. Both are fp16: int4 codes - 8 are exact, NF4 levels and dy * scale
// are rounded to 2^-12 of themselves. A power of two per row of dy keeps dy * scale in fp16's range: the first 16 weight rows
// place its largest magnitude at 2^8, and when a later one would pass 2^15 the sums are scaled down with it (rare). Values down to
// 2^-22 of the largest keep all their bits, the rest is off by 2^-33 of it.
// A CTA owns one piece of columns (256, or 128 with blocks of 32) and a range of weight rows; its warps take every kDgWarps-th 16 rows, their
// sums meet in shared memory in warp order, and the ranges' planes are added in order by the kernel below. us: 13824 x 5120 int4, eight
// rows, 22 and 4 for the planes (160 with one thread per eight columns and the products in 32 bits); 16 rows over 16 NF4 experts of 5120 x 2560,
// 90.
constexpr int kDgWarps = 16, kDgDepth = 3, kDgRows = 2048;        // kDgRows: most weight rows of a range (their dy is in shared memory)

template <bool NF4>
__device__ __forceinline__ void decode_rows(uint32_t a, uint32_t b, const uint8_t (&table)[NF4 ? kTable : 16], uint32_t lane4, uint32_t (&h)[8]) {
  // h[i]: code i of word a in the low half, of word b in the high half
  if constexpr (NF4) {
    const uint32_t even = (a & 0x0f0f0f0fu) | ((b << 4) & 0xf0f0f0f0u), odd = ((a >> 4) & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[2 * i] = *reinterpret_cast<const uint32_t*>(table + (((i == 0 ? even << 7 : even >> (8 * i - 7)) & 0x7f80u) | lane4));
      h[2 * i + 1] = *reinterpret_cast<const uint32_t*>(table + (((i == 0 ? odd << 7 : odd >> (8 * i - 7)) & 0x7f80u) | lane4));
    }
  } else {
    const uint32_t lo = __byte_perm(a, b, 0x5410), hi = __byte_perm(a, b, 0x7632);
    const __half2 off = __floats2half2_rn(1032.f, 1032.f);                // 1024 + code - 1032, exact
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t v = (((i < 4 ? lo : hi) >> (4 * (i & 3))) & 0x000f000fu) | 0x64006400u;
      const __half2 w = __hsub2(*reinterpret_cast<__half2*>(&v), off);
      h[i] = *reinterpret_cast<const uint32_t*>(&w);
    }
  }
}

struct DgArgs {
  const bf16* dy;
  long long ldy;
  Weight w;
  const int* offsets;
  float* part;
  int R, E, N, K;
};

template <bool NF4, int STEP, bool WHOLE>
__global__ void __launch_bounds__(kDgWarps * 32, 1) dgrad_4bit_kernel(const DgArgs p) {
  using Ring = PieceRing<STEP, WHOLE, kDgDepth>;
  constexpr int kHalves = STEP / 32;                    // groups of four codes per lane, weight row and step
  constexpr int kCols = kU * STEP;                      // columns of the CTA
  constexpr int kRow = Ring::kRow;
  extern __shared__ __align__(16) uint8_t sm4[];
  __shared__ __align__(128) uint8_t table[NF4 ? kTable : 16];
  const int r0 = p.offsets ? (int)blockIdx.y : (int)blockIdx.y * kRows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Segment sg = segment_of(p.offsets, p.E, p.R, r0, kRows, lane);
  if (sg.rows == 0) return;
  const int g = lane >> 2, t = lane & 3;
  const int k0 = blockIdx.x * kCols;
  const int M = sg.rows < 0 ? 1 : sg.rows, steps = p.K / STEP;
  float* plane = p.part + ((long long)blockIdx.z * p.R + r0) * p.K;
  if (sg.rows < 0) {
    for (int k = k0 + threadIdx.x; k < min(k0 + kCols, p.K); k += blockDim.x) plane[k] = 0.f;
    return;
  }
  const int tiles = (p.N + 15) / 16;
  const int t_lo = (int)((long long)tiles * blockIdx.z / gridDim.z), t_hi = (int)((long long)tiles * (blockIdx.z + 1) / gridDim.z);
  float* dys = reinterpret_cast<float*>(sm4 + kDgWarps * Ring::kBytes);                   // [weight rows of the range][8]
  uint8_t* ring = sm4 + warp * Ring::kBytes;
  Ring feed(smem_u32(ring), lane);
  feed.start(p.w, sg.e, lane, t_lo + warp, t_hi, kDgWarps, blockIdx.x, blockIdx.x + 1);
#pragma unroll
  for (int i = 0; i < kDgDepth - 1; ++i) feed.fetch(p.w, lane);
  if (NF4) build_table(table);
  const int n_lo = t_lo * 16, n_count = (t_hi - t_lo) * 16;
  if (p.N % 8 == 0 && p.ldy % 8 == 0) {                 // (dy starts on a 16-byte boundary)
    for (int i = threadIdx.x; i < n_count; i += blockDim.x) {         // 8 rows of dy x 8 values: as many items as weight rows
      const int m = i / (n_count >> 3), r = (i - m * (n_count >> 3)) * 8;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
      if (m < M && n_lo + r < p.N) unpack8(*reinterpret_cast<const bf16x8*>(p.dy + (long long)(r0 + m) * p.ldy + n_lo + r), f);
#pragma unroll
      for (int j = 0; j < 8; ++j) dys[(r + j) * 8 + m] = f[j];
    }
  } else {
    for (int i = threadIdx.x; i < n_count * 8; i += blockDim.x) {
      const int m = i / n_count, r = i - m * n_count, n = n_lo + r;
      dys[r * 8 + m] = m < M && n < p.N ? __bfloat162float(p.dy[(long long)(r0 + m) * p.ldy + n]) : 0.f;
    }
  }
  __syncthreads();

  const uint32_t lane4 = lane * 4;
  float acc[kU][2 * kHalves][4];
#pragma unroll
  for (int u = 0; u < kU; ++u)
#pragma unroll
    for (int j = 0; j < 2 * kHalves; ++j) acc[u][j][0] = acc[u][j][1] = acc[u][j][2] = acc[u][j][3] = 0.f;
  int top = -1000;                                      // exponent that stands at 2^8 in row g of dy
  const int s_cta = blockIdx.x * kU;                    // first step of the CTA's columns
#pragma unroll 1
  for (int tile = t_lo + warp; tile < t_hi; tile += kDgWarps) {
    feed.wait();
    __syncwarp();                                       // every lane's copies of this piece have landed, the piece before has been read
    feed.fetch(p.w, lane);
    const uint8_t* codes = ring + feed.get;
    // this lane's weight rows of the tile are t, t + 4, t + 8, t + 12
    float v[kU][4];
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float d = dys[((tile - t_lo) * 16 + t + 4 * i) * 8 + g];
      const float4 sc = *reinterpret_cast<const float4*>(codes + 16 * kRow + (t + 4 * i) * 16);
      v[0][i] = d * sc.x; v[1][i] = d * sc.y; v[2][i] = d * sc.z; v[3][i] = d * sc.w;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (!WHOLE && s_cta + u >= steps) v[u][i] = 0.f;
        const uint32_t b = __float_as_uint(v[u][i]) & 0x7fffffffu;
        if (b < 0x7f800000u) big = max(big, b);
      }
    }
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int e = (int)(big >> 23) - 127;
    const bool grow = big != 0 && e > top + 6;
    if (__any_sync(0xffffffffu, grow)) {
      // sums of the rows that grow are scaled down with them; the accumulator's columns are rows 2 t and 2 t + 1 of dy
      const int to = grow ? max(e, -110) : top;
      const int down = top - to;                        // <= 0; from "nothing yet" the sums are zeros (or not finite)
      const float f = top < -110 ? 1.f : __uint_as_float((uint32_t)(127 + max(down, -126)) << 23);
      top = to;
      const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int j = 0; j < 2 * kHalves; ++j) {
          acc[u][j][0] *= f0; acc[u][j][1] *= f1; acc[u][j][2] *= f0; acc[u][j][3] *= f1;
        }
    }
    const float f = top < -110 ? 1.f : __uint_as_float((uint32_t)(127 + 8 - top) << 23);       // (nothing but zeros so far: any)
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (WHOLE || s_cta + u < steps) {
        const uint32_t b0 = half2_bits(v[u][0] * f, v[u][1] * f), b1 = half2_bits(v[u][2] * f, v[u][3] * f);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = t + 4 * i;
          if constexpr (STEP == 64)
            w[i] = *reinterpret_cast<const uint32_t*>(codes + row * kRow + (Ring::chunk(row, 2 * u + (g >> 2)) << 4) + (g & 3) * 4);
          else
            w[i] = *reinterpret_cast<const uint16_t*>(codes + row * kRow + (Ring::chunk(row, u) << 4) + g * 2);
        }
        uint32_t h0[8], h1[8];
        decode_rows<NF4>(w[0], w[1], table, lane4, h0);
        decode_rows<NF4>(w[2], w[3], table, lane4, h1);
#pragma unroll
        for (int j = 0; j < 2 * kHalves; ++j) mma16816<true>(acc[u][j], h0[2 * j], h0[2 * j + 1], h1[2 * j], h1[2 * j + 1], b0, b1);
      }
    }
    feed.next();
  }
  // the rings and dy are read, and nothing is on its way into them: the memory takes the sums
  copy_wait<0>();
  __syncthreads();
  constexpr int kPitch = kCols + 4;
  float* red = reinterpret_cast<float*>(sm4) + warp * 8 * kPitch;         // [warp][8][kPitch]
  const float back = top < -110 ? 0.f : __uint_as_float((uint32_t)(127 - 8 + max(top, -110)) << 23);
  const float k0s = __shfl_sync(0xffffffffu, back, 8 * t) * (NF4 ? 1.f : 1.f / 7.f), k1s = __shfl_sync(0xffffffffu, back, 8 * t + 4) * (NF4 ? 1.f : 1.f / 7.f);
#pragma unroll
  for (int u = 0; u < kU; ++u)
#pragma unroll
    for (int j = 0; j < 2 * kHalves; ++j) {
      const int k = u * STEP + g * (STEP / 8) + 2 * j;
      *reinterpret_cast<float2*>(red + (2 * t) * kPitch + k) = make_float2(acc[u][j][0] * k0s, acc[u][j][2] * k0s);
      *reinterpret_cast<float2*>(red + (2 * t + 1) * kPitch + k) = make_float2(acc[u][j][1] * k1s, acc[u][j][3] * k1s);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < M * kCols; i += blockDim.x) {
    const int m = i / kCols, k = i % kCols;
    if (k0 + k >= p.K) continue;
    const float* q = reinterpret_cast<const float*>(sm4) + m * kPitch + k;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kDgWarps; ++w) s += q[w * 8 * kPitch];
    plane[(long long)m * p.K + k0 + k] = s;
  }
}

__global__ void __launch_bounds__(256) add_planes_kernel(const float* __restrict__ part, bf16* __restrict__ out, long long vecs,
                                                         int planes) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= vecs) return;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  for (int s = 0; s < planes; ++s) {
    const float4* q = reinterpret_cast<const float4*>(part + (s * vecs + i) * 8);
    const float4 a = q[0], b = q[1];
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  *reinterpret_cast<bf16x8*>(out + i * 8) = pack8(v);
}

bool dims_ok(int R, int E, int N, int K, int block) {
  return R >= 1 && R <= 65535 && E >= 1 && E <= kMaxExperts && N >= 1 && block >= 32 && block % 32 == 0 && K >= block && K % block == 0;
}

constexpr int kSmem4 = 227 * 1024 - 1024;       // of an SM, one CTA
int min_of(int a, int b) { return a < b ? a : b; }

int num_sms(int dev) {
  static int sms[64] = {};
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}
template <bool NF4, int STEP, bool WHOLE, int DEPTH>
int launch4d(const Args4& p, int grid, int smem, int dev, cudaStream_t st) {
  static bool configured[64] = {};
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(linear_4bit_kernel<NF4, STEP, WHOLE, DEPTH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kSmem4 - (NF4 ? kTable : 0));
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  linear_4bit_kernel<NF4, STEP, WHOLE, DEPTH><<<grid, p.kw * p.nw * 32, smem, st>>>(p);
  return (int)cudaGetLastError();
}

template <bool NF4, int STEP>
int launch4(Args4& p, int dev, cudaStream_t st) {
  const int steps = p.K / STEP, pieces = (steps + kU - 1) / kU, tiles = (p.N + 15) / 16;
  const int piece = 16 * kU * STEP / 2 + 16 * kU * 4, want = min_of(kRows, p.R), sms = num_sms(dev);
  // Ten warps share a tile where there are few tiles, five where every warp gets some pieces all the same: their barrier and final sum come
  // half as often. us, K = 2560, one NF4 row, ten | five: 16 x K 4.6 | 4.8, 15360 x K 12.2 | 12.7, 18944 x K 13.6 | 13.0,
  // 75776 x K 41.3 | 36.8; K = 5120, eight int4 rows: 16 x K 7.8 | 10.4, 15360 x K 21.5 | 19.9. (About every second row of the
  // grouped form starts a pass.)
  const long long most_pieces = (long long)tiles * pieces * (p.offsets ? (p.R + 1) / 2 : 1);
  const int split = most_pieces >= 4ll * kMaxWarps * sms ? kMaxSplit / 2 : kMaxSplit;
  const int turns = (pieces + split - 1) / split;
  p.kw = (pieces + turns - 1) / turns;
  // Two CTAs of half the warps share an SM where all rows of x fit: one's prologue and last tiles run beside the other. Shared memory: the
  // table, every warp's ring of three pieces (two, where that makes room for x), partial sums, x of a pass. Where x does not
  // fit, fewer groups of warps (down to half), and where it does not fit then either, fewer rows per pass: the codes are read
  // again, from L2.
  int depth = 3, smem = 0;
  auto fits = [&](int per_sm, int nw) {
    p.nw = min_of(nw, tiles);
    const int warps = p.kw * p.nw;
    const int fixed = 2 * warps * 8 * kRedRow * 4 + (NF4 ? steps * 32 : 0) + (p.offsets ? 2 * (p.E + 1) * 4 : 0);
    const int room = kSmem4 / per_sm - (per_sm - 1) * 1024 - (NF4 ? kTable : 0) - fixed;
    depth = room - 3 * warps * piece >= want * 2 * p.K ? 3 : 2;
    p.rows = min_of(want, (room - depth * warps * piece) / (2 * p.K));
    smem = fixed + depth * warps * piece + p.rows * 2 * p.K;
    return p.rows == want;
  };
  const int most_nw = kMaxWarps / p.kw;
  int per_sm = 2;
  if (!fits(2, kMaxWarps / 2 / p.kw)) {
    per_sm = 1;
    int nw = most_nw;
    while (!fits(1, nw) && nw > (most_nw + 1) / 2) --nw;
  }
  if (p.rows < 1) return -100;
  // in the grouped form each row may be a pass of its own
  const long long most = (long long)(p.offsets ? p.R : (p.R + p.rows - 1) / p.rows) * ((tiles + p.nw - 1) / p.nw);
  if (most > 0x7fffffff) return -100;
  const int ctas = per_sm * sms, grid = most < ctas ? (int)most : ctas;
  if (depth == 3) return steps % kU ? launch4d<NF4, STEP, false, 3>(p, grid, smem, dev, st) : launch4d<NF4, STEP, true, 3>(p, grid, smem, dev, st);
  return steps % kU ? launch4d<NF4, STEP, false, 2>(p, grid, smem, dev, st) : launch4d<NF4, STEP, true, 2>(p, grid, smem, dev, st);
}

template <bool NF4, int STEP, bool WHOLE>
int launch_dgw(const DgArgs& p, int planes, int dev, cudaStream_t st) {
  constexpr int kCols = kU * STEP, kRings = kDgWarps * PieceRing<STEP, WHOLE, kDgDepth>::kBytes, kRed = kDgWarps * 8 * (kCols + 4) * 4;
  constexpr int kSmem = kDgRows * 32 + kRings > kRed ? kDgRows * 32 + kRings : kRed;
  static_assert(kSmem + (NF4 ? kTable : 0) <= kSmem4, "shared memory of a CTA");
  static bool configured[64] = {};
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(dgrad_4bit_kernel<NF4, STEP, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  const dim3 grid((p.K + kCols - 1) / kCols, p.offsets ? p.R : (p.R + kRows - 1) / kRows, planes);
  dgrad_4bit_kernel<NF4, STEP, WHOLE><<<grid, kDgWarps * 32, kSmem, st>>>(p);
  return (int)cudaGetLastError();
}
template <bool NF4, int STEP>
int launch_dg(const DgArgs& p, int planes, int dev, cudaStream_t st) {
  return p.K % (kU * STEP) == 0 ? launch_dgw<NF4, STEP, true>(p, planes, dev, st) : launch_dgw<NF4, STEP, false>(p, planes, dev, st);
}

}  // namespace

extern "C" {

// x [R, K] (row stride ldx) -> y [R, N]; codes [E, N, K / 2] bytes, scale [E, N, K / block], bias [N] or null (only without offsets).
int eri_linear_4bit(const void* x, long long ldx, const void* codes, const float* scale, const int* offsets, const void* bias, void* y, int R, int E,
                    int N, int K, int block, int nf4, void* stream) {
  if (!dims_ok(R, E, N, K, block) || (bias && offsets) || ldx % 8 || (((uintptr_t)x | (uintptr_t)codes) & 15)) return -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  const Weight w = {(const uint8_t*)codes, scale, N, K, K / 2, K / block, block / (block % 64 == 0 ? 64 : 32)};
  Args4 p = {(const bf16*)x, ldx, w, offsets, (const bf16*)bias, (bf16*)y, R, E, N, K, 0, 0, 0};
  cudaStream_t st = (cudaStream_t)stream;
  if (block % 64 == 0) return nf4 ? launch4<true, 64>(p, dev, st) : launch4<false, 64>(p, dev, st);
  return nf4 ? launch4<true, 32>(p, dev, st) : launch4<false, 32>(p, dev, st);
}

// Planes of the workspace [planes, R, K] fp32 that eri_linear_4bit_dgrad wants: ranges of weight rows, so that the CTAs fill the SMs and a
// range's dy fits shared memory.
int eri_linear_4bit_planes(int R, int N, int K, int block, int grouped) {
  const int cols = kU * (block % 64 == 0 ? 64 : 32), blocks = ((K + cols - 1) / cols) * (grouped ? (R + 1) / 2 : (R + kRows - 1) / kRows);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  int s = num_sms(dev) / blocks;
  const int most = (N + 16 * kDgWarps - 1) / (16 * kDgWarps), least = ((N + 15) / 16 + kDgRows / 16 - 1) / (kDgRows / 16);
  if (s > most) s = most;
  if (s < least) s = least;
  return s < 1 ? 1 : s;
}

// dy [R, N] (row stride ldy) -> dx [R, K] contiguous.
int eri_linear_4bit_dgrad(const void* dy, long long ldy, const void* codes, const float* scale, const int* offsets, float* work, void* dx,
                          int R, int E, int N, int K, int block, int nf4, void* stream) {
  if (!dims_ok(R, E, N, K, block) || (((uintptr_t)dy | (uintptr_t)dx | (uintptr_t)codes | (uintptr_t)work) & 15)) return -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  const int planes = eri_linear_4bit_planes(R, N, K, block, offsets != nullptr);
  if (planes > 65535) return -100;
  const Weight w = {(const uint8_t*)codes, scale, N, K, K / 2, K / block, block / (block % 64 == 0 ? 64 : 32)};
  const DgArgs p = {(const bf16*)dy, ldy, w, offsets, work, R, E, N, K};
  cudaStream_t st = (cudaStream_t)stream;
  const int code = block % 64 == 0 ? (nf4 ? launch_dg<true, 64>(p, planes, dev, st) : launch_dg<false, 64>(p, planes, dev, st))
                                   : (nf4 ? launch_dg<true, 32>(p, planes, dev, st) : launch_dg<false, 32>(p, planes, dev, st));
  if (code) return code;
  const long long vecs = (long long)R * (K / 8);
  add_planes_kernel<<<(unsigned)((vecs + 255) / 256), 256, 0, st>>>(work, (bf16*)dx, vecs, planes);
  return (int)cudaGetLastError();
}

}  // extern "C"
