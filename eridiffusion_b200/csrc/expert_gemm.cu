// Matrix products grouped by expert: rows [offsets[e], offsets[e + 1]) of a token-major activation meet matrix e of a bank
// W [E, N, K]. The offsets live on the device; nothing of the launch depends on their values.
//
//   kFwd   Y[r, n]     = sum_k X[r, k] W[e(r), n, k]
//   kDx    dX[r, k]    = sum_n dY[r, n] W[e(r), n, k]
//   kDw    dW[e, n, k] = sum_{r in e} dY[r, n] X[r, k]
//
// Rows before offsets[0] and from offsets[E] on belong to no expert: kFwd and kDx write zeros there, kDw leaves them out.
//
// All three run as D[lane, column] with the matrix side on the 256 accumulator lanes of a CTA pair (tcgen05.mma, cta_group::2)
// and the ragged side on BT columns: kFwd and kDx put BT consecutive rows of one expert on the columns, so an expert of a few
// rows costs a tile of 32 columns instead of one of 256 lanes, and every tile reads its share of the weights once. kDw puts
// the K columns of X on the lanes, 256 columns of dY on the columns and reduces over the expert's rows. In all three a
// lane is the fastest index of the output.
//
// Rows of a tile that belong to the next expert are loaded and multiplied but not stored (columns are independent). In kDw
// the rows are what is summed: the last step of an expert's rows goes through a fix-up warp of each CTA that overwrites the
// rows of the next expert with zeros in both operands (zero times infinity would not vanish) before the product may run.
//
// Roles per CTA: warp 0 TMA, warp 1 UMMA issue (leader), warps 2-9 epilogue (a TMEM quadrant is shared by two warps, each with half
// of the columns), warp 10 fix-up (kDw). Persistent: a pair takes every grid-th tile.
//
// Bound: with few rows by reading the weights once (64 rows, 16 experts of 5120 x 2560: 64 us forward at 6.6 TB/s); with thousands of
// rows per expert by the tensor cores (16384 rows, 8 experts of 5120 x 2560: 269 / 286 / 273 us, 0.96 / 0.90 / 0.94 of the measured
// burst rate); in between by the operand intake of short tiles, which share 256 weight rows among few columns (8192 rows, 16
// experts of 4096 x 2048: 107 / 117 / 138 us, 0.77 / 0.71 / 0.60). kDw of few rows is a fill: 130 us for 419 MB, plain fills 110.
#include "ptx.cuh"
#include "tma_host.h"

using namespace eri;
typedef __nv_bfloat16 bf16;

namespace {

ERI_DEBUG_BOUNDS_DEFINE(expert_gemm)

__device__ int g_err;           // first wait that ran out (see eri_expert_gemm_check_error)

enum Mode { kFwd = 0, kDx = 1, kDw = 2 };

constexpr int kMaxExperts = 1024;
constexpr int BM = 128;         // lanes per CTA (256 per pair)
constexpr int BK = 64;          // depth of a step
constexpr int A_BYTES = BM * BK * 2;
// The epilogue stages kEpi columns of 128 lanes at a time, two buffers for each half of the tile. Rows of 272 bytes: the eight 16-byte
// rows that a matrix store touches lie in different banks.
constexpr int kEpi = 16, kEpiPitch = BM * 2 + 16, kEpiBytes = kEpi * kEpiPitch;

struct ExpertParams {
  const int* offsets;
  bf16* out;
  int R, E, N, K;
  int P, C;            // lanes' extent, reduction's extent (kDw: columns' extent)
  int accum;           // kDw: added to what out holds
  long long dbg_out_bytes;   // debug build only
};

template <int BT>
struct Cfg {
  static constexpr int kHalf = BT / 2;                    // columns staged by a CTA
  static constexpr int kB = kHalf * BK * 2;
  static constexpr int kStage = A_BYTES + kB;
  static constexpr int kStages = BT == 256 ? 6 : BT == 128 ? 8 : BT == 64 ? 10 : 11;
  static constexpr int kTmem = 2 * BT;
  static constexpr int kRing = kStages * kStage + 4 * kEpiBytes;
  static constexpr int kSmem = kRing + 1024 + 512;
};

// 16 accumulator lanes x 16 columns: thread i gets lanes i / 4 (r[0], r[1], r[4], r[5]) and i / 4 + 8, columns 2 (i % 4) + {0, 1} and 8 more.
__device__ __forceinline__ void tmem_ld_16x16(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// Four 8 x 8 blocks between registers (two neighbouring columns each) and shared memory, transposed: a row there is a column here.
__device__ __forceinline__ void store_blocks_t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void load_blocks_t(uint32_t addr, uint32_t (&v)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

struct Tile {
  int e, lo, hi;      // expert and the rows of this tile (kDw: all rows of the expert)
  int p0, c0;         // first lane of the pair, first column (kDw)
  int steps;
  int n;              // columns of the product: the tile's rows rounded up to 32 (kDw: BT)
};

template <int BT, int MODE>
struct Sched {
  const int* bound;   // [E + 1] ascending
  const int* before;  // [E + 1] tiles of lower experts (kFwd, kDx)
  int E, num_p, num_c, steps, total;
  __device__ __forceinline__ Tile get(int t) const {
    Tile r;
    if (MODE == kDw) {
      const int per = num_p * num_c;
      r.e = t / per;
      const int i = t - r.e * per;
      r.p0 = (i % num_p) * 2 * BM;
      r.c0 = (i / num_p) * BT;
      r.lo = bound[r.e];
      r.hi = bound[r.e + 1];
      r.steps = (r.hi - r.lo + BK - 1) / BK;
      r.n = BT;
    } else {
      int lo = 0, hi = E;          // before[lo] <= t < before[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= t) lo = mid; else hi = mid;
      }
      r.e = lo;
      const int i = t - before[lo], rows = bound[lo + 1] - bound[lo], tt = (rows + BT - 1) / BT;
      r.p0 = (i / tt) * 2 * BM;
      r.c0 = 0;
      r.lo = bound[lo] + (i % tt) * BT;
      r.hi = min(r.lo + BT, bound[lo + 1]);
      r.steps = steps;
      r.n = (r.hi - r.lo + 31) & ~31;
    }
    return r;
  }
};

template <int BT, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MODE == kDw ? 352 : 320, 1)
expert_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmB16, const __grid_constant__ ExpertParams p) {
  using C = Cfg<BT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kRing);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* tail_full = acc_empty + 2;
  uint64_t* tail_done = tail_full + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail_done + C::kStages);
  int* bound = reinterpret_cast<int*>(smem + C::kRing + 512);   // [E + 1]
  int* before = bound + p.E + 1;                                              // [E + 1]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tail_full[s], 1);
      mbar_init(&tail_done[s], 2);           // fix-up warps of both CTAs (used on the leader only)
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 16);        // epilogue warps of both CTAs (used on the leader only)
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, C::kTmem);
    tmem_relinquish2();
  }
  for (int e = threadIdx.x; e <= p.E; e += blockDim.x) bound[e] = p.offsets[e];
  tc_fence_before();
  __syncthreads();
  const int num_p = (p.P + 2 * BM - 1) / (2 * BM);
  if (warp == 0) {
    // bounds that ascend inside [0, R] whatever the offsets hold, so that no index below can leave its buffer
    int run = 0, tiles = 0;
    for (int e0 = 0; e0 <= p.E; e0 += 32) {
      const int e = e0 + lane;
      int b = e <= p.E ? max(0, min(bound[e], p.R)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) b = max(b, up);
      }
      b = max(b, run);
      if (e <= p.E) bound[e] = b;
      run = __shfl_sync(0xffffffffu, b, 31);
    }
    __syncwarp();
    if (MODE != kDw)
      for (int e0 = 0; e0 <= p.E; e0 += 32) {
        const int e = e0 + lane;
        const int mine = e < p.E ? (bound[e + 1] - bound[e] + BT - 1) / BT * num_p : 0;
        int scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, scan, o);
          if (lane >= o) scan += up;
        }
        if (e <= p.E) before[e] = tiles + scan - mine;
        tiles += __shfl_sync(0xffffffffu, scan, 31);
      }
  }
  __syncthreads();
  cluster_sync_all();              // both CTAs' barriers are initialised before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  Sched<BT, MODE> sched;
  sched.bound = bound;
  sched.before = before;
  sched.E = p.E;
  sched.num_p = num_p;
  sched.num_c = MODE == kDw ? (p.C + BT - 1) / BT : 1;
  sched.steps = (p.C + BK - 1) / BK;
  sched.total = MODE == kDw ? p.E * num_p * sched.num_c : before[p.E];
  const int first = (int)blockIdx.x >> 1, stride = (int)gridDim.x >> 1;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first; ok && t < sched.total; t += stride) {
        const Tile tl = sched.get(t);
        const int p0 = tl.p0 + (int)rank * BM;
        for (int k = 0; k < tl.steps; ++k) {
          if (!mbar_wait(&empty[stage], phase ^ 1)) {
            atomicExch(&g_err, 41);
            ok = false;
            break;
          }
          uint8_t* sA = smem + stage * C::kStage;
          uint8_t* sB = sA + A_BYTES;
          const uint32_t bar = map_to_cta(smem_u32(&full[stage]), 0);
          if (MODE == kDw) {
            const int r = tl.lo + k * BK, c0 = tl.c0 + (int)rank * C::kHalf;
            if (r + BK > tl.hi) {          // rows of the next expert come along: this CTA's fix-up warp passes the step on
              uint64_t* tb = &tail_full[stage];
              if (leader) mbar_arrive(&full[stage]);
              mbar_expect_tx(tb, C::kStage);
              tma_load_2d(sA, &tmA, tb, p0, r);
              tma_load_2d(sA + BK * 128, &tmA, tb, p0 + 64, r);
              tma_load_2d(sB, &tmB, tb, c0, r);
              tma_load_2d(sB + BK * 128, &tmB, tb, c0 + 64, r);
            } else {
              if (leader) mbar_expect_tx(&full[stage], 2 * C::kStage);
              tma_load_2d_pair(sA, &tmA, bar, p0, r);
              tma_load_2d_pair(sA + BK * 128, &tmA, bar, p0 + 64, r);
              tma_load_2d_pair(sB, &tmB, bar, c0, r);
              tma_load_2d_pair(sB + BK * 128, &tmB, bar, c0 + 64, r);
            }
          } else {
            if (leader) mbar_expect_tx(&full[stage], 2 * A_BYTES + tl.n * BK * 2);
            if (MODE == kFwd) {
              tma_load_3d_pair(sA, &tmA, bar, k * BK, p0, tl.e);
            } else {
              tma_load_3d_pair(sA, &tmA, bar, p0, k * BK, tl.e);
              tma_load_3d_pair(sA + BK * 128, &tmA, bar, p0 + 64, k * BK, tl.e);
            }
            // a whole tile's half in one copy, a shorter one in groups of 16 rows: what a step takes in is what bounds it
            const int r = tl.lo + (int)rank * (tl.n >> 1);
            if (tl.n == BT) {
              tma_load_2d_pair(sB, &tmB, bar, k * BK, r);
            } else {
              for (int i = 0; i < tl.n >> 1; i += 16) tma_load_2d_pair(sB + i * 128, &tmB16, bar, k * BK, r + i);
            }
          }
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (leader && elect_one()) {
      constexpr bool a_mn = MODE != kFwd, b_mn = MODE == kDw;
      int stage = 0, it = 0;
      uint32_t phase = 0, tails = 0;         // tails: phase of every stage's tail_done
      bool ok = true;
      for (int t = first; ok && t < sched.total; t += stride, ++it) {
        const Tile tl = sched.get(t);
        const int steps = tl.steps;
        const uint32_t idesc = umma_idesc_bf16(256, tl.n, a_mn, b_mn);
        const int buf = it & 1;
        if (!mbar_wait(&acc_empty[buf], ((uint32_t)(it >> 1) & 1) ^ 1)) {
          atomicExch(&g_err, 42);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BT;
        for (int k = 0; k < steps; ++k) {
          ok = mbar_wait(&full[stage], phase);
          if (MODE == kDw && ok && tl.lo + (k + 1) * BK > tl.hi) {
            ok = mbar_wait(&tail_done[stage], (tails >> stage) & 1);
            tails ^= 1u << stage;
          }
          if (!ok) {
            atomicExch(&g_err, 43);
            break;
          }
          tc_fence_after();
          const uint32_t sA = smem_u32(smem + stage * C::kStage), sB = sA + A_BYTES;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk) {
            const uint64_t da = a_mn ? umma_desc_mn128(sA + kk * 2048, BK * 128) : umma_desc_kmajor(sA, 128) + kk * 2;
            const uint64_t db = b_mn ? umma_desc_mn128(sB + kk * 2048, BK * 128) : umma_desc_kmajor(sB, 128) + kk * 2;
            umma2_bf16(d_tmem, da, db, idesc, (k | kk) != 0);
          }
          const uint32_t em = smem_u32(&empty[stage]);
          umma2_commit_addr(em);
          umma2_commit_addr(map_to_cta(em, 1));
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (ok) {
          const uint32_t a = smem_u32(&acc_full[buf]);
          umma2_commit_addr(a);
          umma2_commit_addr(map_to_cta(a, 1));
        }
      }
    }
  } else if (MODE == kDw && warp == 10) {
    int stage = 0;
    uint32_t phases = 0;         // one bit per stage: a stage is not filled again before its fix-up has arrived
    for (int t = first; t < sched.total; t += stride) {
      const Tile tl = sched.get(t);
      const int rem = (tl.hi - tl.lo) % BK;
      stage = (stage + tl.steps) % C::kStages;
      if (!rem) continue;
      const int st = (stage + C::kStages - 1) % C::kStages;
      if (!mbar_wait(&tail_full[st], (phases >> st) & 1)) {
        if (lane == 0) atomicExch(&g_err, 45);
        break;
      }
      phases ^= 1u << st;
      // a reduction row is 128 bytes in each of the four slabs (the swizzle permutes inside those 128 bytes)
      uint8_t* s = smem + st * C::kStage;
      for (int i = lane; i < (BK - rem) * 8; i += 32)
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(s + q * BK * 128 + rem * 128 + i * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tail_done[st]), 0));
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    bool failed = false;
    if (MODE != kDw) {
      // rows of no expert
      const long long head = (long long)bound[0] * p.P, tail0 = (long long)bound[p.E] * p.P;
      const long long n8 = (head + (long long)p.R * p.P - tail0) >> 3;
      for (long long i = (long long)blockIdx.x * 256 + (threadIdx.x - 64); i < n8; i += (long long)gridDim.x * 256) {
        const long long at = i * 8 < head ? i * 8 : tail0 + (i * 8 - head);
        *reinterpret_cast<uint4*>(p.out + at) = make_uint4(0, 0, 0, 0);
      }
    }
    // A column of D is 128 consecutive elements of the output per CTA, one per accumulator lane: kEpi columns at a time are transposed
    // through shared memory (eight 8 x 8 blocks per warp, two matrix stores) so that 16 lanes write 256 consecutive bytes.
    // Two-byte stores straight from the accumulator, 64 bytes per warp, wrote a gradient of [16, 5120, 2560] at 1.1 TB/s.
    uint8_t* stg = smem + C::kStages * C::kStage + half * 2 * kEpiBytes;
    // matrix i of a store is given by lanes 8 i .. 8 i + 7: columns 8 (i / 2) + .., lanes 8 (i % 2) + .. of a half of the quadrant
    const uint32_t m_off = (uint32_t)(((lane >> 4) * 8 + (lane & 7)) * kEpiPitch + (q * 32 + ((lane >> 3) & 1) * 8) * 2);
    const int v_row = q * (kEpi / 4) + (lane >> 4), v_col = (lane & 15) * 8;      // rows v_row, v_row + 2, .. of the staged columns
    int it = 0, sb = 0;
    for (int t = first; t < sched.total; t += stride, ++it) {
      const Tile tl = sched.get(t);
      const int buf = it & 1;
      if (!failed && !mbar_wait(&acc_full[buf], (uint32_t)(it >> 1) & 1)) {
        if (lane == 0) atomicExch(&g_err, 44);
        failed = true;                               // no further wait; what is left becomes NaN
      }
      tc_fence_after();
      const int p0 = tl.p0 + (int)rank * BM;
      const uint32_t acc = tmem_base + ((uint32_t)(q * 32) << 16) + buf * BT + half * C::kHalf;
      // columns of this half that are stored, and where the first one goes
      const int col0 = half * C::kHalf;
      const int cols = MODE == kDw ? min(C::kHalf, p.C - tl.c0 - col0) : min(C::kHalf, tl.hi - tl.lo - col0);
      bf16* o = p.out + (MODE == kDw ? ((long long)tl.e * p.C + tl.c0 + col0) : (long long)(tl.lo + col0)) * p.P + p0 + v_col;
      const bool v_ok = p0 + v_col < p.P;
      uint32_t r[2][8];                              // the two halves of the quadrant
      if (cols > 0) {
        tmem_ld_16x16(acc, r[0]);
        tmem_ld_16x16(acc + (16u << 16), r[1]);
      }
      for (int c = 0; c < cols; c += kEpi, sb ^= 1) {
        uint8_t* s = stg + sb * kEpiBytes;
        const uint32_t s_m = smem_u32(s) + m_off;
        if (MODE == kDw && p.accum) {                // what the output holds, so that sum and rounding happen once
#pragma unroll
          for (int i = 0; i < kEpi / 8; ++i)
            if (v_ok && c + v_row + 2 * i < cols)
              *reinterpret_cast<uint4*>(s + (v_row + 2 * i) * kEpiPitch + v_col * 2) =
                  *reinterpret_cast<const uint4*>(o + (long long)(c + v_row + 2 * i) * p.P);
          named_barrier(1 + half, 128);
        }
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = failed ? __int_as_float(0x7fffffff) : MODE == kDw && tl.steps == 0 ? 0.f : __uint_as_float(r[h][i]);     // (an expert without rows)
          if (MODE == kDw && p.accum) {
            uint32_t old[4];
            load_blocks_t(s_m + h * 32, old);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 b = bf162_bits_to_float2(old[i]);
              f[2 * i] += b.x;
              f[2 * i + 1] += b.y;
            }
          }
          store_blocks_t(s_m + h * 32, pack_bf162(f[0], f[1]), pack_bf162(f[2], f[3]), pack_bf162(f[4], f[5]), pack_bf162(f[6], f[7]));
        }
        if (c + kEpi < cols) {                       // the next columns, under the barrier and the stores
          tmem_ld_16x16(acc + c + kEpi, r[0]);
          tmem_ld_16x16(acc + c + kEpi + (16u << 16), r[1]);
        }
        named_barrier(1 + half, 128);                // the other buffer's reads are behind every warp that passes
#pragma unroll
        for (int i = 0; i < kEpi / 8; ++i) {
          const int row = c + v_row + 2 * i;
          bf16* d = o + (long long)row * p.P;
          if (v_ok && row < cols && ERI_DBG_RANGE(p.out, p.dbg_out_bytes, d, 16, 81))
            *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(s + (v_row + 2 * i) * kEpiPitch + v_col * 2);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&acc_empty[buf]), 0));
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer may still read this CTA's shared memory / signal its barriers
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc2(tmem_base, C::kTmem);
  }
}

int num_sms(int dev) {
  static int sms[64] = {};
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}

template <int BT, int MODE>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb16, const ExpertParams& p, long long tiles, int dev, cudaStream_t st) {
  constexpr int kMost = Cfg<BT>::kSmem + 2 * (kMaxExperts + 1) * (int)sizeof(int);
  static_assert(kMost <= 232448, "shared memory of a CTA");
  static bool configured[64] = {};
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(expert_gemm_kernel<BT, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) return (int)e;
    configured[dev] = true;
  }
  const int smem = Cfg<BT>::kSmem + 2 * (p.E + 1) * (int)sizeof(int);
  const int pairs = num_sms(dev) / 2;
  const int grid = (int)(tiles < pairs ? (tiles < 1 ? 1 : tiles) : pairs);
  expert_gemm_kernel<BT, MODE><<<grid * 2, MODE == kDw ? 352 : 320, smem, st>>>(ta, tb, tb16, p);
  return (int)cudaGetLastError();
}

int map2(CUtensorMap* m, const void* ptr, int cols, int rows, long long ld, int box_rows) {
  uint64_t d[2] = {(uint64_t)cols, (uint64_t)rows};
  uint64_t s[1] = {(uint64_t)ld * 2};
  uint32_t b[2] = {64, (uint32_t)box_rows};
  return make_tensor_map(m, ptr, 2, d, s, b, 128);
}
int map3(CUtensorMap* m, const void* ptr, int K, int N, int E, int box_rows) {
  uint64_t d[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)E};
  uint64_t s[2] = {(uint64_t)K * 2, (uint64_t)N * K * 2};
  uint32_t b[3] = {64, (uint32_t)box_rows, 1};
  return make_tensor_map(m, ptr, 3, d, s, b, 128);
}

template <int BT>
int run_rows(int mode, const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb16, const ExpertParams& p, long long tiles,
             int dev, cudaStream_t st) {
  return mode == kFwd ? launch<BT, kFwd>(ta, tb, tb16, p, tiles, dev, st) : launch<BT, kDx>(ta, tb, tb16, p, tiles, dev, st);
}

}  // namespace

extern "C" {

int eri_expert_gemm_check_error() {
  int h = 0, z = 0;
  if (cudaMemcpyFromSymbol(&h, g_err, sizeof(int)) != cudaSuccess) return 0;
  if (h) cudaMemcpyToSymbol(g_err, &z, sizeof(int));
  return h;
}

// mode 0: out [R, N] from rows = x [R, K] (stride ld_rows) and w; mode 1: out [R, K] from rows = dy [R, N] and w;
// mode 2: out [E, N, K] (+)= from rows = x [R, K] and rows2 = dy [R, N]. w [E, N, K] and out are contiguous, every base on a
// 16-byte boundary, N, K and row strides multiples of 8. offsets: E + 1 values on the device. columns: 0, or 32 / 64 / 128 / 256
// rows of a tile (modes 0 and 1).
int eri_expert_gemm(int mode, const void* rows, long long ld_rows, const void* rows2, long long ld_rows2, const void* w,
                    const int* offsets, void* out, int R, int E, int N, int K, int columns, int accum, long long dbg_out_bytes,
                    void* stream) {
  if (mode < 0 || mode > 2 || R < 1 || E < 1 || E > kMaxExperts || N < 8 || K < 8 || N % 8 || K % 8 || ld_rows % 8 || ld_rows2 % 8) return -1;
  if (((uintptr_t)rows | (uintptr_t)rows2 | (uintptr_t)w | (uintptr_t)out) & 15) return -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -2;
  cudaStream_t st = (cudaStream_t)stream;
  ExpertParams p = {};
  p.offsets = offsets; p.out = (bf16*)out; p.R = R; p.E = E; p.N = N; p.K = K; p.accum = accum; p.dbg_out_bytes = dbg_out_bytes;
  p.P = mode == kFwd ? N : K;
  p.C = mode == kFwd ? K : N;
  const long long num_p = (p.P + 2 * BM - 1) / (2 * BM);
  CUtensorMap ta, tb, tb16;
  if (mode == kDw) {
    if (map2(&ta, rows, K, R, ld_rows, BK) || map2(&tb, rows2, N, R, ld_rows2, BK)) return -20;
    const long long tiles = (long long)E * num_p * ((N + 255) / 256);
    if (tiles > 0x7fffffff) return -3;
    return launch<256, kDw>(ta, tb, tb, p, tiles, dev, st);
  }
  int bt = columns;
  if (!bt) {
    // Rows of an expert on average against the tile's columns. A short tile multiplies and loads only its rows, so a tall one costs
    // little there; it has fewer stages in flight, a low one reads the weights once more per tile. us, forward / dX, 16
    // experts, 4096 x 2048 (first row 5120 x 2560):  32 | 64 | 128 | 256 columns
    //   4 rows    64.5/68.8 | 66.3/70.9 | 68.0/72.5 | 70.4/73.6       64 rows   61.0/65.0 | 53.0/50.9 | 48.9/46.7 | 51.1/47.0
    //   32 rows   47.2/50.4 | 48.1/46.0 | 47.5/45.4 | 49.7/45.4       128 rows  97.3/95.2 | 67.9/69.9 | 57.6/55.5 | 54.9/52.0
    // Other banks, L2 flushed, 64 | 128 | 256 columns:  64 experts of 1408 x 2048    128 of 768 x 2048          4 of 8192 x 2048
    //   32 rows                                         84/82 | 84/78 | 86/78        90/88 | 90/86 | 92/84      37/39 | 37/43 | 39/47
    //   128 rows                                        100/100 | 88/86 | 94/84      107/121 | 96/100 | 102/94  43/41 | 43/45 | 41/53
    //   512 rows                                        285/281 | 184/180 | 158/152  (256) 166/193 | 129/137 | 115/119  100/105 | 68/72 | 66/94
    // The rule is within a tenth of the best but for dX of few experts, whose tiles do not fill the pairs evenly: four of 8192 x 2048
    // 53 where 41 is possible (128 rows) and 94 for 72 (512), eight of 5120 x 2560 62 for 53 (64 rows) and 72 for 57 (128).
    const int per = R / E;
    bt = per <= 8 ? 32 : per <= 16 ? 64 : per <= 96 ? 128 : 256;
  }
  if (bt != 32 && bt != 64 && bt != 128 && bt != 256) return -4;
  // each expert starts a tile of its own: at most R / bt full ones and one partial tile per expert that has rows
  const long long tiles = ((long long)R / bt + (E < R ? E : R)) * num_p;
  if (tiles > 0x7fffffff) return -3;
  if (map3(&ta, w, K, N, E, mode == kFwd ? BM : BK) || map2(&tb, rows, mode == kFwd ? K : N, R, ld_rows, bt / 2) ||
      map2(&tb16, rows, mode == kFwd ? K : N, R, ld_rows, 16))
    return -20;
  switch (bt) {
    case 32: return run_rows<32>(mode, ta, tb, tb16, p, tiles, dev, st);
    case 64: return run_rows<64>(mode, ta, tb, tb16, p, tiles, dev, st);
    case 128: return run_rows<128>(mode, ta, tb, tb16, p, tiles, dev, st);
    default: return run_rows<256>(mode, ta, tb, tb16, p, tiles, dev, st);
  }
}

}  // extern "C"

ERI_DEBUG_BOUNDS_EXPORT(expert_gemm)
