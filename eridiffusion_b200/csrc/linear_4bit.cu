// Products of a few rows with a weight stored in 4 bits (int4 or NF4 codes, two to a byte with the even element in the low half, one
// fp32 scale per `block` consecutive elements of a weight row): the codes are read once and never expanded in memory.
//
//   eri_linear_4bit        y[r, n]  = sum_k x[r, k] level(q[e, n, k]) scale[e, n, k / block] (+ bias[n])
//   eri_linear_4bit_dgrad  dx[r, k] = sum_n dy[r, n] level(q[e, n, k]) scale[e, n, k / block]
//
// e: the expert of row r, offsets[e] <= r < offsets[e + 1] (offsets null: one weight for all rows). Rows of no expert are zeros. A CTA
// takes up to kRows rows of one expert; the CTA of any other row of theirs leaves at once.
#include "ptx.cuh"

using namespace eri;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kRows = 8;

__constant__ float c_level[2][16] = {
    {-8.f / 7, -7.f / 7, -6.f / 7, -5.f / 7, -4.f / 7, -3.f / 7, -2.f / 7, -1.f / 7, 0.f, 1.f / 7, 2.f / 7, 3.f / 7, 4.f / 7, 5.f / 7,
     6.f / 7, 7.f / 7},
    {-1.0f, -0.6961928009986877f, -0.5250730514526367f, -0.39491748809814453f, -0.28444138169288635f, -0.18477343022823334f,
     -0.09105003625154495f, 0.0f, 0.07958029955625534f, 0.16093020141124725f, 0.24611230194568634f, 0.33791524171829224f,
     0.44070982933044434f, 0.5626170039176941f, 0.7229568362236023f, 1.0f}};

struct Segment {
  int e, rows;        // rows of this CTA from row r on: 0 = another CTA's, -1 = row r belongs to no expert
};
// offsets ascend; whatever they hold, the rows stay in [0, R).
__device__ __forceinline__ Segment segment_of(const int* offsets, int E, int R, int r) {
  if (!offsets) return Segment{0, r % kRows == 0 ? min(kRows, R - r) : 0};
  int lo = 0, hi = E + 1;                // the last e with offsets[e] <= r, plus one
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= r) lo = mid + 1; else hi = mid;
  }
  const int e = lo - 1;
  if (e < 0 || e >= E) return Segment{0, -1};
  const int first = max(0, offsets[e]), end = min(R, offsets[e + 1]);
  if (r < first || r >= end) return Segment{0, -1};
  return Segment{e, (r - first) % kRows == 0 ? min(kRows, end - r) : 0};
}

__global__ void __launch_bounds__(256) linear_4bit_kernel(const bf16* __restrict__ x, long long ldx, const uint8_t* __restrict__ codes,
                                                          const float* __restrict__ scale, const int* __restrict__ offsets,
                                                          const bf16* __restrict__ bias, bf16* __restrict__ y, int R, int E, int N, int K, int block, int nf4) {
  const int r0 = blockIdx.y;
  const Segment sg = segment_of(offsets, E, R, r0);
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  __shared__ float lv[16];
  if (threadIdx.x < 16) lv[threadIdx.x] = c_level[nf4][threadIdx.x];
  __syncthreads();
  if (sg.rows == 0 || n >= N) return;
  if (sg.rows < 0) {
    if (lane == 0) y[(long long)r0 * N + n] = __float2bfloat16(0.f);
    return;
  }
  const uint8_t* q = codes + ((long long)sg.e * N + n) * (K >> 1);
  const float* sc = scale + ((long long)sg.e * N + n) * (K / block);
  float acc[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) acc[m] = 0.f;
  for (int k = lane * 8; k < K; k += 256) {
    const uint32_t c = *reinterpret_cast<const uint32_t*>(q + (k >> 1));
    const float s = sc[k / block];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = lv[(c >> (4 * j)) & 15] * s;
#pragma unroll
    for (int m = 0; m < kRows; ++m)
      if (m < sg.rows) {
        float v[8];
        unpack8(*reinterpret_cast<const bf16x8*>(x + (long long)(r0 + m) * ldx + k), v);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[m] = fmaf(w[j], v[j], acc[m]);
      }
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m) {
    const float s = warp_sum(acc[m]) + (bias ? __bfloat162float(bias[n]) : 0.f);
    if (lane == 0 && m < sg.rows) y[(long long)(r0 + m) * N + n] = __float2bfloat16(s);
  }
}

// A thread owns eight columns and walks the weight rows of its split; the splits' planes are added in order by the second kernel.
__global__ void __launch_bounds__(128) dgrad_4bit_kernel(const bf16* __restrict__ dy, long long ldy, const uint8_t* __restrict__ codes,
                                                         const float* __restrict__ scale, const int* __restrict__ offsets,
                                                         float* __restrict__ part, int R, int E, int N, int K, int block, int nf4) {
  const int r0 = blockIdx.y;
  const Segment sg = segment_of(offsets, E, R, r0);
  if (sg.rows == 0) return;
  __shared__ float lv[16];
  if (threadIdx.x < 16) lv[threadIdx.x] = c_level[nf4][threadIdx.x];
  __syncthreads();
  const int k = (blockIdx.x * 128 + threadIdx.x) * 8;
  if (k >= K) return;
  const int rows = sg.rows < 0 ? 1 : sg.rows;
  float acc[kRows][8];
#pragma unroll
  for (int m = 0; m < kRows; ++m)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[m][j] = 0.f;
  if (sg.rows > 0) {
    const int n0 = (int)((long long)N * blockIdx.z / gridDim.z), n1 = (int)((long long)N * (blockIdx.z + 1) / gridDim.z);
    for (int n = n0; n < n1; ++n) {
      const long long row = (long long)sg.e * N + n;
      const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + row * (K >> 1) + (k >> 1));
      const float s = scale[row * (K / block) + k / block];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = lv[(c >> (4 * j)) & 15] * s;
#pragma unroll
      for (int m = 0; m < kRows; ++m)
        if (m < rows) {
          const float d = __bfloat162float(dy[(long long)(r0 + m) * ldy + n]);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[m][j] = fmaf(d, w[j], acc[m][j]);
        }
    }
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m)
    if (m < rows) {
      float4* o = reinterpret_cast<float4*>(part + ((long long)blockIdx.z * R + r0 + m) * K + k);
      o[0] = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
      o[1] = make_float4(acc[m][4], acc[m][5], acc[m][6], acc[m][7]);
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
  return R >= 1 && R <= 65535 && E >= 1 && N >= 1 && block >= 32 && block % 32 == 0 && K >= block && K % block == 0;
}

}  // namespace

extern "C" {

// x [R, K] (row stride ldx) -> y [R, N]; codes [E, N, K / 2] bytes, scale [E, N, K / block], bias [N] or null (only without offsets).
int eri_linear_4bit(const void* x, long long ldx, const void* codes, const float* scale, const int* offsets, const void* bias, void* y, int R, int E,
                    int N, int K, int block, int nf4, void* stream) {
  if (!dims_ok(R, E, N, K, block) || (bias && offsets) || ldx % 8 || (((uintptr_t)x | (uintptr_t)codes) & 15)) return -1;
  linear_4bit_kernel<<<dim3((N + 7) / 8, R), 256, 0, (cudaStream_t)stream>>>((const bf16*)x, ldx, (const uint8_t*)codes, scale, offsets,
                                                                             (const bf16*)bias, (bf16*)y, R, E, N, K, block, nf4 ? 1 : 0);
  return (int)cudaGetLastError();
}

// Planes of the workspace [planes, R, K] fp32 that eri_linear_4bit_dgrad wants.
int eri_linear_4bit_planes(int R, int N, int K) {
  const int blocks = ((K / 8 + 127) / 128) * ((R + kRows - 1) / kRows);
  int s = (148 * 8 + blocks - 1) / blocks;
  if (s > (N + 31) / 32) s = (N + 31) / 32;
  return s < 1 ? 1 : s > 64 ? 64 : s;
}

// dy [R, N] (row stride ldy) -> dx [R, K] contiguous.
int eri_linear_4bit_dgrad(const void* dy, long long ldy, const void* codes, const float* scale, const int* offsets, float* work, void* dx,
                          int R, int E, int N, int K, int block, int nf4, void* stream) {
  if (!dims_ok(R, E, N, K, block) || (((uintptr_t)dx | (uintptr_t)codes | (uintptr_t)work) & 15)) return -1;
  const int planes = eri_linear_4bit_planes(R, N, K);
  dgrad_4bit_kernel<<<dim3((K / 8 + 127) / 128, R, planes), 128, 0, (cudaStream_t)stream>>>(
      (const bf16*)dy, ldy, (const uint8_t*)codes, scale, offsets, work, R, E, N, K, block, nf4 ? 1 : 0);
  const long long vecs = (long long)R * (K / 8);
  add_planes_kernel<<<(unsigned)((vecs + 255) / 256), 256, 0, (cudaStream_t)stream>>>(work, (bf16*)dx, vecs, planes);
  return (int)cudaGetLastError();
}

}  // extern "C"
