// Low-rank adapters of many requests beside a shared projection: y[t] += scale_a B_a (A_a x[t]) for every row t whose request has an
// adapter a, on the float32 rows that the shared product left.  Projections that are stacked into one product (q | k | v, gate | up) have a
// pair (A, B) for each of these slices; A's rows are the slices' ranks one after the other.
//
//   A [slot, slices * rank, K]   B [slot, N, rank]   scale [slot]   ids [rows] (outside 0 .. slots - 1: no adapter)
//
// Ranks are padded to a multiple of 8 with zeros.  The low-rank row v = A x stays float32: the result is a float32 sum of products of the
// operands as they are, like the shared product's.
#include "common.h"

#define AD_MAX_SLICES 8

struct AdapterArgs {
  const int* ids;
  const void* x;        // [rows, K]
  const void* a;
  const void* b;
  const float* scale;
  float* y;             // [rows, N]
  int rows, K, N, slots, rank, slices;
  int interleaved;      // two slices, eight columns of each in turn
  int ends[AD_MAX_SLICES];
};

__device__ inline int slice_of(const AdapterArgs& a, int n) {
  if (a.interleaved) return (n >> 3) & 1;
  int s = 0;
#pragma unroll
  for (int i = 0; i < AD_MAX_SLICES - 1; ++i) s += i + 1 < a.slices && n >= a.ends[i];
  return s;
}

// eight neighbouring elements as floats (VEC: at an address aligned to eight elements)
template <typename T, bool VEC>
__device__ inline void load8(const T* p, int left, float (&v)[8]) {
  if constexpr (VEC) {
    const float4 lo = load_float4(p), hi = load_float4(p + 4);
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
    v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_float(p[i]) : 0.f;
  }
}

// ---- a few rows ------------------------------------------------------------------------------
// A block takes one row and `cols` columns and works the row's low-rank values out for itself, those of its columns' slices.
// grid: (ceil(N / cols), rows); block: 256.  v: LDS.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void adapter_rows_kernel(AdapterArgs a, int cols) {
  extern __shared__ float v[];          // [slices of these columns, rank]
  const int row = blockIdx.y, n0 = blockIdx.x * cols, n1 = min(n0 + cols, a.N);
  const int slot = a.ids[row];
  if (slot < 0 || slot >= a.slots) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s0 = a.interleaved ? 0 : slice_of(a, n0), s1 = a.interleaved ? 1 : slice_of(a, n1 - 1);
  const int ranks = (s1 - s0 + 1) * a.rank;
  const T* x = (const T*)a.x + (size_t)row * a.K;
  const T* A = (const T*)a.a + ((size_t)slot * a.slices + s0) * a.rank * a.K;
  for (int j = wave * 4; j < ranks; j += 16) {
    float sum[4] = {};
    for (int k = lane * 8; k < a.K; k += 512) {
      float xv[8];
      load8<T, VEC>(x + k, a.K - k, xv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float av[8];
        load8<T, VEC>(A + (size_t)(j + i) * a.K + k, a.K - k, av);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[i] = fmaf(av[e], xv[e], sum[i]);
      }
    }
    const float total = wave_sums<4>(sum);      // (lane 16 i: the i-th)
    if ((lane & 15) == 0) v[j + (lane >> 4)] = total;
  }
  __syncthreads();
  const float scale = a.scale[slot];
  for (int n = n0 + threadIdx.x; n < n1; n += 256) {
    const T* B = (const T*)a.b + ((size_t)slot * a.N + n) * a.rank;
    const float* vs = v + (slice_of(a, n) - s0) * a.rank;
    float sum = 0.f;
    for (int j = 0; j < a.rank; j += 8) {
      float bv[8];
      load8<T, true>(B + j, 8, bv);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(bv[e], vs[j + e], sum);
    }
    float* y = a.y + (size_t)row * a.N + n;
    *y = fmaf(scale, sum, *y);
  }
}

// y [rows, N] float32 += the adapters' share.  a [slots, slices * rank, K], b [slots, N, rank] of dt, rank a multiple of 8; vec: K is a multiple of
// 8 and x and a are aligned to 16 bytes.  ends: the columns at which the slices end (the last is N).
extern "C" int tp_adapter_add(const int* ids, const void* x, int dt, const void* a, const void* b, const float* scale, float* y, int rows, int K, int N,
                              int slots, int rank, int slices, int interleaved, const int* ends, int vec, hipStream_t s) {
  if (rows <= 0 || N <= 0) return 0;
  TP_REQUIRE(dt == TP_BF16 || dt == TP_F32, "adapter_add: unsupported element type");
  TP_REQUIRE(K > 0 && slots > 0 && rank > 0 && rank % 8 == 0 && slices >= 1 && slices <= AD_MAX_SLICES, "adapter_add: bad sizes");
  TP_REQUIRE(!interleaved || (slices == 2 && N % 16 == 0), "adapter_add: two interleaved slices");
  TP_REQUIRE(rows <= 65535, "adapter_add: too many rows");
  AdapterArgs g = {ids, x, a, b, scale, y, rows, K, N, slots, rank, slices, interleaved, {}};
  for (int i = 0; i < slices; ++i) g.ends[i] = ends[i];
  const int cols = 256;
  const dim3 grid((N + cols - 1) / cols, rows);
  const size_t lds = (size_t)slices * rank * sizeof(float);
  TP_REQUIRE(lds <= 65536, "adapter_add: ranks of all slices beyond 16,384");
  if (dt == TP_BF16) {
    if (vec) adapter_rows_kernel<bf16_t, true><<<grid, 256, lds, s>>>(g, cols);
    else adapter_rows_kernel<bf16_t, false><<<grid, 256, lds, s>>>(g, cols);
  } else {
    if (vec) adapter_rows_kernel<float, true><<<grid, 256, lds, s>>>(g, cols);
    else adapter_rows_kernel<float, false><<<grid, 256, lds, s>>>(g, cols);
  }
  TP_CHECK_LAUNCH("adapter_add");
  return 0;
}
