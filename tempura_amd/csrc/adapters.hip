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
// A block takes one row and `cols` columns and works the row's low-rank values out for itself, those of its columns' slices: one launch
// instead of two, which costs each block rank * K elements of A from the L2 (128 KB with rank 16 and K = 4,096, 2 us of a CU's path), asked for by
// sixteen waves at once.
// grid: (ceil(N / cols), rows).  v: LDS.
#define AD_ROW_THREADS 1024
template <typename T, bool VEC>
__global__ __launch_bounds__(AD_ROW_THREADS) void adapter_rows_kernel(AdapterArgs a, int cols) {
  extern __shared__ float v[];          // [slices of these columns, rank]
  const int row = blockIdx.y, n0 = blockIdx.x * cols, n1 = min(n0 + cols, a.N);
  const int slot = a.ids[row];
  if (slot < 0 || slot >= a.slots) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s0 = a.interleaved ? 0 : slice_of(a, n0), s1 = a.interleaved ? 1 : slice_of(a, n1 - 1);
  const int ranks = (s1 - s0 + 1) * a.rank;
  const T* x = (const T*)a.x + (size_t)row * a.K;
  const T* A = (const T*)a.a + ((size_t)slot * a.slices + s0) * a.rank * a.K;
  // (a thread's column: its sum so far and its weights travel beside A)
  const int n = n0 + (int)threadIdx.x;
  const T* B = (const T*)a.b + ((size_t)slot * a.N + min(n, n1 - 1)) * a.rank;
  float first[8];
  load8<T, true>(B, 8, first);
  const float scale = a.scale[slot];
  float* y = a.y + (size_t)row * a.N;
  const float old = n < n1 ? y[n] : 0.f;
  constexpr int R = 2;                  // ranks of a wave at a time
  for (int j = wave * R; j < ranks; j += R * (AD_ROW_THREADS / 64)) {
    float sum[R] = {};
#pragma unroll 4
    for (int k = lane * 8; k < a.K; k += 512) {
      float xv[8];
      load8<T, VEC>(x + k, a.K - k, xv);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float av[8];
        load8<T, VEC>(A + (size_t)(j + i) * a.K + k, a.K - k, av);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[i] = fmaf(av[e], xv[e], sum[i]);
      }
    }
    const float total = wave_sums<R>(sum);      // (lane 32 i: the i-th)
    if ((lane & 31) == 0) v[j + (lane >> 5)] = total;
  }
  __syncthreads();
  for (int c = n; c < n1; c += AD_ROW_THREADS) {
    const float* vs = v + (slice_of(a, c) - s0) * a.rank;
    float sum = 0.f;
    for (int j = 0; j < a.rank; j += 8) {
      float bv[8];
      if (c == n && j == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) bv[e] = first[e];
      } else {
        load8<T, true>((const T*)a.b + ((size_t)slot * a.N + c) * a.rank + j, 8, bv);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(bv[e], vs[j + e], sum);
    }
    y[c] = fmaf(scale, sum, c == n ? old : y[c]);
  }
}

// ---- many rows -------------------------------------------------------------------------------
// Rows with the same adapter are brought together first: a unit is up to UNIT rows of one adapter, wherever they stand in the batch.
//   plan: [0] units; [4 ..] units of four ints (slot, first place, rows, 0); then the rows by place
// (The order of a unit's rows follows the atomics below and may change from run to run: a row's sums do not hang on its place.)
#define AD_UNIT 64
#define AD_PARTS 8     // of K, at most
typedef __bf16 ad_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ad_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int ad_u32x4 __attribute__((ext_vector_type(4)));

// grid: one block.  LDS: two ints a slot.
__global__ __launch_bounds__(1024) void adapter_plan_kernel(const int* __restrict__ ids, int rows, int slots, int4* __restrict__ units, int* __restrict__ order,
                                                           int* __restrict__ n_units) {
  extern __shared__ int count[];      // [slots] rows, then the next place of the slot; [slots] its first unit
  int* first_unit = count + slots;
  __shared__ int wave_rows[16], wave_units[16], base_rows, base_units;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < slots; i += 1024) count[i] = 0;
  if (threadIdx.x == 0) base_rows = base_units = 0;
  __syncthreads();
  // (neighbouring rows mostly have the same adapter: a wave counts its lanes with the same one and adds once)
  for (int i0 = wave * 64; i0 < rows; i0 += 1024) {
    const int i = i0 + lane, s = i < rows ? ids[i] : -1;
    unsigned long long left = __ballot(s >= 0 && s < slots);
    while (left != 0) {
      const int src = (int)__builtin_ctzll(left), one = __builtin_amdgcn_readlane(s, src);
      const unsigned long long same = __ballot(s == one);
      if (lane == src) atomicAdd(&count[one], (int)__popcll(same));
      left &= ~same;
    }
  }
  __syncthreads();
  for (int s0 = 0; s0 < slots; s0 += 1024) {        // running sums over the slots, 1,024 at a time
    const int s = s0 + threadIdx.x;
    const int c = s < slots ? count[s] : 0, u = (c + AD_UNIT - 1) / AD_UNIT;
    int cr = c, cu = u;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int a = __shfl_up(cr, d, 64), b = __shfl_up(cu, d, 64);
      if (lane >= d) {
        cr += a;
        cu += b;
      }
    }
    if (lane == 63) {
      wave_rows[wave] = cr;
      wave_units[wave] = cu;
    }
    __syncthreads();
    int at = base_rows + cr - c, unit = base_units + cu - u, all_r = 0, all_u = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) {
        at += wave_rows[w];
        unit += wave_units[w];
      }
      all_r += wave_rows[w];
      all_u += wave_units[w];
    }
    for (int i = 0; i < u; ++i) units[unit + i] = make_int4(s, at + i * AD_UNIT, min(AD_UNIT, c - i * AD_UNIT), 0);
    __syncthreads();
    if (s < slots) count[s] = at;
    if (threadIdx.x == 0) {
      base_rows += all_r;
      base_units += all_u;
    }
    __syncthreads();
  }
  for (int i0 = wave * 64; i0 < rows; i0 += 1024) {
    const int i = i0 + lane, s = i < rows ? ids[i] : -1;
    unsigned long long left = __ballot(s >= 0 && s < slots);
    while (left != 0) {
      const int src = (int)__builtin_ctzll(left), one = __builtin_amdgcn_readlane(s, src);
      const unsigned long long same = __ballot(s == one);
      int at = 0;
      if (lane == src) at = atomicAdd(&count[one], (int)__popcll(same));
      at = __builtin_amdgcn_readlane(at, src) + __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
      if (s == one) order[at] = i;
      left &= ~same;
    }
  }
  if (threadIdx.x == 0) *n_units = base_units;
}

// 16 bytes of a row from element k on, zeros behind its end (VEC: aligned, and the end is a multiple of the piece)
template <typename T, bool VEC>
__device__ inline ad_u32x4 load_piece(const T* row, int k, int K) {
  constexpr int P = 16 / sizeof(T);
  if constexpr (VEC) {
    return k < K ? *(const ad_u32x4*)(row + k) : (ad_u32x4){0, 0, 0, 0};
  } else {
    union {
      T e[P];
      ad_u32x4 v;
    } u;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      u.e[i] = T{};
      if (k + i < K) u.e[i] = row[k + i];
    }
    return u.v;
  }
}
// c += a . b over the pieces' elements (16 bytes a lane: the lane's row of a, or column of b, of its quarter of the elements)
template <typename T>
__device__ inline void mfma_piece(const ad_u32x4& a, const ad_u32x4& b, ad_f32x4& c) {
  if constexpr (sizeof(T) == 2) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8, a), __builtin_bit_cast(ad_bf16x8, b), c, 0, 0, 0);
  } else {
    const ad_f32x4 x = __builtin_bit_cast(ad_f32x4, a), y = __builtin_bit_cast(ad_f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
  }
}

// v[part, place, ranks] = A x of a unit's rows over one part of K: v^T[rank, row] = A[rank, :] . x[row, :]^T, 16 * RT ranks a block, the four waves
// taking every fourth step of the part, added in LDS in their order.
// grid: (units, parts, blocks of ranks)
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a, const int4* __restrict__ units, const int* __restrict__ order,
                                                           const int* __restrict__ n_units, float* __restrict__ v, int part_k) {
  constexpr int STEP = 64 / sizeof(T);     // elements a step: four pieces of 16 bytes
  if ((int)blockIdx.x >= *n_units) return;
  const int4 u = units[blockIdx.x];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int ranks = a.rank * a.slices, r0 = blockIdx.z * 16 * RT;
  const int k0 = blockIdx.y * part_k, k1 = min(a.K, k0 + part_k);
  const T* xr[4];
  const T* ar[RT];
#pragma unroll
  for (int t = 0; t < 4; ++t) xr[t] = (const T*)a.x + (size_t)order[u.y + min(t * 16 + c, u.z - 1)] * a.K;
#pragma unroll
  for (int t = 0; t < RT; ++t) ar[t] = (const T*)a.a + ((size_t)u.x * ranks + min(r0 + t * 16 + c, ranks - 1)) * a.K;
  const int tiles = (u.z + 15) >> 4;
  ad_f32x4 acc[RT][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[i][t] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
  for (int k = k0 + wave * STEP; k < k1; k += 4 * STEP) {
    const int at = k + g * (STEP / 4);
    ad_u32x4 xf[4], af[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) af[i] = load_piece<T, VEC>(ar[i], at, k1);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t < tiles) xf[t] = load_piece<T, VEC>(xr[t], at, k1);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t < tiles) {
#pragma unroll
        for (int i = 0; i < RT; ++i) mfma_piece<T>(af[i], xf[t], acc[i][t]);
      }
  }
  __shared__ float red[4][16 * RT][17];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t >= tiles) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[wave][i * 16 + 4 * g + r][c] = acc[i][t][r];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * RT; e += 256) {
      const int rank = e % (16 * RT), row = e / (16 * RT);
      if (t * 16 + row < u.z && r0 + rank < ranks)
        v[((size_t)blockIdx.y * a.rows + u.y + t * 16 + row) * ranks + r0 + rank] = (red[0][rank][row] + red[1][rank][row]) + (red[2][rank][row] + red[3][rank][row]);
    }
  }
}

// y[row, n] += scale * B[n, :] . v[row, :] of a unit's rows: y^T[n, row], 16 columns and 16 rows a tile, so that a lane has four neighbouring columns
// of its row.  The low-rank values, the sum of their parts times the scale, go through LDS once a block: float32 as they are; for bfloat16
// weights as three bfloat16 pieces, the leading, middle and last eight bits, whose sum is the value, so nothing is rounded (2 rank columns
// products more on matrix cores that wait for y anyway).  Bound by reading and writing y.
// A lane's weights of another slice than the one at hand are zero.  grid: (units, blocks of cols columns)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a, const int4* __restrict__ units, const int* __restrict__ order,
                                                         const int* __restrict__ n_units, const float* __restrict__ v, int parts, int cols) {
  constexpr int P = 16 / sizeof(T), STEP = 4 * P;        // ranks a piece and a step
  constexpr int PIECES = sizeof(T) == 2 ? 3 : 1, CHUNK = 64, STEPS = CHUNK / STEP;      // ranks at a time
  constexpr int ROW = CHUNK * sizeof(T) + 16;            // bytes of a row in LDS, a bank group more than the values
  if ((int)blockIdx.x >= *n_units) return;
  const int4 u = units[blockIdx.x];
  __shared__ __attribute__((aligned(16))) unsigned char low[PIECES][AD_UNIT * ROW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.y * cols, n1 = min(n0 + cols, a.N), ranks = a.rank * a.slices, tiles = (u.z + 15) >> 4;
  const float scale = a.scale[u.x];
  size_t yrow[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) yrow[t] = (size_t)order[u.y + min(t * 16 + c, u.z - 1)] * a.N;
  const int s0 = a.interleaved ? 0 : slice_of(a, n0), s1 = a.interleaved ? 1 : slice_of(a, n1 - 1);
  for (int s = s0; s <= s1; ++s) {
    const int from = a.interleaved ? n0 : max(n0, s > 0 ? a.ends[s - 1] : 0), to = a.interleaved ? n1 : min(n1, a.ends[s]);
    for (int j0 = 0; j0 < a.rank; j0 += CHUNK) {
      __syncthreads();
      const int quads = min(CHUNK, (a.rank - j0 + STEP - 1) / STEP * STEP) / 4;      // (four values at a time; zeros up to a whole step)
      for (int e = threadIdx.x; e < tiles * 16 * quads; e += 256) {
        const int row = e / quads, j = e % quads * 4;
        ad_f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        if (row < u.z && j0 + j < a.rank) {
          const float* p = v + ((size_t)u.y + row) * ranks + s * a.rank + j0 + j;
          ad_f32x4 part[AD_PARTS];
#pragma unroll
          for (int k = 0; k < AD_PARTS; ++k)
            if (k < parts) part[k] = *(const ad_f32x4*)(p + (size_t)k * a.rows * ranks);
#pragma unroll
          for (int k = 0; k < AD_PARTS; ++k)
            if (k < parts) sum += part[k];
          sum *= scale;
        }
        if constexpr (PIECES == 1) {
          *(ad_f32x4*)(low[0] + row * ROW + j * 4) = sum;
        } else {
          float left[4] = {sum[0], sum[1], sum[2], sum[3]};
#pragma unroll
          for (int p = 0; p < PIECES; ++p) {
            unsigned bits[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              bits[i] = __builtin_bit_cast(unsigned, left[i]) & 0xffff0000u;
              left[i] = fabsf(sum[i]) <= 3.4028234e38f ? left[i] - __builtin_bit_cast(float, bits[i]) : 0.f;   // (infinite or no number: the first piece says it)
            }
            *(uint2*)(low[p] + row * ROW + j * 2) = make_uint2((bits[0] >> 16) | bits[1], (bits[2] >> 16) | bits[3]);
          }
        }
      }
      __syncthreads();
      for (int n = (from & ~15) + wave * 32; n < to; n += 128) {
        // 32 columns: two tiles
        ad_f32x4 acc[2][4], old[2][4];
        ad_u32x4 bf[2][STEPS];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = n + 16 * i + c;
          const bool mine = col >= from && col < to && (!a.interleaved || ((col >> 3) & 1) == s);
          const T* B = (const T*)a.b + ((size_t)u.x * a.N + min(col, a.N - 1)) * a.rank;
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            const int j = j0 + k * STEP + g * P;
            bf[i][k] = mine && j < a.rank ? *(const ad_u32x4*)(B + j) : (ad_u32x4){0, 0, 0, 0};
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            acc[i][t] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
            const int col = n + 16 * i + 4 * g;
            if (VEC) {
              if (t < tiles && col < a.N) old[i][t] = *(const ad_f32x4*)(a.y + yrow[t] + col);
            } else if (t < tiles) {
#pragma unroll
              for (int r = 0; r < 4; ++r) old[i][t][r] = col + r < a.N ? a.y[yrow[t] + col + r] : 0.f;
            }
          }
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
          if (j0 + k * STEP >= a.rank) break;
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (t < tiles) {
#pragma unroll
              for (int p = 0; p < PIECES; ++p) {
                const ad_u32x4 lf = *(const ad_u32x4*)(low[p] + (t * 16 + c) * ROW + (k * 4 + g) * 16);
#pragma unroll
                for (int i = 0; i < 2; ++i) mfma_piece<T>(bf[i][k], lf, acc[i][t]);
              }
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (t * 16 + c < u.z) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int col = n + 16 * i + 4 * g;
              // (a tile that reaches into the columns of another wave, slice or block leaves those alone)
              const bool all = col >= from && col + 4 <= to;
              if (VEC && all) {
                *(ad_f32x4*)(a.y + yrow[t] + col) = old[i][t] + acc[i][t];
              } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (col + r >= from && col + r < to) a.y[yrow[t] + col + r] = old[i][t][r] + acc[i][t][r];
              }
            }
          }
      }
    }
  }
}

template <typename T, bool VEC>
static void adapter_down(const AdapterArgs& g, dim3 grid, int rt, const int4* units, const int* order, const int* n, float* v, int part_k, hipStream_t s) {
  if (rt == 1) adapter_down_kernel<T, 1, VEC><<<grid, 256, 0, s>>>(g, units, order, n, v, part_k);
  else if (rt == 2) adapter_down_kernel<T, 2, VEC><<<grid, 256, 0, s>>>(g, units, order, n, v, part_k);
  else adapter_down_kernel<T, 4, VEC><<<grid, 256, 0, s>>>(g, units, order, n, v, part_k);
}

// y [rows, N] float32 += the adapters' share.  a [slots, slices * rank, K], b [slots, N, rank] of dt, rank a multiple of 8; vec: K is a multiple of
// 8 and x and a are aligned to 16 bytes.  ends: the columns at which the slices end (the last is N).  parts 0: a block a row; else rows brought
// together by adapter, K in `parts` parts, with scratch of 4 + 4 * units + rows ints (units: rows / 64 + the smaller of slots and rows), rounded up to
// a multiple of 4, and parts * rows * slices * rank floats behind them.
extern "C" int tp_adapter_add(const int* ids, const void* x, int dt, const void* a, const void* b, const float* scale, float* y, int rows, int K, int N,
                              int slots, int rank, int slices, int interleaved, const int* ends, int vec, int parts, void* scratch, hipStream_t s) {
  if (rows <= 0 || N <= 0) return 0;
  TP_REQUIRE(dt == TP_BF16 || dt == TP_F32, "adapter_add: unsupported element type");
  TP_REQUIRE(K > 0 && slots > 0 && rank > 0 && rank % 8 == 0 && slices >= 1 && slices <= AD_MAX_SLICES, "adapter_add: bad sizes");
  TP_REQUIRE(!interleaved || (slices == 2 && N % 16 == 0), "adapter_add: two interleaved slices");
  AdapterArgs g = {ids, x, a, b, scale, y, rows, K, N, slots, rank, slices, interleaved, {}};
  for (int i = 0; i < slices; ++i) g.ends[i] = ends[i];
  if (parts > 0) {
    TP_REQUIRE(scratch != nullptr && slots <= 4096 && parts <= AD_PARTS, "adapter_add: no room for a plan");
    const int units = rows / AD_UNIT + (slots < rows ? slots : rows), ranks = rank * slices;
    int* n_units = (int*)scratch;
    int4* list = (int4*)scratch + 1;
    int* order = (int*)(list + units);
    float* v = (float*)((int4*)scratch + 1 + units + (rows + 3) / 4);
    adapter_plan_kernel<<<1, 1024, (size_t)slots * 8, s>>>(ids, rows, slots, list, order, n_units);
    const int rt = ranks <= 16 ? 1 : ranks <= 32 ? 2 : 4;
    const int part_k = ((K + parts - 1) / parts + 255) / 256 * 256;
    const dim3 down(units, (K + part_k - 1) / part_k, (ranks + 16 * rt - 1) / (16 * rt));
    const int cols = 512;
    const dim3 up(units, (N + cols - 1) / cols);
    const bool yvec = N % 4 == 0;
    if (dt == TP_BF16) {
      if (vec) adapter_down<bf16_t, true>(g, down, rt, list, order, n_units, v, part_k, s);
      else adapter_down<bf16_t, false>(g, down, rt, list, order, n_units, v, part_k, s);
      if (yvec) adapter_up_kernel<bf16_t, true><<<up, 256, 0, s>>>(g, list, order, n_units, v, down.y, cols);
      else adapter_up_kernel<bf16_t, false><<<up, 256, 0, s>>>(g, list, order, n_units, v, down.y, cols);
    } else {
      if (vec) adapter_down<float, true>(g, down, rt, list, order, n_units, v, part_k, s);
      else adapter_down<float, false>(g, down, rt, list, order, n_units, v, part_k, s);
      if (yvec) adapter_up_kernel<float, true><<<up, 256, 0, s>>>(g, list, order, n_units, v, down.y, cols);
      else adapter_up_kernel<float, false><<<up, 256, 0, s>>>(g, list, order, n_units, v, down.y, cols);
    }
    TP_CHECK_LAUNCH("adapter_add");
    return 0;
  }
  TP_REQUIRE(rows <= 65535, "adapter_add: too many rows");
  // (as many columns a block as threads, unless that leaves CUs without a block)
  int cols = AD_ROW_THREADS;
  while (cols > 256 && (long)rows * ((N + cols - 1) / cols) < 128) cols /= 2;
  const dim3 grid((N + cols - 1) / cols, rows);
  const size_t lds = (size_t)slices * rank * sizeof(float);
  TP_REQUIRE(lds <= 65536, "adapter_add: ranks of all slices beyond 16,384");
  if (dt == TP_BF16) {
    if (vec) adapter_rows_kernel<bf16_t, true><<<grid, AD_ROW_THREADS, lds, s>>>(g, cols);
    else adapter_rows_kernel<bf16_t, false><<<grid, AD_ROW_THREADS, lds, s>>>(g, cols);
  } else {
    if (vec) adapter_rows_kernel<float, true><<<grid, AD_ROW_THREADS, lds, s>>>(g, cols);
    else adapter_rows_kernel<float, false><<<grid, AD_ROW_THREADS, lds, s>>>(g, cols);
  }
  TP_CHECK_LAUNCH("adapter_add");
  return 0;
}
