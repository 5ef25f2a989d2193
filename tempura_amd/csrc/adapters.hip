// Low-rank adapters of many requests beside a shared projection: y[t] += scale_a B_a (A_a x[t]) for every row t whose request has an
// adapter a, on the float32 rows that the shared product left.  Projections that are stacked into one product (q | k | v, gate | up) have a
// pair (A, B) for each of these slices; A's rows are the slices' ranks one after the other.
//
//   A [slot, slices * rank, K]   B [slot, N, rank]   scale [slot]   ids [rows] (outside 0 .. slots - 1: no adapter)
//
// Ranks are padded to a multiple of 8 with zeros.  The low-rank row v = A x stays float32: the result is a float32 sum of products of the
// operands as they are, like the shared product's.
#include <type_traits>

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

// eight neighbouring elements as floats (VEC: at an address aligned to 16 bytes; else at any that an element may have, which global loads here allow)
template <typename T, bool VEC>
__device__ inline void load8(const T* p, float (&v)[8]) {
  if constexpr (VEC) {
    const float4 lo = load_float4(p), hi = load_float4(p + 4);
    v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
    v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
  } else {
    T e[8];
    __builtin_memcpy(e, p, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
  }
}

// ---- a few rows ------------------------------------------------------------------------------
// sum[i] = A[i, :] . x over a wave's lanes, eight elements a lane at a time (lane 64 / R * i of the result holds the i-th)
template <typename T, bool VEC, int R>
__device__ inline float wave_dots(const T* A, const T* x, int K) {
  const int lane = threadIdx.x & 63;
  float sum[R] = {};
  int k = lane * 8;
#pragma unroll 8 / R
  for (; k + 8 <= K; k += 512) {
    float xv[8];
    load8<T, VEC>(x + k, xv);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float av[8];
      load8<T, VEC>(A + (size_t)i * K + k, av);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[i] = fmaf(av[e], xv[e], sum[i]);
    }
  }
  if constexpr (!VEC) {      // (the elements behind the last eight, in the lane whose turn they are)
    for (int n = k; n < K && n < k + 8; ++n) {
#pragma unroll
      for (int i = 0; i < R; ++i) sum[i] = fmaf(to_float(A[(size_t)i * K + n]), to_float(x[n]), sum[i]);
    }
  }
  return wave_sums<R>(sum);
}

// A block takes one row and `cols` columns and works the row's low-rank values out for itself, those of its columns' slices: one launch
// instead of two, which costs each block rank * K elements of A from the L2 (128 KB with rank 16 and K = 4,096, 2 us of a CU's path), asked for by
// sixteen waves at once.  DONE: `low` [rows, slices * rank] holds them already (adapter_rows_down_kernel).
// grid: (ceil(N / cols), rows).  v: LDS.
#define AD_ROW_THREADS 1024
// R: ranks of a wave at a time.
template <typename T, bool VEC, int R, bool DONE>
__global__ __launch_bounds__(AD_ROW_THREADS) void adapter_rows_kernel(AdapterArgs a, const float* __restrict__ low, int cols) {
  extern __shared__ float v[];          // [slices of these columns, rank]
  const int row = blockIdx.y, n0 = blockIdx.x * cols, n1 = min(n0 + cols, a.N);
  const int slot = a.ids[row];
  if (slot < 0 || slot >= a.slots) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int s0 = a.interleaved ? 0 : slice_of(a, n0), s1 = a.interleaved ? 1 : slice_of(a, n1 - 1);
  const int ranks = (s1 - s0 + 1) * a.rank;
  // (a thread's column: its sum so far and its weights travel beside A)
  const int n = n0 + (int)threadIdx.x;
  const T* B = (const T*)a.b + ((size_t)slot * a.N + min(n, n1 - 1)) * a.rank;
  float first[8];
  load8<T, true>(B, first);
  const float scale = a.scale[slot];
  float* y = a.y + (size_t)row * a.N;
  const float old = n < n1 ? y[n] : 0.f;
  if constexpr (DONE) {
    for (int j = threadIdx.x; j < ranks; j += blockDim.x) v[j] = low[((size_t)row * a.slices + s0) * a.rank + j];
  } else {
    const T* x = (const T*)a.x + (size_t)row * a.K;
    const T* A = (const T*)a.a + ((size_t)slot * a.slices + s0) * a.rank * a.K;
    for (int j = wave * R; j < ranks; j += R * (AD_ROW_THREADS / 64)) {
      const float total = wave_dots<T, VEC, R>(A + (size_t)j * a.K, x, a.K);
      if (lane % (64 / R) == 0) v[j + lane / (64 / R)] = total;
    }
  }
  __syncthreads();
  if (n >= n1) return;
  const float* vs = v + (slice_of(a, n) - s0) * a.rank;
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(first[e], vs[e], sum);
  for (int j = 8; j < a.rank; j += 8) {
    float bv[8];
    load8<T, true>(B + j, bv);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(bv[e], vs[j + e], sum);
  }
  y[n] = fmaf(scale, sum, old);
}

// low[row, ranks] = A x of rows taken one by one, a rank a wave: where A's rows are so long, or so many, that a block of the kernel above would be busy
// with them for long.  grid: (ceil(ranks / 4), rows)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void adapter_rows_down_kernel(AdapterArgs a, float* __restrict__ low) {
  const int row = blockIdx.y, slot = a.ids[row], ranks = a.slices * a.rank, j = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (slot < 0 || slot >= a.slots || j >= ranks) return;
  const float total = wave_dots<T, VEC, 1>((const T*)a.a + ((size_t)slot * ranks + j) * a.K, (const T*)a.x + (size_t)row * a.K, a.K);
  if ((threadIdx.x & 63) == 0) low[(size_t)row * ranks + j] = total;
}

// ---- many rows -------------------------------------------------------------------------------
// The rows are taken in windows of 64 neighbours, and of a window the rows with the same adapter together: rows of one request are neighbours, so a
// window has one or two adapters, or, where single tokens stand side by side, some more.  Every block finds its rows from the window's 64 ids
// with a handful of wave-wide votes: a list made by a launch of its own would cost 4 to 9 us and two more trips to memory at each block's start.
#define AD_WINDOW 64
#define AD_PARTS 8     // of K, at most
typedef __bf16 ad_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ad_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int ad_u32x4 __attribute__((ext_vector_type(4)));
#define AD_GPTR(p) ((const __attribute__((address_space(1))) void*)(p))
#define AD_LPTR(p) ((__attribute__((address_space(3))) void*)(p))

// The rows of window `window` with its which-th adapter (in the order of their first rows; rows without one count as adapter -1): how many, and
// which adapter.  order: LDS, the rows.  For whole blocks.
__device__ inline int window_rows(const AdapterArgs& a, int window, int which, int* order, int& slot) {
  const int lane = threadIdx.x & 63, row = window * AD_WINDOW + lane;
  int id = row < a.rows ? a.ids[row] : -2;
  if (id < -2 || id >= a.slots || (id == -2 && row < a.rows)) id = -1;
  unsigned long long left = __ballot(id != -2), same = 0;
  slot = -2;
  for (int i = 0; i <= which && left != 0; ++i) {
    slot = __builtin_amdgcn_readlane(id, (int)__builtin_ctzll(left));
    same = __ballot(id == slot);
    left &= ~same;
    if (i < which) same = 0;
  }
  if (same != 0 && threadIdx.x < 64 && id == slot)
    order[__builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0))] = row;
  __syncthreads();
  return (int)__popcll(same);
}

// 16 bytes of a row from element k on, zeros behind its end (VEC: aligned, and the end is a multiple of the piece; FULL: the end is not in reach)
template <typename T, bool VEC, bool FULL>
__device__ inline ad_u32x4 load_piece(const T* row, int k, int K) {
  constexpr int P = 16 / sizeof(T);
  if constexpr (VEC) {
    return FULL || k < K ? *(const ad_u32x4*)(row + k) : (ad_u32x4){0, 0, 0, 0};
  } else {
    union {
      T e[P];
      ad_u32x4 v;
    } u;
    if constexpr (FULL) {
      __builtin_memcpy(u.e, row + k, 16);
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        u.e[i] = T{};
        if (k + i < K) u.e[i] = row[k + i];
      }
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

// v[part, row, ranks] = A x over one part of K, 16 * RT ranks a block: v^T[rank, row] = A[rank, :] . x[row, :]^T.
// grid: (windows, parts, blocks of ranks * each), a block taking every each-th adapter of its window (the first adapters' blocks in front: those that find
// none would else take places between the others in the turn in which blocks are handed to the CUs).
// This form loads fragments straight into registers, the four waves taking every fourth step, added in LDS in their order: for rows whose length is no
// multiple of 128 bytes (VEC: but of eight elements) or that are not aligned.
template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a, float* __restrict__ v, int each, int part_k) {
  constexpr int STEP = 64 / sizeof(T);     // elements a step: four pieces of 16 bytes
  __shared__ int order[AD_WINDOW];
  __shared__ float red[4][16 * RT][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const int ranks = a.rank * a.slices, zb = gridDim.z / each, r0 = blockIdx.z % zb * 16 * RT;
  const int k0 = blockIdx.y * part_k, k1 = min(a.K, k0 + part_k);
  for (int which = blockIdx.z / zb;; which += each) {
    int slot;
    __syncthreads();
    const int count = window_rows(a, blockIdx.x, which, order, slot);
    if (count == 0) return;
    if (slot < 0) continue;
    const T* xr[4];
    const T* ar[RT];
#pragma unroll
    for (int t = 0; t < 4; ++t) xr[t] = (const T*)a.x + (size_t)order[min(t * 16 + c, count - 1)] * a.K;
#pragma unroll
    for (int t = 0; t < RT; ++t) ar[t] = (const T*)a.a + ((size_t)slot * ranks + min(r0 + t * 16 + c, ranks - 1)) * a.K;
    const int tiles = (count + 15) >> 4;
    ad_f32x4 acc[RT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[i][t] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
    auto step = [&](int k, auto full) __attribute__((always_inline)) {
      const int at = k + g * (STEP / 4);
      ad_u32x4 xf[4], af[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) af[i] = load_piece<T, VEC, full.value>(ar[i], at, k1);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (t < tiles) xf[t] = load_piece<T, VEC, full.value>(xr[t], at, k1);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (t < tiles) {
#pragma unroll
          for (int i = 0; i < RT; ++i) mfma_piece<T>(af[i], xf[t], acc[i][t]);
        }
    };
    int k = k0 + wave * STEP;
    for (; k + STEP <= k1; k += 4 * STEP) step(k, std::true_type{});
    if (k < k1) step(k, std::false_type{});
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
        if (t * 16 + row < count && r0 + rank < ranks)
          v[((size_t)blockIdx.y * a.rows + order[t * 16 + row]) * ranks + r0 + rank] =
              (red[0][rank][row] + red[1][rank][row]) + (red[2][rank][row] + red[3][rank][row]);
      }
    }
  }
}

// The same with x and A on their way to LDS, 128 bytes of each of 64 rows and 16 * RT ranks a step (whole cache lines; fragments loaded into their registers
// are 64-byte pieces of sixteen rows, which a CU's path to memory takes at half the rate: 4,096 rows of 4,096 with rank 64 16 to 22 us).  A ring of NS steps
// that the four waves fill, one barrier a step; a wave has 16 rows and all the block's ranks.  In LDS chunk x of 16 bytes of a row lies at
// x ^ (row mod 8), so that the rows that are read together fall into different banks.  K and part_k: multiples of 128 bytes.
template <typename T, int RT, int NS>
__global__ __launch_bounds__(256) void adapter_down_lds_kernel(AdapterArgs a, float* __restrict__ v, int each, int part_k) {
  constexpr int SK = 128 / sizeof(T);                       // elements of a row a step
  constexpr int AL = RT == 4 ? 2 : 1, LOADS = 2 + AL;       // a wave's loads of 1 KB (eight rows): of x, of A (RT 1: two waves load the others' rows again)
  constexpr int STAGE = 8192 + RT * 2048;
  __shared__ __attribute__((aligned(1024))) unsigned char ring[NS * STAGE];
  __shared__ int order[AD_WINDOW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int ranks = a.rank * a.slices, zb = gridDim.z / each, r0 = blockIdx.z % zb * 16 * RT;
  const int k0 = blockIdx.y * part_k, steps = (min(a.K, k0 + part_k) - k0) / SK;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)ring;
  for (int which = blockIdx.z / zb;; which += each) {
    int slot;
    __syncthreads();
    const int count = window_rows(a, blockIdx.x, which, order, slot);
    if (count == 0) return;
    if (slot < 0) continue;
    const unsigned char* src[LOADS];
    int place[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int t = j < 2 ? wave * 2 + j : (wave * AL + j - 2) % (2 * RT);          // which eight rows
      const int row = t * 8 + (lane >> 3), chunk = (lane & 7) ^ (row & 7);
      const T* base = j < 2 ? (const T*)a.x + (size_t)order[min(row, count - 1)] * a.K : (const T*)a.a + ((size_t)slot * ranks + min(r0 + row, ranks - 1)) * a.K;
      src[j] = (const unsigned char*)(base + k0) + chunk * 16;
      place[j] = (j < 2 ? 0 : 8192) + t * 1024;
    }
    auto issue = [&](int i, int st) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        __builtin_amdgcn_global_load_lds(AD_GPTR(src[j] + (size_t)i * 128), AD_LPTR(ring + st * STAGE + place[j]), 16, 0, 0);
    };
    // (steps that are not there: the last one again, so that the waits always count as many loads)
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) issue(min(i, steps - 1), i);
    ad_f32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
    const bool busy = wave * 16 < count;
    int st = 0;
    for (int i = 0; i < steps; ++i) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * LOADS) : "memory");
      __builtin_amdgcn_s_barrier();               // every wave's share of this step has come, and the step before is read by all
      asm volatile("" ::: "memory");
      issue(min(i + NS - 1, steps - 1), st == 0 ? NS - 1 : st - 1);
      const unsigned base = lds0 + st * STAGE;
      st = st + 1 == NS ? 0 : st + 1;
      if (!busy) continue;
      ad_u32x4 xf[2], af[2][RT];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned at = ((h * 4 + g) ^ (c & 7)) * 16;
        asm volatile("ds_read_b128 %0, %1" : "=v"(xf[h]) : "v"(base + (wave * 16 + c) * 128 + at));
#pragma unroll
        for (int t = 0; t < RT; ++t) asm volatile("ds_read_b128 %0, %1" : "=v"(af[h][t]) : "v"(base + 8192 + (t * 16 + c) * 128 + at));
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        asm volatile("" : "+v"(xf[h]));
#pragma unroll
        for (int t = 0; t < RT; ++t) asm volatile("" : "+v"(af[h][t]));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) mfma_piece<T>(af[h][t], xf[h], acc[t]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (nothing is on its way into LDS when the next adapter's steps are)
    if (wave * 16 + c < count) {
      float* to = v + ((size_t)blockIdx.y * a.rows + order[wave * 16 + c]) * ranks + r0;
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (r0 + t * 16 + 4 * g < ranks) *(ad_f32x4*)(to + t * 16 + 4 * g) = acc[t];
    }
  }
}

// y[row, n] = scale * B[n, :] . v[row, :] (zero without an adapter), or added to it: y^T[n, row], 16 columns and 16 rows a tile.  A wave has 16 * CT
// columns, whose weights it keeps in registers for all of the window's rows; its tiles of 16 rows leave through LDS, so that rows are written in pieces of
// 64 * CT bytes (straight from the tiles they would be 64 bytes of each of sixteen rows, one after the other in the same memory channel).
// The low-rank values, the sum of their parts times the scale, go through LDS once a block: float32 as they are; for bfloat16 weights as three bfloat16
// pieces, the leading, middle and last eight bits, whose sum is the value, so nothing is rounded (products more on matrix cores that wait for
// memory anyway).  A lane's weights of another slice than the one at hand are zero.  Bound by writing y (and reading it, where it is added to).
// grid: (windows, blocks of 64 * CT columns, each)
template <typename T, int CT, bool VEC>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a, const float* __restrict__ v, int each, int parts, int write) {
  constexpr int P = 16 / sizeof(T), STEP = 4 * P;        // ranks a piece and a step
  constexpr int PIECES = sizeof(T) == 2 ? 3 : 1, CHUNK = 64, STEPS = CHUNK / STEP;      // ranks at a time
  constexpr int ROW = CHUNK * sizeof(T) + 16;            // bytes of a row of low-rank values in LDS, a bank group more than the values
  constexpr int WIDE = 16 * CT, OUT = WIDE + 4;          // columns of a wave, and floats of a row on its way out
  constexpr int MOST = AD_WINDOW * CHUNK / 4 / 256;
  __shared__ __attribute__((aligned(16))) unsigned char low[PIECES][AD_WINDOW * ROW];
  __shared__ __attribute__((aligned(16))) float tile[4][16 * OUT];
  __shared__ int order[AD_WINDOW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
  const int n0 = blockIdx.y * 4 * WIDE, n1 = min(n0 + 4 * WIDE, a.N), ranks = a.rank * a.slices;
  const int w0 = n0 + wave * WIDE, w1 = min(w0 + WIDE, a.N);
  const int s0 = a.interleaved ? 0 : slice_of(a, n0), s1 = a.interleaved ? 1 : slice_of(a, n1 - 1);
  for (int which = blockIdx.z;; which += each) {
    int slot;
    __syncthreads();
    const int count = window_rows(a, blockIdx.x, which, order, slot);
    if (count == 0) return;
    if (slot < 0) {
      if (write) {
        for (int i = 0; i < count; ++i) {
          float* y = a.y + (size_t)order[i] * a.N;
          for (int n = n0 + threadIdx.x; n < n1; n += 256) y[n] = 0.f;
        }
      }
      continue;
    }
    const int tiles = (count + 15) >> 4;
    const float scale = a.scale[slot];
    for (int s = s0; s <= s1; ++s) {
      const int from = a.interleaved ? w0 : max(w0, s > 0 ? a.ends[s - 1] : 0), to = a.interleaved ? w1 : min(w1, a.ends[s]);     // this wave's columns
      for (int j0 = 0; j0 < a.rank; j0 += CHUNK) {
        const bool add = !write || j0 > 0;
        ad_u32x4 bf[CT][STEPS];
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const int col = w0 + 16 * i + c;
          const bool mine = col >= from && col < to && (!a.interleaved || ((col >> 3) & 1) == s);
          const T* B = (const T*)a.b + ((size_t)slot * a.N + min(col, a.N - 1)) * a.rank;
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            const int j = j0 + k * STEP + g * P;
            bf[i][k] = (ad_u32x4){0, 0, 0, 0};
            if (mine && j < a.rank) bf[i][k] = *(const ad_u32x4*)(B + j);
          }
        }
        __syncthreads();
        // (four values at a time, zeros up to a whole step of ranks; two parts of all of a thread's values are asked for together)
        const int quads = min(CHUNK, (a.rank - j0 + STEP - 1) / STEP * STEP) / 4, items = tiles * 16 * quads;
        ad_f32x4 sum[MOST];
#pragma unroll
        for (int it = 0; it < MOST; ++it) sum[it] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < parts; k += 2) {
          ad_f32x4 part[2][MOST];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int it = 0; it < MOST; ++it) {
              const int e = threadIdx.x + it * 256, row = e / quads, j = j0 + e % quads * 4;
              part[h][it] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
              if (e < items && row < count && j < a.rank && k + h < parts)
                part[h][it] = *(const ad_f32x4*)(v + ((size_t)(k + h) * a.rows + order[row]) * ranks + s * a.rank + j);
            }
#pragma unroll
          for (int it = 0; it < MOST; ++it) sum[it] = (sum[it] + part[0][it]) + part[1][it];
        }
#pragma unroll
        for (int it = 0; it < MOST; ++it) {
          const int e = threadIdx.x + it * 256, row = e / quads, j = e % quads * 4;
          if (e >= items) break;
          float left[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) left[i] = sum[it][i] * scale;
          if constexpr (PIECES == 1) {
            *(float4*)(low[0] + row * ROW + j * 4) = make_float4(left[0], left[1], left[2], left[3]);
          } else {
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
              unsigned bits[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool finite = fabsf(left[i]) <= 3.4028234e38f;      // (else the first piece says it)
                bits[i] = __builtin_bit_cast(unsigned, left[i]) & 0xffff0000u;
                left[i] = finite ? left[i] - __builtin_bit_cast(float, bits[i]) : 0.f;
              }
              *(uint2*)(low[p] + row * ROW + j * 2) = make_uint2((bits[0] >> 16) | bits[1], (bits[2] >> 16) | bits[3]);
            }
          }
        }
        __syncthreads();
        if (from >= to) continue;
        for (int t = 0; t < tiles; ++t) {
          ad_f32x4 acc[CT];
#pragma unroll
          for (int i = 0; i < CT; ++i) acc[i] = (ad_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            if (j0 + k * STEP >= a.rank) break;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
              const ad_u32x4 lf = *(const ad_u32x4*)(low[p] + (t * 16 + c) * ROW + (k * 4 + g) * 16);
#pragma unroll
              for (int i = 0; i < CT; ++i) mfma_piece<T>(bf[i][k], lf, acc[i]);
            }
          }
          // (the wave's own part of LDS: its writes and reads follow each other without a barrier)
#pragma unroll
          for (int i = 0; i < CT; ++i) *(ad_f32x4*)(tile[wave] + c * OUT + i * 16 + 4 * g) = acc[i];
          __builtin_amdgcn_wave_barrier();
          constexpr int LANES = WIDE / 4, ROWS = 64 / LANES;      // of a row; rows at a time
#pragma unroll
          for (int i = 0; i < 16 / ROWS; ++i) {
            const int row = i * ROWS + lane / LANES, col = lane % LANES * 4;
            // (another slice's columns between this one's: zero times these low-rank values, no numbers where the values are infinite)
            if (t * 16 + row >= count || (a.interleaved && (((w0 + col) >> 3) & 1) != s)) continue;
            ad_f32x4 value = *(const ad_f32x4*)(tile[wave] + row * OUT + col);
            float* y = a.y + (size_t)order[t * 16 + row] * a.N + w0 + col;
            if (VEC && w0 + col >= from && w0 + col + 4 <= to) {
              if (add) value += *(const ad_f32x4*)y;
              *(ad_f32x4*)y = value;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (w0 + col + r >= from && w0 + col + r < to) y[r] = add ? y[r] + value[r] : value[r];
            }
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
  }
}

template <typename T, bool VEC>
static void adapter_down(const AdapterArgs& g, dim3 grid, int rt, float* v, int each, int part_k, hipStream_t s) {
  if (rt == 1) adapter_down_kernel<T, 1, VEC><<<grid, 256, 0, s>>>(g, v, each, part_k);
  else if (rt == 2) adapter_down_kernel<T, 2, VEC><<<grid, 256, 0, s>>>(g, v, each, part_k);
  else adapter_down_kernel<T, 4, VEC><<<grid, 256, 0, s>>>(g, v, each, part_k);
}

template <typename T>
static void adapter_many(const AdapterArgs& g, int parts, int vec, int write, float* v, hipStream_t s) {
  constexpr int SK = 128 / sizeof(T);
  const int windows = (g.rows + AD_WINDOW - 1) / AD_WINDOW, ranks = g.rank * g.slices;
  // (blocks that find no further adapter in their window end at once)
  const int each = windows >= 32 ? 4 : 8;
  const int rt = ranks <= 16 ? 1 : ranks <= 32 ? 2 : 4;
  const int part_k = ((g.K + parts - 1) / parts + 4 * SK - 1) / (4 * SK) * (4 * SK);
  const dim3 down(windows, (g.K + part_k - 1) / part_k, (ranks + 16 * rt - 1) / (16 * rt) * each);
  if (vec && g.K % SK == 0) {
    if (rt == 1) adapter_down_lds_kernel<T, 1, 6><<<down, 256, 0, s>>>(g, v, each, part_k);
    else if (rt == 2) adapter_down_lds_kernel<T, 2, 6><<<down, 256, 0, s>>>(g, v, each, part_k);
    else adapter_down_lds_kernel<T, 4, 4><<<down, 256, 0, s>>>(g, v, each, part_k);
  } else if (vec) {
    adapter_down<T, true>(g, down, rt, v, each, part_k, s);
  } else {
    adapter_down<T, false>(g, down, rt, v, each, part_k, s);
  }
  // (128 columns a wave, unless that leaves CUs without a block: then 32)
  const bool y16 = g.N % 4 == 0 && ((uintptr_t)g.y & 15) == 0, wide = (long)windows * ((g.N + 511) / 512) >= 192;
  const dim3 up(windows, wide ? (g.N + 511) / 512 : (g.N + 127) / 128, each);
  if (wide) {
    if (y16) adapter_up_kernel<T, 8, true><<<up, 256, 0, s>>>(g, v, each, down.y, write);
    else adapter_up_kernel<T, 8, false><<<up, 256, 0, s>>>(g, v, each, down.y, write);
  } else {
    if (y16) adapter_up_kernel<T, 2, true><<<up, 256, 0, s>>>(g, v, each, down.y, write);
    else adapter_up_kernel<T, 2, false><<<up, 256, 0, s>>>(g, v, each, down.y, write);
  }
}

// y [rows, N] float32 += the adapters' share.  a [slots, slices * rank, K], b [slots, N, rank] of dt, rank a multiple of 8; vec: K is a multiple of
// 8 and x and a are aligned to 16 bytes.  ends: the columns at which the slices end (the last is N).  parts 0: row by row, in one launch, or with
// scratch of rows * slices * rank floats in two; else rows taken together by adapter, K in up to `parts` parts, with scratch of parts times as many floats
// aligned to 16 bytes; `write`: y is written
// instead (zeros for rows without an adapter).
extern "C" int tp_adapter_add(const int* ids, const void* x, int dt, const void* a, const void* b, const float* scale, float* y, int rows, int K, int N,
                              int slots, int rank, int slices, int interleaved, const int* ends, int vec, int parts, int write, float* scratch, hipStream_t s) {
  if (rows <= 0 || N <= 0) return 0;
  TP_REQUIRE(dt == TP_BF16 || dt == TP_F32, "adapter_add: unsupported element type");
  TP_REQUIRE(K > 0 && slots > 0 && rank > 0 && rank % 8 == 0 && slices >= 1 && slices <= AD_MAX_SLICES, "adapter_add: bad sizes");
  TP_REQUIRE(!interleaved || (slices == 2 && N % 16 == 0), "adapter_add: two interleaved slices");
  AdapterArgs g = {ids, x, a, b, scale, y, rows, K, N, slots, rank, slices, interleaved, {}};
  for (int i = 0; i < slices; ++i) g.ends[i] = ends[i];
  if (parts > 0) {
    TP_REQUIRE(scratch != nullptr && parts <= AD_PARTS, "adapter_add: no room for the low-rank rows");
    if (dt == TP_BF16) adapter_many<bf16_t>(g, parts, vec, write, scratch, s);
    else adapter_many<float>(g, parts, vec, write, scratch, s);
    TP_CHECK_LAUNCH("adapter_add");
    return 0;
  }
  TP_REQUIRE(!write, "adapter_add: a block a row adds");
  TP_REQUIRE(rows <= 65535, "adapter_add: too many rows");
  // (as many columns a block as threads, unless that leaves CUs without a block)
  int cols = AD_ROW_THREADS;
  while (cols > 256 && (long)rows * ((N + cols - 1) / cols) < 128) cols /= 2;
  const dim3 grid((N + cols - 1) / cols, rows);
  const size_t lds = (size_t)slices * rank * sizeof(float);
  TP_REQUIRE(lds <= 65536, "adapter_add: ranks of all slices beyond 16,384");
#define AD_ROWS(T, VEC)                                                                                                     \
  if (scratch != nullptr) {                                                                                                 \
    adapter_rows_down_kernel<T, VEC><<<dim3((slices * rank + 3) / 4, rows), 256, 0, s>>>(g, scratch);                       \
    adapter_rows_kernel<T, VEC, 1, true><<<grid, cols, lds, s>>>(g, scratch, cols);                                         \
  } else if (rank <= 16) {                                                                                                  \
    adapter_rows_kernel<T, VEC, 1, false><<<grid, AD_ROW_THREADS, lds, s>>>(g, nullptr, cols);                              \
  } else {                                                                                                                  \
    adapter_rows_kernel<T, VEC, 2, false><<<grid, AD_ROW_THREADS, lds, s>>>(g, nullptr, cols);                              \
  }
  if (dt == TP_BF16 && vec) {
    AD_ROWS(bf16_t, true)
  } else if (dt == TP_BF16) {
    AD_ROWS(bf16_t, false)
  } else if (vec) {
    AD_ROWS(float, true)
  } else {
    AD_ROWS(float, false)
  }
#undef AD_ROWS
  TP_CHECK_LAUNCH("adapter_add");
  return 0;
}
