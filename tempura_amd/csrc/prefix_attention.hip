// Attention of a step whose requests begin with the same keys, the shared pages read once for a group of requests instead of
// once for each of them.
//
// A group is a run of neighbouring requests of the batch whose block tables begin with the same pages: its first P keys.  Every
// query of the group sees all of them, so for one key head all (token, head) pairs of the group are the rows of ONE product with
// those keys, no mask between them; behind them each request has keys of its own, of which its tokens see those up to themselves.
// A block takes one key head, 16, 64 or 128 rows and one part of the keys (a group's shared ones or a request's own) and leaves the
// rows' partial results: O (unnormalised), maximum and sum.  A second kernel joins a row's parts in ascending order:
//   m = max m_s,   out = sum_s 2^(m_s - m) O_s / (sum_s 2^(m_s - m) l_s + 2^(sink - m)).
//
// The step of 32 keys is computed transposed, so that no operand is transposed in LDS (values are cached transposed):
//   S^T[key, row] = K[key, :] . Q[row, :]^T      O^T[d, row] += V^T[d, keys] . P^T[keys, row]
// with v_mfma_f32_16x16x32_bf16, float32 caches with v_mfma_f32_16x16x4_f32.  A 16x16 result gives lane (c = lane % 16, g = lane / 16)
// the rows 4 g + r of column c.  bfloat16: the two key tiles of a step take their keys in the order 8 (i / 4) + 4 t + i % 4, so a lane
// ends up with the eight CONSECUTIVE keys 8 g .. of its row, the operand of the next product.  float32: the order is 16 t + i, a lane has
// the keys 16 t + 4 g + r, and the product with register r of tile t takes exactly these as its four k.  A fragment is 16 bytes a lane either way.
// Statistics and sums are float32; the probabilities of bfloat16 caches are rounded to bfloat16 for the second product (errors of up to
// 2^-8 of each, which average out in the sum, itself rounded to bfloat16 at the end).
//
// Two forms of a block of four waves, both fed by direct global-to-LDS loads in whole kilobytes: 16 rows, which every wave takes with a run of
// the part's steps of its own (prefix_part), and 64 or 128, of which every wave takes a quarter through all steps (prefix_part_rows).  The first asks for
// the keys once for every 16 rows, from an L2 that has them, but divides a part's steps by four and needs no barrier: best where rows and keys are few
// for the chip.  32 heads of 128 over 8, requests behind shared keys (16 / 64 / 128 rows a block, each with its best parts, us): 16 behind 2,048
// 12.7 / 14.2 / 14.9, 32 behind 2,048 14.9 / 17.1 / 19.9, 64 behind 4,096 27.3 / 26.1 / 27.8, 32 behind 16,384 36.3 / 32.9 / 31.6.
// Bound by: few rows, the trips to memory that a part begins and ends with (8 requests behind 2,048 keys: 12 us for 16 MB); many rows, the rate at which a
// CU takes a step of one block's products beside another's exponentials (16 requests of up to 24 tokens behind 6,000 keys: 44 us, 440 TFLOP/s).
#include <math.h>

#include "common.h"

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int pa_u32x4 __attribute__((ext_vector_type(4)));

#define PA_WAVES 4
#define PA_MAX_PARTS 128    // a row's parts: the joining kernel holds two parts' statistics a lane
#define PA_LPTR(p) ((__attribute__((address_space(3))) void*)(p))
#define PA_WAIT_VM(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")
#define PA_WAIT_LDS() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

struct PrefixArgs {
  const void* q;             // [tokens, heads, D]
  const void* k_cache;       // [pages, kv heads, page size, D]
  const void* v_cache;       // [pages, kv heads, D, page size]
  const int* block_tables;
  const int* cu_seqlens;
  const int* context_lens;
  const int* group_starts;   // [groups + 1] requests
  const int* group_keys;     // [groups] keys that the group's requests share
  const int* shared_keys;    // [requests] the same, for each request
  float* sums;               // [token, head, part, D]
  float* stats;              // [token, head, part, 2]: maximum, sum
  int table_width, page_shift, n_heads, n_kv, groups, requests;
  int single;                // every request brings one token: request r's is token r
  int shared_blocks;         // blocks (of rows and parts) that take shared keys, a key head each; the own keys' come behind them.  An upper
                             // bound: those beyond the last group end at once
  int own_rows;              // blocks of rows of a request
  int shared_steps, own_steps;   // steps of 32 keys a part has
  int shared_parts, parts;   // a row's places for parts: those of the shared keys, all
  float scale_log2;          // scale * log2(e)
  float cap_log2, cap_in;    // scores under a cap: cap * log2(e), and what turns q . k into score / cap (bfloat16: 2 log2(e) score / cap); 0: no cap
};

__device__ inline unsigned pa_pack(float a, float b) {
  const pa_f32x2 f = {a, b};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(f, pa_bf16x2));
}
__device__ inline pa_u32x4 pa_lds(unsigned addr) {
  pa_u32x4 v;
  asm volatile("ds_read_b128 %0, %1" : "=v"(v) : "v"(addr));
  return v;
}
__device__ inline void pa_lds_at(unsigned addr, int offset, pa_u32x4& v) { asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(offset)); }
// the maximum over the four lanes of a column
__device__ inline float pa_column_max(float v) {
  LanePair p = lanes_32(v);
  p = lanes_16(fmaxf(p.a, p.b));
  return fmaxf(p.a, p.b);
}

// What a block's waves compute: rows and keys of one part.
struct PartRows {
  int token0, rows, row0;    // the rows are pairs (token, head of the key head) from pair row0 of token0's first on, `rows` in all
  int first, end;            // keys
  int limit0;                // the last key that token0 sees (a token's successor sees one more); large: every key
  const int* table;
  int part;
};

// Where a lane stands in a step of 32 keys (E: bytes of an element): its place in each kilobyte that is loaded, and its fragments' places in LDS.
// In LDS a step is its keys as 32 rows of D elements, chunk x of 16 bytes of the row with place i in its tile at (x + f(i)) mod the chunks,
// so that the 16 rows a quarter of a wave reads fall into different banks; behind them its values in kilobytes of VD elements and half of the keys,
// the e-th 16 bytes of an element at place VD e + d % VD.
template <int E, int D>
struct PrefixLane {
  static constexpr int CH = D * E / 16, SH = CH >= 16 ? 0 : CH == 8 ? 1 : 2;      // 16-byte chunks of a key
  static constexpr int KF = CH / 4, DT = D / 16, VF = E / 2;                      // a lane's chunks: of a key, tiles of elements, of an element's 32 keys
  static constexpr int KI = D * E / 32, STAGE = 2 * KI * 1024, VD = 64 / E;       // loads of a step's keys (values likewise), its bytes
  unsigned kaddr[2], vaddr;
  int c, g;
  __device__ inline PrefixLane(int lane) : c(lane & 15), g(lane >> 4) {
#pragma unroll
    for (int t = 0; t < 2; ++t) kaddr[t] = (E == 2 ? 8 * (c >> 2) + 4 * t + (c & 3) : 16 * t + c) * (CH * 16);
    // (bfloat16: the keys 8 g .. lie in half g / 2, chunk g % 2; float32: the keys 16 t + 4 g .. in half t, chunk g)
    vaddr = KI * 1024 + (E == 2 ? (g >> 1) * 1024 + (g & 1) * 512 : g * 256) + c * 16;
  }
  // of load t of the keys: its offset from the first key of its half; of the values: from the half's first place of the load's first element
  static __device__ inline unsigned key_offset(int t, int lane) {
    const int row = (64 * t + lane) / CH, pc = (64 * t + lane) % CH;
    const int i = E == 2 ? 4 * (row >> 3) + (row & 3) : row & 15;
    return (unsigned)((row & 15) * (D * E) + ((pc - (i >> SH) + CH) % CH) * 16);
  }
  static __device__ inline unsigned value_offset(int lane, int ps) { return (unsigned)((lane % VD) * (ps * E) + (lane / VD) * 16); }
  __device__ inline void read_keys(unsigned base, pa_u32x4 (&kk)[2][KF]) const {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int f = 0; f < KF; ++f) kk[t][f] = pa_lds(base + kaddr[t] + ((f * 4 + g + (c >> SH)) % CH) * 16);
  }
  __device__ inline void read_values(unsigned base, pa_u32x4 (&vv)[DT][VF]) const {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int t = 0; t < VF; ++t) {
        const unsigned at = base + vaddr;
        pa_lds_at(at, (E == 2 ? (dt >> 1) * 2048 + (dt & 1) * 256 : dt * 2048 + t * 1024), vv[dt][t]);
      }
  }
  template <int A, int B>
  static __device__ inline void arrived(pa_u32x4 (&v)[A][B]) {
    PA_WAIT_LDS();
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
      for (int j = 0; j < B; ++j) asm volatile("" : "+v"(v[i][j]));
  }
};

// 16 bytes a lane from base + the lane's offset into a kilobyte of LDS.  (As buffer loads from a uniform base: no vector arithmetic a load.)
template <bool NT>
__device__ inline void prefix_copy(const unsigned char* base, unsigned offset, unsigned char* lds) {
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, PA_LPTR(lds), 16, offset, 0, 0, NT ? 2 : 0);
}

// One step's scores: S^T of both key tiles.
template <int E, int NQ, int KF>
__device__ inline void prefix_scores(const pa_u32x4 (&kk)[2][KF], const pa_u32x4 (&qf)[NQ][KF], pa_f32x4 (&s)[NQ][2]) {
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
    for (int t = 0; t < 2; ++t) s[nq][t] = (pa_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int f = 0; f < KF; ++f)
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (E == 2) {
          s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, kk[t][f]), __builtin_bit_cast(pa_bf16x8, qf[nq][f]),
                                                             s[nq][t], 0, 0, 0);
        } else {
          const pa_f32x4 kv = __builtin_bit_cast(pa_f32x4, kk[t][f]), qv = __builtin_bit_cast(pa_f32x4, qf[nq][f]);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[e], qv[e], s[nq][t], 0, 0, 0);
        }
      }
}

// Scores under a cap, cap * tanh(score / cap), in units of log 2.  float32: tanhf, exact to a few half steps of the result.  bfloat16: tanh(x) = 1 - 2 / (2^(2 x log2 e) + 1);
// both limits come out right (2^large is infinite, its reciprocal 0), but it is a difference of numbers near the cap, off by a few 1e-8 of the cap (1e-5 of a score
// at a cap of 100, where rounding the weights to bfloat16 is 4e-3 of each), which for float32 would grow beyond everything else.
template <int E, int NQ>
__device__ inline void prefix_cap(const PrefixArgs& a, pa_f32x4 (&s)[NQ][2]) {
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = s[nq][t][r] * a.cap_in;
        s[nq][t][r] = E == 4 ? a.cap_log2 * tanhf(x) : fmaf(-2.0f * a.cap_log2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x) + 1.0f), a.cap_log2);
      }
}

// Keys outside the part or above the row's limit are not in the sums.
template <int E, int NQ>
__device__ inline void prefix_mask(const PartRows& w, int j0, int g, const int (&limit)[NQ], pa_f32x4 (&s)[NQ][2]) {
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    const int hi = min(w.end - 1, limit[nq]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int key = j0 + (E == 2 ? 8 * g + j : 16 * (j >> 2) + 4 * g + (j & 3));
      if (key < w.first || key > hi) s[nq][j >> 2][j & 3] = -INFINITY;
    }
  }
}

// The scores' probabilities, as the next product's operand (pf): 2^(score - m), one fused multiply-add and one exponential each.  m is a maximum seen
// before, and stays while no score is more than PA_SLACK above it: probabilities up to 2^PA_SLACK are as exact, relative to each other, as those up to 1
// (float32 sums, bfloat16 roundings), and the sums so far need not be scaled, nor the lanes' maxima compared, in almost any step.  (With a maximum that
// is one in every step, one of 32 rows moves it in most of the first thirty.)
#define PA_SLACK 8.0f
template <int E, int NQ, int DT>
__device__ inline void prefix_softmax(float scale, pa_f32x4 (&s)[NQ][2], float (&m)[NQ], float (&l)[NQ], pa_u32x4 (&pf)[NQ][E / 2], pa_f32x4 (&o)[NQ][DT]) {
  float top[NQ];
  bool above = false;
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    top[nq] = scale * fmaxf(fmaxf(fmaxf(s[nq][0][0], s[nq][0][1]), fmaxf(s[nq][0][2], s[nq][0][3])),     // (the scale is positive)
                            fmaxf(fmaxf(s[nq][1][0], s[nq][1][1]), fmaxf(s[nq][1][2], s[nq][1][3])));
    above |= top[nq] > m[nq] + PA_SLACK;
  }
  if (__builtin_amdgcn_ballot_w64(above) != 0) {
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      const float m_new = fmaxf(m[nq], pa_column_max(top[nq]));
      const float shrink = __builtin_amdgcn_exp2f(m[nq] - (m_new == -INFINITY ? 0.f : m_new));
      l[nq] *= shrink;
      m[nq] = m_new;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[nq][dt][r] *= shrink;
    }
  }
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    const float use = m[nq] == -INFINITY ? 0.f : m[nq];   // (a row that has seen no key yet)
    pa_f32x4 v[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[t][r] = __builtin_amdgcn_exp2f(fmaf(s[nq][t][r], scale, -use));
    // (this lane's keys; the lanes of a column are added at the end)
    l[nq] += ((v[0][0] + v[0][1]) + (v[0][2] + v[0][3])) + ((v[1][0] + v[1][1]) + (v[1][2] + v[1][3]));
    if constexpr (E == 2) {
      pf[nq][0] = (pa_u32x4){pa_pack(v[0][0], v[0][1]), pa_pack(v[0][2], v[0][3]), pa_pack(v[1][0], v[1][1]), pa_pack(v[1][2], v[1][3])};
    } else {
      pf[nq][0] = __builtin_bit_cast(pa_u32x4, v[0]);
      pf[nq][1] = __builtin_bit_cast(pa_u32x4, v[1]);
    }
  }
}

// Places behind the part's last key hold whatever an earlier owner of the page left there; their probabilities are 0, but 0 * NaN and 0 * Inf are
// not, so they are cleared.
template <int E, int DT, int VF>
__device__ inline void prefix_clear(int end, int j0, int g, pa_u32x4 (&vv)[DT][VF]) {
#pragma unroll
  for (int t = 0; t < VF; ++t) {
    const int left = end - (j0 + (E == 2 ? 8 * g : 16 * t + 4 * g));
    pa_u32x4 keep;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      keep[e] = E == 2 ? (2 * e < left ? 0x0000ffffu : 0u) | (2 * e + 1 < left ? 0xffff0000u : 0u) : e < left ? 0xffffffffu : 0u;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vv[dt][t] &= keep;
  }
}

// acc += a . b over a step's keys, of one tile of elements and one of rows
template <int E, int VF>
__device__ inline void prefix_product(const pa_u32x4 (&a)[VF], const pa_u32x4 (&b)[VF], pa_f32x4& acc) {
  if constexpr (E == 2) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, a[0]), __builtin_bit_cast(pa_bf16x8, b[0]), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const pa_f32x4 x = __builtin_bit_cast(pa_f32x4, a[t]), y = __builtin_bit_cast(pa_f32x4, b[t]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    }
  }
}

// o += values x probabilities
template <int E, int NQ, int DT, int VF>
__device__ inline void prefix_values(const pa_u32x4 (&vv)[DT][VF], const pa_u32x4 (&pf)[NQ][VF], pa_f32x4 (&o)[NQ][DT]) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) prefix_product<E, VF>(vv[dt], pf[nq], o[nq][dt]);
}

// Where a row may not see all of the step's keys a value that is not finite has to stay away from the rows in front of it (0 * Inf and 0 * NaN are not 0).  If there is
// one, which portions of numbers never have, zeros take the place of such values, and the sums get what they would have brought: a product counts for each row and
// element those that the row sees, 1 for a positive infinity, 64 for a negative one and 4,096 for what is no number (at most 32 of each: exact).  (In integer
// arithmetic: comparisons' masks would take the scalar registers that the steps' addresses live in.  Steps of numbers pay the check: 6,240 rows behind 6,000 keys 43.7 -> 44.0
// us, 32 single tokens of 1,000 own keys beside a portion of 64 51.6 -> 52.2, float32
// 378 -> 393.)
template <int E, int NQ, int DT, int VF>
__device__ inline void prefix_odd_values(const PartRows& w, int j0, int g, const int (&limit)[NQ], pa_u32x4 (&vv)[DT][VF], pa_f32x4 (&o)[NQ][DT]) {
  constexpr unsigned EXP = E == 2 ? 0x7f807f80u : 0x7f800000u, STEP = E == 2 ? 0x00800080u : 0x00800000u, TOP = E == 2 ? 0x80008000u : 0x80000000u;
  unsigned odd = 0;      // (an exponent of all ones carries into the sign's place)
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int t = 0; t < VF; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= ((vv[dt][t][e] & EXP) + STEP) & TOP;
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) == 0, 1)) return;
  auto all = [](unsigned n) { return 0u - min(n, 1u); };      // all bits, unless n is 0
  constexpr unsigned ONE = 0x3f80u, MINUS = 0x4280u, NONE = 0x4580u;      // 1, 64 and 4,096: the upper halves of their float32 bits
  pa_u32x4 sees[NQ][VF];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    const int from = max(w.first, j0), upto = max(from, min(w.end - 1, limit[nq]) + 1);
    auto seen = [&](int key) { return (unsigned)((from - 1 - key) >> 31) & (unsigned)((key - upto) >> 31) & ONE; };
#pragma unroll
    for (int t = 0; t < VF; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = j0 + (E == 2 ? 8 * g + 2 * e : 16 * t + 4 * g + e);
        sees[nq][t][e] = E == 2 ? seen(key) | seen(key + 1) << 16 : seen(key) << 16;
      }
  }
  // (the upper 16 bits of a float32 value say whether it is finite, and its sign; the lower ones beside them whether it is an infinity)
  auto mark = [&](unsigned v, unsigned rest) {
    const unsigned none = all((v & 0x7fu) | rest), minus = all(v & 0x8000u);
    return all(((v & 0x7f80u) + 0x80u) & 0x8000u) & ((none & NONE) | (~none & ((minus & MINUS) | (~minus & ONE))));
  };
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    pa_u32x4 marks[VF];
#pragma unroll
    for (int t = 0; t < VF; ++t) {
      // (one tile behind the other, so that they need no registers beyond those of the steps without such values)
      asm volatile("" : "+v"(vv[dt][t]));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned v = vv[dt][t][e], hi = mark(v >> 16, E == 4 ? v & 0xffffu : 0u), lo = E == 2 ? mark(v & 0xffffu, 0u) : 0u;
        marks[t][e] = hi << 16 | lo;
        vv[dt][t][e] = v & ~(E == 2 ? (all(hi) & 0xffff0000u) | (all(lo) & 0x0000ffffu) : all(hi));
      }
      asm volatile("" : "+v"(vv[dt][t]), "+v"(marks[t]));
    }
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      pa_f32x4 count = {0.f, 0.f, 0.f, 0.f};
      prefix_product<E, VF>(marks, sees[nq], count);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const unsigned n = (unsigned)count[r];
        const float plus = __builtin_bit_cast(float, all(n & 63u) & 0x7f800000u), minus = __builtin_bit_cast(float, all(n & 4032u) & 0xff800000u);
        o[nq][dt][r] += (plus + minus) + __builtin_bit_cast(float, all(n >> 12) & 0x7fc00000u);
      }
    }
  }
}

// q of a wave's rows from `at` of the part's on, their places among all (token, head) rows and the last key each sees.
template <int E, int D, int NQ, int KF>
__device__ inline void prefix_queries(const PrefixArgs& a, const PartRows& w, int kvh, int at, int c, int g, pa_u32x4 (&qf)[NQ][KF], int (&limit)[NQ],
                                      size_t (&row)[NQ]) {
  const int group = a.n_heads / a.n_kv;
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    const int pair = w.row0 + min(at + nq * 16 + c, w.rows - 1), token = pair / group;
    row[nq] = (size_t)(w.token0 + token) * a.n_heads + kvh * group + pair % group;
    const unsigned char* q = (const unsigned char*)a.q + row[nq] * (D * E) + g * 16;
#pragma unroll
    for (int i = 0; i < KF; ++i) qf[nq][i] = *(const pa_u32x4*)(q + i * 64);
    limit[nq] = w.limit0 == 0x7fffffff ? w.limit0 : w.limit0 + token;
  }
}

// Few rows: every wave takes all of them and a run of the part's steps, through a ring of its own of one step, filled again as soon as its
// fragments are in registers; no barrier until the waves' sums are added.  (Two blocks a CU: eight steps on their way.)  OWN: a request's own keys,
// which one block reads and of which a row may not see all.
template <int E, int D, int NQ, bool OWN>
__device__ inline void prefix_part(const PrefixArgs& a, unsigned char* stages, const PartRows& w, int kvh) {
  using L = PrefixLane<E, D>;
  constexpr int KF = L::KF, DT = L::DT, VF = L::VF, KI = L::KI;
  static_assert(2 * KI <= 63 && L::STAGE >= (D * 17 + 32) * 4, "the waits below; room for the sums of a tile");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L at(lane);
  const int g = at.g, c = at.c;
  const int psh = a.page_shift, ps = 1 << psh, pmask = ps - 1;
  unsigned koff[KI];
#pragma unroll
  for (int t = 0; t < KI; ++t) koff[t] = L::key_offset(t, lane);
  const unsigned voff = L::value_offset(lane, ps);
  const size_t page_bytes = (size_t)a.n_kv * D * ps * E;
  const unsigned char* kbase = (const unsigned char*)a.k_cache + (size_t)kvh * ps * D * E;
  const unsigned char* vbase = (const unsigned char*)a.v_cache + (size_t)kvh * ps * D * E;
  unsigned char* ring = stages + wave * L::STAGE;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)ring;
  // (block tables through the constant address space: uniform loads from it are scalar loads)
  const __attribute__((address_space(4))) int* table = (const __attribute__((address_space(4))) int*)(uintptr_t)w.table;
  const int base16 = w.first & ~15;                           // (a step's halves of 16 keys lie in one page each)
  const int steps = (w.end - base16 + 31) >> 5, run = (steps + PA_WAVES - 1) / PA_WAVES;
  const int w0 = wave * run, n = max(0, min(steps - w0, run));
  const int last16 = (w.end - 1) & ~15;
  int pp0 = 0, pp1 = 0;
  auto pages_of = [&](int i) {
    const int j0 = base16 + (w0 + i) * 32;
    pp0 = max(table[j0 >> psh], 0);      // (an entry that names no page reads page 0, not what lies in front of the pool)
    pp1 = max(table[min(j0 + 16, last16) >> psh], 0);
  };
  auto issue_keys = [&](int i) __attribute__((always_inline)) {
    const int j0 = base16 + (w0 + i) * 32, j1 = min(j0 + 16, last16);
    const unsigned char* b0 = kbase + (size_t)(unsigned)pp0 * page_bytes + (unsigned)((j0 & pmask) * (D * E));
    const unsigned char* b1 = kbase + (size_t)(unsigned)pp1 * page_bytes + (unsigned)((j1 & pmask) * (D * E));
#pragma unroll
    for (int t = 0; t < KI; ++t) prefix_copy<OWN>(t >= KI / 2 ? b1 : b0, koff[t], ring + t * 1024);
  };
  auto issue_values = [&](int i) __attribute__((always_inline)) {
    const int j0 = base16 + (w0 + i) * 32, j1 = min(j0 + 16, last16);
    const unsigned char* b0 = vbase + (size_t)(unsigned)pp0 * page_bytes + (unsigned)((j0 & pmask) * E);
    const unsigned char* b1 = vbase + (size_t)(unsigned)pp1 * page_bytes + (unsigned)((j1 & pmask) * E);
#pragma unroll
    for (int t = 0; t < KI; ++t) prefix_copy<OWN>(((t & 1) ? b1 : b0) + (size_t)((t >> 1) * L::VD * E) * ps, voff, ring + (KI + t) * 1024);
  };
  pa_u32x4 qf[NQ][KF];
  int limit[NQ];
  size_t row[NQ];
  float m[NQ], l[NQ];
  pa_f32x4 o[NQ][DT];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    m[nq] = -INFINITY;
    l[nq] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[nq][dt] = (pa_f32x4){0.f, 0.f, 0.f, 0.f};
  }
  if (n > 0) {
    pages_of(0);
    prefix_queries<E, D, NQ, KF>(a, w, kvh, 0, c, g, qf, limit, row);
    issue_keys(0);
    issue_values(0);
    if (n > 1) pages_of(1);
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)      // (q is waited for here, in front of the loop, whose waits would else wait for everything)
#pragma unroll
      for (int i = 0; i < KF; ++i) asm volatile("" : "+v"(qf[nq][i]));
    float cap = a.cap_in;
    const float scale = cap > 0.f ? 1.f : a.scale_log2;
    for (int i = 0; i < n; ++i) {
      asm volatile("" : "+s"(cap));      // (a branch of a few instructions, not two loops)
      const bool more = i + 1 < n;
      const int j0 = base16 + (w0 + i) * 32;
      PA_WAIT_VM(KI);
      pa_u32x4 kk[2][KF], vv[DT][VF];
      at.read_keys(lds0, kk);
      L::arrived(kk);
      if (more) issue_keys(i + 1);
      pa_f32x4 sc[NQ][2];
      pa_u32x4 pf[NQ][VF];
      prefix_scores<E, NQ, KF>(kk, qf, sc);
      if (cap > 0.f) prefix_cap<E, NQ>(a, sc);
      if (j0 < w.first || j0 + 32 > w.end || w.limit0 < j0 + 31) prefix_mask<E, NQ>(w, j0, g, limit, sc);
      prefix_softmax<E, NQ, DT>(scale, sc, m, l, pf, o);
      if (more) PA_WAIT_VM(KI);
      else PA_WAIT_VM(0);
      at.read_values(lds0, vv);
      L::arrived(vv);
      if (more) {
        issue_values(i + 1);
        if (i + 2 < n) pages_of(i + 2);
      }
      if (j0 + 32 > w.end) prefix_clear<E, DT, VF>(w.end, j0, g, vv);
      if (OWN && w.limit0 < j0 + 31) prefix_odd_values<E, NQ, DT, VF>(w, j0, g, limit, vv, o);
      prefix_values<E, NQ, DT, VF>(vv, pf, o);
    }
  }

  // The waves' sums, added in their order through LDS, a tile of 16 rows at a time (rows a bank apart: 17 floats an element)
  const int group = a.n_heads / a.n_kv;
  float* red = (float*)stages;
  float* stat = red + PA_WAVES * D * 17;
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    __syncthreads();     // (every ring is empty; the tile before is read)
    float sum = l[nq];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (g == 0) {
      stat[wave * 32 + c] = m[nq];
      stat[wave * 32 + 16 + c] = sum;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[(wave * D + dt * 16 + 4 * g + r) * 17 + c] = o[nq][dt][r];
    __syncthreads();
    const int rows = min(16, w.rows - nq * 16);
    for (int e = threadIdx.x; e < D * rows; e += PA_WAVES * 64) {
      const int d = e % D, col = e / D;
      float top = stat[col];
#pragma unroll
      for (int v = 1; v < PA_WAVES; ++v) top = fmaxf(top, stat[v * 32 + col]);
      const float use = top == -INFINITY ? 0.f : top;
      float acc = 0.f, total = 0.f;
#pragma unroll
      for (int v = 0; v < PA_WAVES; ++v) {
        const float f = __builtin_amdgcn_exp2f(stat[v * 32 + col] - use);
        acc = fmaf(f, red[(v * D + d) * 17 + col], acc);
        total = fmaf(f, stat[v * 32 + 16 + col], total);
      }
      const int pair = w.row0 + nq * 16 + col;
      const size_t to = ((size_t)(w.token0 + pair / group) * a.n_heads + kvh * group + pair % group) * a.parts + w.part;
      a.sums[to * D + d] = acc;
      if (d == 0) *(float2*)(a.stats + to * 2) = make_float2(top, total);
    }
  }
}

// Many rows: the four waves take 16 * NQ rows each and walk the part's steps together, through a ring of NS steps that all of them fill, a quarter each,
// NS - 1 steps ahead; one barrier a step.  So a CU loads a step once for 64 * NQ rows, and one wave's products run beside another's exponentials.
template <int E, int D, int NQ, int NS, bool OWN>
__device__ inline void prefix_part_rows(const PrefixArgs& a, unsigned char* stages, const PartRows& w, int kvh) {
  using L = PrefixLane<E, D>;
  constexpr int KF = L::KF, DT = L::DT, VF = L::VF, KI = L::KI;
  constexpr int LOADS = 2 * KI / PA_WAVES;
  static_assert(NS >= 2 && (2 * KI) % PA_WAVES == 0 && (NS - 1) * LOADS <= 63, "a quarter of a step's loads");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L at(lane);
  const int g = at.g, c = at.c;
  const int psh = a.page_shift, ps = 1 << psh, pmask = ps - 1;
  const size_t page_bytes = (size_t)a.n_kv * D * ps * E;
  const unsigned char* kbase = (const unsigned char*)a.k_cache + (size_t)kvh * ps * D * E;
  const unsigned char* vbase = (const unsigned char*)a.v_cache + (size_t)kvh * ps * D * E;
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)stages;
  const __attribute__((address_space(4))) int* table = (const __attribute__((address_space(4))) int*)(uintptr_t)w.table;
  const int base16 = w.first & ~15, n = (w.end - base16 + 31) >> 5, last16 = (w.end - 1) & ~15;
  // this wave's loads of a step: LOADS of the 2 KI kilobytes, the keys' first.  A wave's loads lie in one half of the keys, and of keys or values alone
  // (but for the smallest heads: two waves load keys, two values, either way)
  const int t0 = wave * LOADS;
  const bool of_keys = t0 < KI;
  unsigned off[LOADS];
  int half[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int t = t0 + j;
    off[j] = of_keys ? L::key_offset(t, lane) : L::value_offset(lane, ps) + (unsigned)(((t - KI) >> 1) * L::VD * E) * ps;
    half[j] = of_keys ? (t >= KI / 2) : (t - KI) & 1;
  }
  int pp0 = 0, pp1 = 0;
  auto pages_of = [&](int i) {
    const int j0 = base16 + i * 32;
    pp0 = max(table[j0 >> psh], 0);      // (an entry that names no page reads page 0, not what lies in front of the pool)
    pp1 = max(table[min(j0 + 16, last16) >> psh], 0);
  };
  const unsigned char* mine = of_keys ? kbase : vbase;
  const int key_bytes = of_keys ? D * E : E;
  auto issue = [&](int i, int st) __attribute__((always_inline)) {
    const int j0 = base16 + i * 32, j1 = min(j0 + 16, last16);
    const unsigned char* b0 = mine + (size_t)(unsigned)pp0 * page_bytes + (unsigned)((j0 & pmask) * key_bytes);
    const unsigned char* b1 = mine + (size_t)(unsigned)pp1 * page_bytes + (unsigned)((j1 & pmask) * key_bytes);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) prefix_copy<false>(half[j] ? b1 : b0, off[j], stages + st * L::STAGE + (t0 + j) * 1024);
  };
  pa_u32x4 qf[NQ][KF];
  int limit[NQ];
  size_t row[NQ];
  float m[NQ], l[NQ];
  pa_f32x4 o[NQ][DT];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    m[nq] = -INFINITY;
    l[nq] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[nq][dt] = (pa_f32x4){0.f, 0.f, 0.f, 0.f};
  }
  prefix_queries<E, D, NQ, KF>(a, w, kvh, wave * NQ * 16, c, g, qf, limit, row);
  // (steps that are not there: the last one again, so that the loads on their way are always as many as the waits below count)
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) {
    pages_of(min(i, n - 1));
    issue(min(i, n - 1), i);
  }
  pages_of(min(NS - 1, n - 1));
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
    for (int i = 0; i < KF; ++i) asm volatile("" : "+v"(qf[nq][i]));
  const bool busy = wave * NQ * 16 < w.rows;      // (a wave without rows loads for the others)
  int st = 0;
  float cap = a.cap_in;
  const float scale = cap > 0.f ? 1.f : a.scale_log2;
  for (int i = 0; i < n; ++i) {
    asm volatile("" : "+s"(cap));        // (a branch of a few instructions, not two loops)
    PA_WAIT_VM((NS - 2) * LOADS);
    __builtin_amdgcn_s_barrier();                 // every wave's share of this step has come, and the step before is read by all
    asm volatile("" ::: "memory");
    issue(min(i + NS - 1, n - 1), st == 0 ? NS - 1 : st - 1);
    pages_of(min(i + NS, n - 1));
    const unsigned base = lds0 + st * L::STAGE;
    st = st + 1 == NS ? 0 : st + 1;
    if (!busy) continue;
    const int j0 = base16 + i * 32;
    pa_u32x4 kk[2][KF], vv[DT][VF];
    at.read_keys(base, kk);
    L::arrived(kk);
    pa_f32x4 sc[NQ][2];
    pa_u32x4 pf[NQ][VF];
    prefix_scores<E, NQ, KF>(kk, qf, sc);
    at.read_values(base, vv);
    if (cap > 0.f) prefix_cap<E, NQ>(a, sc);
    if (j0 < w.first || j0 + 32 > w.end || w.limit0 < j0 + 31) prefix_mask<E, NQ>(w, j0, g, limit, sc);
    prefix_softmax<E, NQ, DT>(scale, sc, m, l, pf, o);
    L::arrived(vv);
    if (j0 + 32 > w.end) prefix_clear<E, DT, VF>(w.end, j0, g, vv);
    if (OWN && w.limit0 < j0 + 31) prefix_odd_values<E, NQ, DT, VF>(w, j0, g, limit, vv, o);
    if constexpr (OWN && E == 2) {      // (both ways here end in the same registers: else every step copies the sums)
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) asm volatile("" : "+v"(o[nq][dt]));
    }
    prefix_values<E, NQ, DT, VF>(vv, pf, o);
  }
  PA_WAIT_VM(0);       // (nothing is on its way into LDS when the block ends)
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    float sum = l[nq];
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if ((wave * NQ + nq) * 16 + c >= w.rows) continue;
    const size_t to = row[nq] * a.parts + w.part;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *(pa_f32x4*)(a.sums + to * D + dt * 16 + 4 * g) = o[nq][dt];
    if (g == 0) *(float2*)(a.stats + to * 2) = make_float2(m[nq], sum);
  }
}

// NS 0: 16 * NQ rows whose keys the waves share out; else 64 * NQ rows, 16 * NQ for a wave.
template <int E, int D, int NQ, int NS, bool OWN>
__device__ inline void prefix_block(const PrefixArgs& a, unsigned char* stages, const PartRows& w, int kvh) {
  if constexpr (NS > 0) prefix_part_rows<E, D, NQ, NS, OWN>(a, stages, w, kvh);
  else prefix_part<E, D, NQ, OWN>(a, stages, w, kvh);
}

// NQS, NSS: of blocks with shared keys, the tiles of 16 rows (of a wave, if NSS > 0) and the steps of a ring that the waves share (0: each has its own);
// NQO, NSO: of blocks with own keys.
template <int E, int D, int NQS, int NSS, int NQO, int NSO, int OCC>
__global__ __launch_bounds__(PA_WAVES * 64, OCC) void prefix_attention_kernel(PrefixArgs a) {
  constexpr int STEPS = (NSS > 0 && NSO > 0) ? (NSS > NSO ? NSS : NSO) : NSS > PA_WAVES ? NSS : PA_WAVES;
  __shared__ __attribute__((aligned(1024))) unsigned char stages[STEPS * PrefixLane<E, D>::STAGE];
  constexpr int ROWS = 16 * NQS * (NSS > 0 ? PA_WAVES : 1), OWN = 16 * NQO * (NSO > 0 ? PA_WAVES : 1);
  const int kvh = blockIdx.x % a.n_kv, group = a.n_heads / a.n_kv;
  int b = blockIdx.x / a.n_kv;
  PartRows w;
  if (b < a.shared_blocks) {
    // which group's rows: a lane counts the blocks of one group, 64 groups at a time
    const int lane = threadIdx.x & 63;
    // (a group's blocks of rows one behind the other, so that those that are not there come last: between the others they would take places
    // of the first turn in which blocks are handed to the CUs)
    int rb = b / a.shared_parts;
    w.part = b % a.shared_parts;
    bool found = false;
    for (int g0 = 0; g0 < a.groups && !found; g0 += 64) {
      const int i = g0 + lane;
      int keys = 0, token0 = 0, end = 0, r0 = 0;
      if (i < a.groups) {
        keys = a.group_keys[i];
        r0 = token0 = a.group_starts[i];
        end = a.group_starts[i + 1];
        if (!a.single) {
          token0 = a.cu_seqlens[r0];
          end = a.cu_seqlens[end];
        }
      }
      const int blocks = keys > 0 ? ((end - token0) * group + ROWS - 1) / ROWS : 0;
      int upto = blocks;
      if (a.groups > 1) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int v = __shfl_up(upto, d, 64);
          if (lane >= d) upto += v;
        }
      }
      const unsigned long long hit = __ballot(rb < upto);
      if (hit != 0) {
        const int src = (int)__builtin_ctzll(hit);
        w.row0 = (rb - __builtin_amdgcn_readlane(upto - blocks, src)) * ROWS;
        w.end = min(__builtin_amdgcn_readlane(keys, src), a.table_width << a.page_shift);
        w.token0 = __builtin_amdgcn_readlane(token0, src);
        w.rows = min(ROWS, (__builtin_amdgcn_readlane(end, src) - w.token0) * group - w.row0);
        w.table = a.block_tables + (size_t)__builtin_amdgcn_readlane(r0, src) * a.table_width;
        found = true;
      }
      rb -= __builtin_amdgcn_readlane(upto, 63);
    }
    if (!found) return;
    w.first = w.part * a.shared_steps * 32;
    if (w.first >= w.end) return;
    w.end = min(w.end, w.first + a.shared_steps * 32);
    w.limit0 = 0x7fffffff;
    prefix_block<E, D, NQS, NSS, false>(a, stages, w, kvh);
    return;
  }
  b -= a.shared_blocks;
  const int r = (b / a.own_rows) % a.requests, part = b / a.own_rows / a.requests;
  const int t0 = a.single ? r : a.cu_seqlens[r], tokens = a.single ? 1 : a.cu_seqlens[r + 1] - t0;
  const int ctx = min(a.context_lens[r], a.table_width << a.page_shift), shared = a.shared_keys[r];
  w.token0 = t0;
  w.row0 = (b % a.own_rows) * OWN;
  w.rows = min(OWN, tokens * group - w.row0);
  w.first = part == 0 ? shared : (shared & ~15) + part * a.own_steps * 32;
  w.end = min(ctx, (shared & ~15) + (part + 1) * a.own_steps * 32);
  if (w.rows <= 0 || w.first >= w.end) return;
  w.limit0 = ctx - tokens;
  w.table = a.block_tables + (size_t)r * a.table_width;
  w.part = a.shared_parts + part;
  prefix_block<E, D, NQO, NSO, true>(a, stages, w, kvh);
}

// out[token, head, :] from a row's parts, in a fixed order: those of its request's shared keys, then those of its own.  W waves a row, D / 4 lanes a
// part, 16 bytes a lane; every wave works the weights out for itself (its lane s holds the statistics of parts s and 64 + s).  Bound by trips to
// memory: which parts exist is asked beside all places' statistics (what stands in a place without a part is not used).
template <int E, int D, int W>
__global__ __launch_bounds__(256) void prefix_join_kernel(const float* __restrict__ sums, const float* __restrict__ stats,
                                                          const int* __restrict__ token_req, const int* __restrict__ context_lens,
                                                          const int* __restrict__ shared_keys, void* __restrict__ out, const float* __restrict__ sink,
                                                          int rows, int heads, int requests, int shared_parts, int parts, int shared_steps, int own_steps,
                                                          int single) {
  constexpr int LANES = D / 4, GROUPS = W * 64 / LANES, AHEAD = 4;      // parts at a time, and how many times that is asked for at once
  __shared__ __attribute__((aligned(16))) float red[W > 1 ? W * D : 4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int row = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  if (row >= rows) return;
  const float* s = stats + (size_t)row * parts * 2;
  float2 st[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
  if (lane < parts) st[0] = *(const float2*)(s + lane * 2);
  if (64 + lane < parts) st[1] = *(const float2*)(s + (64 + lane) * 2);
  const float sunk = sink != nullptr ? sink[row % heads] : 0.f;
  const int r = single ? row / heads : token_req[row / heads];
  if (r < 0 || r >= requests) return;      // (a row behind the last request: left as it was)
  const int shared = shared_keys[r], ctx = context_lens[r];
  const int n_shared = min(((shared + 31) / 32 + shared_steps - 1) / shared_steps, shared_parts);
  const int n = n_shared + min(((ctx - (shared & ~15) + 31) / 32 + own_steps - 1) / own_steps, parts - shared_parts);
  // (part i of the n stands in place i, from n_shared on in place shared_parts + i - n_shared)
  const int gap = shared_parts - n_shared;
  const int mine = (W == 1 ? 0 : wave * (64 / LANES)) + lane / LANES;
  const float* o = sums + (size_t)row * parts * D + (lane % LANES) * 4;
  float4 val[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = mine + k * GROUPS;
    val[k] = i < n ? *(const float4*)(o + (size_t)(i < n_shared ? i : i + gap) * D) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int place = k * 64 + lane;
    if (place >= n + gap || (place >= n_shared && place < shared_parts)) st[k] = make_float2(-INFINITY, 0.f);
    top = fmaxf(top, st[k].x);
  }
  top = wave_max(top);
  const float use = top == -INFINITY ? 0.f : top;
  const float f[2] = {__builtin_amdgcn_exp2f(st[0].x - use), __builtin_amdgcn_exp2f(st[1].x - use)};
  float total = wave_sum(fmaf(f[0], st[0].y, f[1] * st[1].y));
  if (sink != nullptr) total += __builtin_amdgcn_exp2f(fmaf(sunk, 1.4426950408889634f, -use));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += AHEAD * GROUPS) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + mine + k * GROUPS, place = i < n_shared ? i : i + gap;
      const float lo = __shfl(f[0], place & 63, 64), hi = __shfl(f[1], place & 63, 64);
      const float w = i < n ? (place < 64 ? lo : hi) : 0.f;
      acc.x = fmaf(w, val[k].x, acc.x);
      acc.y = fmaf(w, val[k].y, acc.y);
      acc.z = fmaf(w, val[k].z, acc.z);
      acc.w = fmaf(w, val[k].w, acc.w);
    }
    if (i0 + AHEAD * GROUPS < n) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int i = i0 + AHEAD * GROUPS + mine + k * GROUPS;
        val[k] = i < n ? *(const float4*)(o + (size_t)(i < n_shared ? i : i + gap) * D) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
#pragma unroll
  for (int d = LANES; d < 64; d <<= 1) {
    acc.x += __shfl_xor(acc.x, d, 64);
    acc.y += __shfl_xor(acc.y, d, 64);
    acc.z += __shfl_xor(acc.z, d, 64);
    acc.w += __shfl_xor(acc.w, d, 64);
  }
  if constexpr (W > 1) {
    if (lane < LANES) *(float4*)(red + wave * D + lane * 4) = acc;
    __syncthreads();
    if (wave != 0) return;
    acc = *(const float4*)(red + (lane % LANES) * 4);
#pragma unroll
    for (int v = 1; v < W; ++v) {
      const float4 more = *(const float4*)(red + v * D + (lane % LANES) * 4);
      acc.x += more.x;
      acc.y += more.y;
      acc.z += more.z;
      acc.w += more.w;
    }
  }
  if (lane >= LANES) return;
  const float inv = 1.0f / total;
  const size_t to = (size_t)row * D + lane * 4;
  if constexpr (E == 2) from_float4((bf16_t*)out + to, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  else from_float4((float*)out + to, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// (two blocks a CU where LDS holds two, but for float32 blocks of 128 rows, whose registers do not)
template <int E, int D, int NQS, int NSS, int NQO, int NSO>
static int prefix_launch(const PrefixArgs& a, int blocks, hipStream_t s) {
  prefix_attention_kernel<E, D, NQS, NSS, NQO, NSO, E == 2 || (NQS == 1 && NSO > 0) ? 2 : 1><<<blocks, PA_WAVES * 64, 0, s>>>(a);
  return 0;
}

template <int E, int D>
static int prefix_sizes(const PrefixArgs& a, int blocks, int rows_shared, int rows_own, hipStream_t s) {
  constexpr int NS = E == 2 ? 4 : 2;
  if (rows_own == 16) {
    if (rows_shared == 16) return prefix_launch<E, D, 1, 0, 1, 0>(a, blocks, s);
    if (rows_shared == 64) return prefix_launch<E, D, 1, NS, 1, 0>(a, blocks, s);
    if (rows_shared == 128) return prefix_launch<E, D, 2, NS, 1, 0>(a, blocks, s);
  } else if (rows_own == 64) {
    if (rows_shared == 64) return prefix_launch<E, D, 1, NS, 1, NS>(a, blocks, s);
    if (rows_shared == 128) return prefix_launch<E, D, 2, NS, 1, NS>(a, blocks, s);
  } else if (rows_own == 128) {
    if (rows_shared == 128) return prefix_launch<E, D, 2, NS, 2, NS>(a, blocks, s);
  }
  tp_set_error("prefix_attention: no kernel for blocks of %d and %d rows", rows_shared, rows_own);
  return 1;
}

// q [n, heads, dim] over pages of keys and transposed values (elements of dt), each request's context by its block table; out [n, heads * dim].
// groups of requests share their first keys (group_starts [groups + 1], group_keys [groups], shared_keys [requests]: see PrefixArgs); every query
// lies behind its request's shared keys; rows of q whose token_req is no request are left as they were.  shared_blocks: at least as many blocks of rows_shared rows (16, 64 or 128) as all groups have; rows_own 16, 64 or 128.  Parts of
// shared_steps / own_steps steps of 32 keys, as many as there are at most.  scratch: n * heads * (shared_parts + own_parts) * (dim + 2) + 2 floats, aligned to 16 bytes.
// sizes: element type, table width, n, requests, groups, heads, key heads, dim, page size, the most tokens of a request, rows_shared, rows_own,
// shared_blocks, shared_steps, shared_parts, own_steps, own_parts.
extern "C" int tp_prefix_attention(const void* q, const void* k_cache, const void* v_cache, const int* block_tables, const int* cu_seqlens,
                                   const int* context_lens, const int* token_req, const int* group_starts, const int* group_keys,
                                   const int* shared_keys, void* out, float* scratch, const float* sink, const int* sizes, float scale, float softcap,
                                   hipStream_t s) {
  const int dt = sizes[0], table_width = sizes[1], n = sizes[2], requests = sizes[3], groups = sizes[4], heads = sizes[5], kv_heads = sizes[6],
            dim = sizes[7], page_size = sizes[8], max_q_len = sizes[9], rows_shared = sizes[10], rows_own = sizes[11], shared_blocks = sizes[12],
            shared_steps = sizes[13], shared_parts = sizes[14], own_steps = sizes[15], own_parts = sizes[16];
  if (n <= 0 || requests <= 0) return 0;
  TP_REQUIRE(dt == TP_BF16 || dt == TP_F32, "prefix_attention: unsupported element type");
  TP_REQUIRE(dim == 32 || dim == 64 || dim == 128, "prefix_attention: heads of 32, 64 or 128 elements");
  TP_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "prefix_attention: pages of a power of two from 16 on");
  TP_REQUIRE(scale > 0.f, "prefix_attention: the scale must be positive");
  TP_REQUIRE(kv_heads > 0 && heads % kv_heads == 0 && groups > 0 && max_q_len > 0, "prefix_attention: bad sizes");
  TP_REQUIRE(shared_steps > 0 && own_steps > 0 && shared_parts > 0 && own_parts > 0 && shared_parts + own_parts <= PA_MAX_PARTS && shared_blocks > 0 && rows_own > 0,
             "prefix_attention: bad parts");
  PrefixArgs a = {};
  a.q = q;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.block_tables = block_tables;
  a.cu_seqlens = cu_seqlens;
  a.context_lens = context_lens;
  a.group_starts = group_starts;
  a.group_keys = group_keys;
  a.shared_keys = shared_keys;
  a.parts = shared_parts + own_parts;
  a.stats = scratch;
  a.sums = scratch + ((size_t)n * heads * a.parts * 2 + 3) / 4 * 4;
  a.table_width = table_width;
  a.page_shift = __builtin_ctz(page_size);
  a.n_heads = heads;
  a.n_kv = kv_heads;
  a.groups = groups;
  a.requests = requests;
  a.single = n == requests && max_q_len == 1;
  a.shared_parts = shared_parts;
  a.own_rows = (int)(((long)max_q_len * (heads / kv_heads) + rows_own - 1) / rows_own);
  a.shared_steps = shared_steps;
  a.own_steps = own_steps;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.cap_log2 = softcap * 1.4426950408889634f;
  a.cap_in = softcap > 0.f ? (dt == TP_BF16 ? 2.0f * a.scale_log2 : scale) / softcap : 0.f;
  const long of_shared = (long)shared_blocks * shared_parts, blocks = (of_shared + (long)a.own_rows * requests * own_parts) * kv_heads;
  TP_REQUIRE(blocks < (1L << 31), "prefix_attention: too many blocks");
  a.shared_blocks = (int)of_shared;
  int rc = 1;
  if (dt == TP_BF16)
    rc = dim == 32 ? prefix_sizes<2, 32>(a, (int)blocks, rows_shared, rows_own, s) : dim == 64 ? prefix_sizes<2, 64>(a, (int)blocks, rows_shared, rows_own, s)
                                                                                            : prefix_sizes<2, 128>(a, (int)blocks, rows_shared, rows_own, s);
  else
    rc = dim == 32 ? prefix_sizes<4, 32>(a, (int)blocks, rows_shared, rows_own, s) : dim == 64 ? prefix_sizes<4, 64>(a, (int)blocks, rows_shared, rows_own, s)
                                                                                            : prefix_sizes<4, 128>(a, (int)blocks, rows_shared, rows_own, s);
  if (rc != 0) return rc;
  TP_CHECK_LAUNCH("prefix_attention");
  // (a row of more than eight parts has four waves while the rows are not many: 1,024 rows of 32 parts 6.2 us, with one wave each 13.1)
  const int rows = n * heads;
  const bool wide = a.parts > 8 && rows <= 4096;
#define PA_JOIN_W(E, D, W) prefix_join_kernel<E, D, W><<<W == 1 ? (rows + 3) / 4 : rows, 256, 0, s>>>(a.sums, a.stats, token_req, context_lens, shared_keys, out, sink, \
                                                                     rows, heads, requests, shared_parts, a.parts, shared_steps, own_steps, a.single)
#define PA_JOIN(E, D) (wide ? PA_JOIN_W(E, D, 4) : PA_JOIN_W(E, D, 1))
  if (dt == TP_BF16) {
    if (dim == 32) PA_JOIN(2, 32);
    else if (dim == 64) PA_JOIN(2, 64);
    else PA_JOIN(2, 128);
  } else {
    if (dim == 32) PA_JOIN(4, 32);
    else if (dim == 64) PA_JOIN(4, 64);
    else PA_JOIN(4, 128);
  }
#undef PA_JOIN_W
#undef PA_JOIN
  TP_CHECK_LAUNCH("prefix_attention (join)");
  return 0;
}
