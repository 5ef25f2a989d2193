// Attention of a step whose requests begin with the same keys, the shared pages read once for a group of requests instead of
// once for each of them.
//
// A group is a run of neighbouring requests of the batch whose block tables begin with the same pages: its first P keys.  Every
// query of the group sees all of them, so for one key head all (token, head) pairs of the group are the rows of ONE product with
// those keys, no mask between them; behind them each request has keys of its own, of which its tokens see those up to themselves.
// A block takes one key head, 16 * NQ rows and one part of the keys (a group's shared ones or a request's own) and leaves the
// rows' partial results: O (unnormalised), maximum and sum.  A second kernel joins a row's parts in ascending order:
//   m = max m_s,   out = sum_s 2^(m_s - m) O_s / (sum_s 2^(m_s - m) l_s + 2^(sink - m)).
//
// The step of 32 keys is computed transposed, so that no operand is transposed in LDS (values are cached transposed):
//   S^T[key, row] = K[key, :] . Q[row, :]^T      O^T[d, row] += V^T[d, keys] . P^T[keys, row]
// with v_mfma_f32_16x16x32_bf16, float32 caches with v_mfma_f32_16x16x4_f32.  A 16x16 result gives lane (c = lane % 16, g = lane / 16)
// the rows 4 g + r of column c.  bfloat16: the two key tiles of a step take their keys in the order 8 (i / 4) + 4 t + i % 4, so a lane
// ends up with the eight CONSECUTIVE keys 8 g .. of its row, the operand of the next product.  float32: the order is 16 t + i, a lane has
// the keys 16 t + 4 g + r, and the product with register r of tile t takes exactly these as its four k.  A fragment is 16 bytes a lane either way.
// Statistics and sums are float32; the probabilities of bfloat16 caches are rounded to bfloat16 for the second product (the largest
// is 1, so their errors, up to 2^-9 of each, average out in the sum, which is rounded to bfloat16 anyway).
//
// Each of a block's four waves takes a run of the part's steps and has a ring of NB steps in LDS for itself, filled by direct
// global-to-LDS loads (whole kilobytes) and emptied without a barrier: a step's keys go on their way as soon as the fragments of the
// keys they replace are in registers, its values likewise.  So every key and value passes a CU's LDS once for up to 64 rows.
#include <math.h>

#include "common.h"

typedef __bf16 pa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x2 __attribute__((ext_vector_type(2)));
typedef float pa_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int pa_u32x4 __attribute__((ext_vector_type(4)));

#define PA_WAVES 4
#define PA_MAX_PARTS 64     // a row's parts: the joining kernel holds one part's statistics a lane
#define PA_GPTR(p) ((const __attribute__((address_space(1))) void*)(p))
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
  int shared_blocks;         // blocks (of rows and parts) that take shared keys, a key head each; the own keys' come behind them
  int shared_rows;           // blocks of rows among them (an upper bound: those beyond the last group end at once)
  int own_rows;              // blocks of rows of a request
  int shared_steps, own_steps;   // steps of 32 keys a part has
  int shared_parts, parts;   // a row's places for parts: those of the shared keys, all
  float scale_log2;          // scale * log2(e)
  float cap_log2, cap_in;    // scores under a cap: cap * log2(e), and what turns q . k into 2 log2(e) score / cap; 0: no cap
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

// E: bytes of an element.  NB: steps of a wave's ring.  NT: keys and values are read by one block only.
template <int E, int D, int NQ, int NB, bool NT>
__device__ inline void prefix_part(const PrefixArgs& a, unsigned char* stages, const PartRows& w, int kvh) {
  constexpr int CH = D * E / 16;                              // 16-byte chunks of a key
  constexpr int SH = CH >= 16 ? 0 : CH == 8 ? 1 : 2;
  constexpr int KF = CH / 4;                                  // a lane's chunks of a key (or of a row of q)
  constexpr int DT = D / 16;
  constexpr int VF = E / 2;                                   // a lane's chunks of an element's 32 keys
  constexpr int KI = D * E / 32, VI = KI, STAGE = (KI + VI) * 1024;
  constexpr int VD = 64 / E;                                  // elements of a kilobyte of values (of half a step's keys): 32 or 16
  static_assert(E == 2 || E == 4, "element size");
  static_assert((NB == 1 || NB == 2) && 2 * VI + KI <= 63, "the waits below");
  static_assert(NB * STAGE >= (D * 17 + 32) * 4, "room for the sums of a tile");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int group = a.n_heads / a.n_kv;
  const int psh = a.page_shift, ps = 1 << psh, pmask = ps - 1;

  // q: this lane's rows of the tiles, and the last key each of them sees
  pa_u32x4 qf[NQ][KF];
  int limit[NQ];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    const int pair = w.row0 + min(nq * 16 + c, w.rows - 1);
    const int token = pair / group, head = kvh * group + pair % group;
    const unsigned char* row = (const unsigned char*)a.q + ((size_t)(w.token0 + token) * a.n_heads + head) * (D * E) + g * 16;
#pragma unroll
    for (int i = 0; i < KF; ++i) qf[nq][i] = *(const pa_u32x4*)(row + i * 64);
    limit[nq] = w.limit0 == 0x7fffffff ? w.limit0 : w.limit0 + token;
  }

  // this lane's place in each load of a step: of the keys the row's chunk, of the values the element's chunk
  unsigned koff[KI];
#pragma unroll
  for (int t = 0; t < KI; ++t) {
    const int row = (64 * t + lane) / CH, pc = (64 * t + lane) % CH;
    const int i = E == 2 ? 4 * (row >> 3) + (row & 3) : row & 15;       // its place in its tile
    koff[t] = (unsigned)((row & 15) * (D * E) + ((pc - (i >> SH) + CH) % CH) * 16);
  }
  const unsigned voff = (unsigned)((lane % VD) * (ps * E) + (lane / VD) * 16);
  const size_t page_bytes = (size_t)a.n_kv * D * ps * E;
  const unsigned char* kbase = (const unsigned char*)a.k_cache + (size_t)kvh * ps * D * E;
  const unsigned char* vbase = (const unsigned char*)a.v_cache + (size_t)kvh * ps * D * E;
  unsigned char* ring = stages + wave * (NB * STAGE);
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) const unsigned char*)ring;
  unsigned kaddr[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) kaddr[t] = (E == 2 ? 8 * (c >> 2) + 4 * t + (c & 3) : 16 * t + c) * (CH * 16);
  unsigned kchunk[KF];
#pragma unroll
  for (int i = 0; i < KF; ++i) kchunk[i] = ((i * 4 + g + (c >> SH)) % CH) * 16;
  // (bfloat16: the keys 8 g .. lie in half g / 2, chunk g % 2; float32: the keys 16 t + 4 g .. in half t, chunk g)
  const unsigned vaddr = KI * 1024 + (E == 2 ? (g >> 1) * 1024 + (g & 1) * 512 : g * 256) + c * 16;

  // (block tables through the constant address space: uniform loads from it are scalar loads)
  const __attribute__((address_space(4))) int* table = (const __attribute__((address_space(4))) int*)(uintptr_t)w.table;
  const int base16 = w.first & ~15;                           // (a step's halves of 16 keys lie in one page each)
  const int steps = (w.end - base16 + 31) >> 5, run = (steps + PA_WAVES - 1) / PA_WAVES;
  const int w0 = wave * run, n = max(0, min(steps - w0, run));
  const int last16 = (w.end - 1) & ~15;
  int pp0 = 0, pp1 = 0;
  auto pages_of = [&](int i) {
    const int j0 = base16 + (w0 + i) * 32;
    pp0 = table[j0 >> psh];
    pp1 = table[min(j0 + 16, last16) >> psh];
  };
  auto issue_keys = [&](int i, int st) __attribute__((always_inline)) {
    const int j0 = base16 + (w0 + i) * 32;
    const unsigned char* half[2] = {kbase + (size_t)(unsigned)pp0 * page_bytes + (size_t)(j0 & pmask) * (D * E),
                                    kbase + (size_t)(unsigned)pp1 * page_bytes + (size_t)(min(j0 + 16, last16) & pmask) * (D * E)};
#pragma unroll
    for (int t = 0; t < KI; ++t)
      __builtin_amdgcn_global_load_lds(PA_GPTR(half[t >= KI / 2] + koff[t]), PA_LPTR(ring + st * STAGE + t * 1024), 16, 0, NT ? 2 : 0);
  };
  auto issue_values = [&](int i, int st) __attribute__((always_inline)) {
    const int j0 = base16 + (w0 + i) * 32;
    const unsigned char* half[2] = {vbase + (size_t)(unsigned)pp0 * page_bytes + (j0 & pmask) * E,
                                    vbase + (size_t)(unsigned)pp1 * page_bytes + (min(j0 + 16, last16) & pmask) * E};
#pragma unroll
    for (int t = 0; t < VI; ++t)
      __builtin_amdgcn_global_load_lds(PA_GPTR(half[t & 1] + (size_t)(t >> 1) * VD * ps * E + voff), PA_LPTR(ring + st * STAGE + (KI + t) * 1024), 16, 0,
                                       NT ? 2 : 0);
  };
#pragma unroll
  for (int i = 0; i < NB; ++i)
    if (i < n) {
      pages_of(i);
      issue_keys(i, i);
      issue_values(i, i);
    }
  if (NB < n) pages_of(NB);

  float m[NQ], l[NQ];
  pa_f32x4 o[NQ][DT];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq) {
    m[nq] = -INFINITY;
    l[nq] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[nq][dt] = (pa_f32x4){0.f, 0.f, 0.f, 0.f};
  }
  int st = 0;
  for (int i = 0; i < n; ++i) {
    const unsigned base = lds0 + st * STAGE;
    const bool behind = NB > 1 && i + 1 < n;      // (a whole step on its way behind this one)
    const bool more = i + NB < n;
    if (behind) PA_WAIT_VM(VI + KI + VI);
    else PA_WAIT_VM(VI);
    const int j0 = base16 + (w0 + i) * 32;
    pa_u32x4 kk[2][KF];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int f = 0; f < KF; ++f) kk[t][f] = pa_lds(base + kaddr[t] + kchunk[f]);
    PA_WAIT_LDS();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int f = 0; f < KF; ++f) asm volatile("" : "+v"(kk[t][f]));
    if (more) issue_keys(i + NB, st);
    pa_f32x4 s[NQ][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        s[nq][t] = (pa_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < KF; ++f) {
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
    // (scores outside the part or above the row's limit: not in the sums; `whole`: none of this step's)
    const bool whole = j0 >= w.first && j0 + 32 <= w.end && w.limit0 >= j0 + 31;
    pa_u32x4 pf[NQ][E == 2 ? 1 : 2];
    float alpha[NQ];
    bool moved[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      float v[8], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = s[nq][j >> 2][j & 3] * a.scale_log2;
      if (a.cap_in > 0.f) {
        // cap * tanh(x) with tanh(x) = 1 - 2 / (2^(2 x log2 e) + 1); both limits come out right (2^large is infinite, its reciprocal 0)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = fmaf(-2.0f * a.cap_log2, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[nq][j >> 2][j & 3] * a.cap_in) + 1.0f), a.cap_log2);
      }
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = j0 + (E == 2 ? 8 * g + j : 16 * (j >> 2) + 4 * g + (j & 3));
          if (key < w.first || key >= w.end || key > limit[nq]) v[j] = -INFINITY;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, v[j]);
      const float m_new = fmaxf(m[nq], pa_column_max(top));
      const float m_use = m_new == -INFINITY ? 0.f : m_new;   // (a row that has seen no key yet)
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __builtin_amdgcn_exp2f(v[j] - m_use);
        sum += v[j];
      }
      moved[nq] = __builtin_amdgcn_ballot_w64(m_new != m[nq]) != 0;
      alpha[nq] = 1.f;
      if (moved[nq]) {
        alpha[nq] = __builtin_amdgcn_exp2f(m[nq] - m_use);
        m[nq] = m_new;
      }
      l[nq] = fmaf(l[nq], alpha[nq], sum);     // (this lane's keys; the lanes of a column are added at the end)
      if constexpr (E == 2) {
        pf[nq][0] = (pa_u32x4){pa_pack(v[0], v[1]), pa_pack(v[2], v[3]), pa_pack(v[4], v[5]), pa_pack(v[6], v[7])};
      } else {
        pf[nq][0] = __builtin_bit_cast(pa_u32x4, (pa_f32x4){v[0], v[1], v[2], v[3]});
        pf[nq][1] = __builtin_bit_cast(pa_u32x4, (pa_f32x4){v[4], v[5], v[6], v[7]});
      }
    }
    if (more && behind) PA_WAIT_VM(KI + KI + VI);
    else if (more) PA_WAIT_VM(KI);
    else if (behind) PA_WAIT_VM(KI + VI);
    else PA_WAIT_VM(0);
    pa_u32x4 vv[DT][VF];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int t = 0; t < VF; ++t)
        vv[dt][t] = pa_lds(base + vaddr + (E == 2 ? (dt >> 1) * 2048 + (dt & 1) * 256 : dt * 2048 + t * 1024));
    PA_WAIT_LDS();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int t = 0; t < VF; ++t) asm volatile("" : "+v"(vv[dt][t]));
    if (more) {
      issue_values(i + NB, st);
      if (i + NB + 1 < n) pages_of(i + NB + 1);
    }
    if (j0 + 32 > w.end) {
      // places behind the last key hold whatever an earlier owner of the page left there; their probabilities are 0, but 0 * NaN
      // and 0 * Inf are not, so they are cleared
#pragma unroll
      for (int t = 0; t < VF; ++t) {
        const int left = w.end - (j0 + (E == 2 ? 8 * g : 16 * t + 4 * g));
        pa_u32x4 keep;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          keep[e] = E == 2 ? (2 * e < left ? 0x0000ffffu : 0u) | (2 * e + 1 < left ? 0xffff0000u : 0u) : e < left ? 0xffffffffu : 0u;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vv[dt][t] &= keep;
      }
    }
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      if (moved[nq]) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[nq][dt][r] *= alpha[nq];
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        if constexpr (E == 2) {
          o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8, vv[dt][0]), __builtin_bit_cast(pa_bf16x8, pf[nq][0]),
                                                              o[nq][dt], 0, 0, 0);
        } else {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const pa_f32x4 vv4 = __builtin_bit_cast(pa_f32x4, vv[dt][t]), p4 = __builtin_bit_cast(pa_f32x4, pf[nq][t]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv4[e], p4[e], o[nq][dt], 0, 0, 0);
          }
        }
      }
    }
    st = st + 1 == NB ? 0 : st + 1;
  }

  // The waves' sums, added in their order through LDS, a tile of 16 rows at a time (rows a bank apart: 17 floats an element)
  float* red = (float*)stages;
  float* stat = red + PA_WAVES * D * 17;
  for (int nq = 0; nq < NQ; ++nq) {
    __syncthreads();     // (every ring is empty; the tile before is read)
#pragma unroll
    for (int k = 0; k < NQ; ++k)
      if (k == nq) {     // (constant places: the sums stay in registers)
        float sum = l[k];
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g == 0) {
          stat[wave * 32 + c] = m[k];
          stat[wave * 32 + 16 + c] = sum;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int r = 0; r < 4; ++r) red[(wave * D + dt * 16 + 4 * g + r) * 17 + c] = o[k][dt][r];
      }
    __syncthreads();
    const int rows = min(16, w.rows - nq * 16);
    for (int e = threadIdx.x; e < D * rows; e += PA_WAVES * 64) {
      const int d = e % D, col = e / D;
      float top = stat[col];
#pragma unroll
      for (int v = 1; v < PA_WAVES; ++v) top = fmaxf(top, stat[v * 32 + col]);
      const float use = top == -INFINITY ? 0.f : top;
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int v = 0; v < PA_WAVES; ++v) {
        const float f = __builtin_amdgcn_exp2f(stat[v * 32 + col] - use);
        acc = fmaf(f, red[(v * D + d) * 17 + col], acc);
        sum = fmaf(f, stat[v * 32 + 16 + col], sum);
      }
      const int pair = w.row0 + nq * 16 + col;
      const size_t at = ((size_t)(w.token0 + pair / group) * a.n_heads + kvh * group + pair % group) * a.parts + w.part;
      a.sums[at * D + d] = acc;
      if (d == 0) *(float2*)(a.stats + at * 2) = make_float2(top, sum);
    }
  }
}

// NQS, NQO: tiles of 16 rows of a block with shared and with own keys.
template <int E, int D, int NQS, int NQO, int NB, int OCC>
__global__ __launch_bounds__(PA_WAVES * 64, OCC) void prefix_attention_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char stages[PA_WAVES * NB * D * 64 * E];
  const int kvh = blockIdx.x % a.n_kv, group = a.n_heads / a.n_kv;
  int b = blockIdx.x / a.n_kv;
  PartRows w;
  if (b < a.shared_blocks) {
    // which group's rows: a lane counts the blocks of one group, 64 groups at a time
    const int lane = threadIdx.x & 63;
    int rb = b % a.shared_rows;
    w.part = b / a.shared_rows;
    bool found = false;
    for (int g0 = 0; g0 < a.groups && !found; g0 += 64) {
      const int i = g0 + lane;
      int keys = 0, tokens = 0, token0 = 0, r0 = 0;
      if (i < a.groups) {
        r0 = a.group_starts[i];
        keys = min(a.group_keys[i], a.context_lens[r0]);     // (pages behind a request's context need not exist)
        token0 = a.cu_seqlens[r0];
        tokens = a.cu_seqlens[a.group_starts[i + 1]] - token0;
      }
      const int blocks = keys > 0 ? (tokens * group + 16 * NQS - 1) / (16 * NQS) : 0;
      int upto = blocks;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(upto, d, 64);
        if (lane >= d) upto += v;
      }
      const unsigned long long hit = __ballot(rb < upto);
      if (hit != 0) {
        const int src = (int)__builtin_ctzll(hit);
        w.row0 = (rb - __builtin_amdgcn_readlane(upto - blocks, src)) * 16 * NQS;
        w.end = __builtin_amdgcn_readlane(keys, src);
        w.token0 = __builtin_amdgcn_readlane(token0, src);
        w.rows = min(16 * NQS, __builtin_amdgcn_readlane(tokens, src) * group - w.row0);
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
    prefix_part<E, D, NQS, NB, false>(a, stages, w, kvh);
    return;
  }
  b -= a.shared_blocks;
  const int r = (b / a.own_rows) % a.requests, part = b / a.own_rows / a.requests;
  const int t0 = a.cu_seqlens[r], tokens = a.cu_seqlens[r + 1] - t0;
  const int ctx = a.context_lens[r], shared = a.shared_keys[r];
  w.token0 = t0;
  w.row0 = (b % a.own_rows) * 16 * NQO;
  w.rows = min(16 * NQO, tokens * group - w.row0);
  w.first = part == 0 ? shared : (shared & ~15) + part * a.own_steps * 32;
  w.end = min(ctx, (shared & ~15) + (part + 1) * a.own_steps * 32);
  if (w.rows <= 0 || w.first >= w.end) return;
  w.limit0 = ctx - tokens;
  w.table = a.block_tables + (size_t)r * a.table_width;
  w.part = a.shared_parts + part;
  prefix_part<E, D, NQO, NB, true>(a, stages, w, kvh);
}

// out[token, head, :] from a row's parts, in ascending order: those of its request's shared keys, then those of its own.  A wave a row; its lane
// s holds part s's statistics.  Bound by one trip to memory: statistics and the first parts' sums are requested together.
template <int E, int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(const float* __restrict__ sums, const float* __restrict__ stats,
                                                          const int* __restrict__ token_req, const int* __restrict__ context_lens,
                                                          const int* __restrict__ shared_keys, void* __restrict__ out, const float* __restrict__ sink,
                                                          int rows, int heads, int shared_parts, int parts, int shared_steps, int own_steps) {
  const int row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const int token = row / heads, r = token_req[token];
  const int shared = shared_keys[r], ctx = context_lens[r];
  const int n_shared = min(((shared + 31) / 32 + shared_steps - 1) / shared_steps, shared_parts);
  const int n_own = min(((ctx - (shared & ~15) + 31) / 32 + own_steps - 1) / own_steps, parts - shared_parts);
  const int n = n_shared + n_own;     // (lane i < n_shared: part i, else part shared_parts + i - n_shared)
  const int part = lane < n_shared ? lane : shared_parts + lane - n_shared;
  float2 st = make_float2(-INFINITY, 0.f);
  if (lane < n) st = *(const float2*)(stats + ((size_t)row * parts + part) * 2);
  const float top = wave_max(st.x), use = top == -INFINITY ? 0.f : top;
  const float f = __builtin_amdgcn_exp2f(st.x - use);
  float total = wave_sum(f * st.y);
  if (sink != nullptr) total += __builtin_amdgcn_exp2f(fmaf(sink[row % heads], 1.4426950408889634f, -use));
  constexpr int P = D >= 128 ? 2 : 1;     // elements a lane
  float acc[P] = {};
  const bool there = lane * P < D;
  if (!there) return;
  for (int i = 0; i < n; ++i) {
    const float fi = lane_value(f, i);
    const float* o = sums + ((size_t)row * parts + (i < n_shared ? i : shared_parts + i - n_shared)) * D + lane * P;
#pragma unroll
    for (int e = 0; e < P; ++e) acc[e] = fmaf(fi, o[e], acc[e]);
  }
  const float inv = 1.0f / total;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    if constexpr (E == 2) ((bf16_t*)out)[(size_t)row * D + lane * P + e] = float_to_bf16(acc[e] * inv);
    else ((float*)out)[(size_t)row * D + lane * P + e] = acc[e] * inv;
  }
}

template <int E, int D, int NQS, int NQO, int NB, int OCC>
static void prefix_launch(const PrefixArgs& a, int blocks, hipStream_t s) {
  prefix_attention_kernel<E, D, NQS, NQO, NB, OCC><<<blocks, PA_WAVES * 64, 0, s>>>(a);
}

template <int E, int D>
static int prefix_sizes(const PrefixArgs& a, int blocks, int tiles_shared, int tiles_own, hipStream_t s) {
  constexpr int OCC = E == 2 ? 2 : 1;
  if (tiles_shared == 1 && tiles_own == 1) prefix_launch<E, D, 1, 1, 1, OCC>(a, blocks, s);
  else if (tiles_shared == 2 && tiles_own == 1) prefix_launch<E, D, 2, 1, 1, OCC>(a, blocks, s);
  else if (tiles_shared == 2 && tiles_own == 2) prefix_launch<E, D, 2, 2, 1, OCC>(a, blocks, s);
  else {
    tp_set_error("prefix_attention: no kernel for %d and %d tiles", tiles_shared, tiles_own);
    return 1;
  }
  return 0;
}

// q [n, heads, dim] over pages of keys and transposed values (elements of dt), each request's context by its block table; out [n, heads * dim].
// groups of requests share their first keys (group_starts [groups + 1], group_keys [groups], shared_keys [requests]: see PrefixArgs); every query
// lies behind its request's shared keys.  shared_rows: at least as many blocks of 16 * tiles_shared rows as all groups have.  Parts of
// shared_steps / own_steps steps of 32 keys, as many as there are at most.  scratch: n * heads * (shared_parts + own_parts) * (dim + 2) floats.
extern "C" int tp_prefix_attention(const void* q, int dt, const void* k_cache, const void* v_cache, const int* block_tables, int table_width,
                                   const int* cu_seqlens, const int* context_lens, const int* token_req, const int* group_starts,
                                   const int* group_keys, const int* shared_keys, void* out, float* scratch, int n, int requests, int groups,
                                   int heads, int kv_heads, int dim, int page_size, float scale, float softcap, const float* sink, int max_q_len,
                                   int tiles_shared, int tiles_own, int shared_rows, int shared_steps, int shared_parts, int own_steps, int own_parts,
                                   hipStream_t s) {
  if (n <= 0 || requests <= 0) return 0;
  TP_REQUIRE(dt == TP_BF16 || dt == TP_F32, "prefix_attention: unsupported element type");
  TP_REQUIRE(dim == 32 || dim == 64 || dim == 128, "prefix_attention: heads of 32, 64 or 128 elements");
  TP_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "prefix_attention: pages of a power of two from 16 on");
  TP_REQUIRE(kv_heads > 0 && heads % kv_heads == 0 && groups > 0 && max_q_len > 0, "prefix_attention: bad sizes");
  TP_REQUIRE(shared_steps > 0 && own_steps > 0 && shared_parts > 0 && own_parts > 0 && shared_parts + own_parts <= PA_MAX_PARTS && shared_rows > 0,
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
  a.sums = scratch + (size_t)n * heads * a.parts * 2;
  a.table_width = table_width;
  a.page_shift = __builtin_ctz(page_size);
  a.n_heads = heads;
  a.n_kv = kv_heads;
  a.groups = groups;
  a.requests = requests;
  a.shared_rows = shared_rows;
  a.shared_parts = shared_parts;
  a.own_rows = (int)(((long)max_q_len * (heads / kv_heads) + 16 * tiles_own - 1) / (16 * tiles_own));
  a.shared_steps = shared_steps;
  a.own_steps = own_steps;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.cap_log2 = softcap * 1.4426950408889634f;
  a.cap_in = softcap > 0.f ? 2.0f * a.scale_log2 / softcap : 0.f;
  const long shared_blocks = (long)shared_rows * shared_parts, blocks = (shared_blocks + (long)a.own_rows * requests * own_parts) * kv_heads;
  TP_REQUIRE(blocks < (1L << 31), "prefix_attention: too many blocks");
  a.shared_blocks = (int)shared_blocks;
  int rc = 1;
  if (dt == TP_BF16)
    rc = dim == 32 ? prefix_sizes<2, 32>(a, (int)blocks, tiles_shared, tiles_own, s) : dim == 64 ? prefix_sizes<2, 64>(a, (int)blocks, tiles_shared, tiles_own, s)
                                                                                            : prefix_sizes<2, 128>(a, (int)blocks, tiles_shared, tiles_own, s);
  else
    rc = dim == 32 ? prefix_sizes<4, 32>(a, (int)blocks, tiles_shared, tiles_own, s) : dim == 64 ? prefix_sizes<4, 64>(a, (int)blocks, tiles_shared, tiles_own, s)
                                                                                            : prefix_sizes<4, 128>(a, (int)blocks, tiles_shared, tiles_own, s);
  if (rc != 0) return rc;
  TP_CHECK_LAUNCH("prefix_attention");
  const int rows = n * heads, grid = (rows + 3) / 4;
#define PA_JOIN(E, D) prefix_join_kernel<E, D><<<grid, 256, 0, s>>>(a.sums, a.stats, token_req, context_lens, shared_keys, out, sink, rows, heads, \
                                                                     shared_parts, a.parts, shared_steps, own_steps)
  if (dt == TP_BF16) {
    if (dim == 32) PA_JOIN(2, 32);
    else if (dim == 64) PA_JOIN(2, 64);
    else PA_JOIN(2, 128);
  } else {
    if (dim == 32) PA_JOIN(4, 32);
    else if (dim == 64) PA_JOIN(4, 64);
    else PA_JOIN(4, 128);
  }
#undef PA_JOIN
  TP_CHECK_LAUNCH("prefix_attention (join)");
  return 0;
}
