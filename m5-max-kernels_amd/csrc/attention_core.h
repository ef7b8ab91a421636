// Attention for gfx950: out = softmax(scores(Q K^T) + mask) V with one pass over the keys, K and V dense or in
// the pages of a cache.
//
// Rows.  The query heads that share a key head are packed: packed row r of a sequence is token r / G, query head
// kvh * G + r % G (G = heads / kv_heads), so one K/V tile serves all of them and a single token still fills G rows.
// A workgroup has 4 waves of 32 rows; a wave keeps its Q in registers.
//
// Masks.  Every mask of these operators (causal, window, document, prefix, length) leaves a row one interval
// [lo, hi) of keys.  Key tiles outside the union of a wave's intervals are skipped, tiles inside all of them need
// no comparison, the others compare the key index.
//
// Products.  v_mfma_f32_32x32x16 on S^T = K Q^T and O^T = V^T P^T.  With S transposed a lane holds scores of one
// query (lane & 31) only: 16 of the 32 keys of a block, the other 16 in lane ^ 32, so that a row's maximum is a
// chain of v_max in registers and one exchange, and row statistics are per-lane scalars.  The accumulator's key
// order (8 (r >> 2) + 4 (lane >> 5) + (r & 3)) is used unchanged as the K order of the second product: register
// octet s of P is its operand for keys 16 s .. 16 s + 15, and V^T is read in the same order, two groups of 4 keys,
// by ds_read_b64_tr_b16 (the transpose of a 4 x 16 block on the way out of LDS).  P never leaves registers.
//
// Softmax.  Running maximum m and sum in FP32: p = exp2(unit (x - m)), x the score, unit = scale * log2(e).  The
// maximum is raised, and O and the sum rescaled, only where a row's tile maximum exceeds it by more than 8 / unit: p
// stays below 2^8, the quotient of O and the sum does not depend on m, and most tiles skip the rescale.  P is rounded
// to the inputs' type for the matrix cores (as the second product's operand has to be); the sum takes the unrounded p.
//
// Scores of any size.  The loop has one multiply-add a score, x unit - (m unit), off by the rounding of m unit: 2^-5 at
// 2^20, and past 2^27 enough to take p out of range.  Rows that end there run again in careful mode (below), with
// unit (x - m).  Splits and waves are joined by unit (m - m') of the unscaled maxima.  A row that sees no key ends with
// a sum of 0 and the maximum it began with, and is 0; one that sees keys of score -inf alone leaves a maximum of -inf,
// and is NaN if every part of it does.
//
// NaN and infinities.  A masked key's score is replaced, whatever it was, but its value row still meets the product
// as 0 * v.  A wave whose sums end non-finite makes its workgroup run again in careful mode: non-finite values
// enter as 0, and their effect on the rows that do see them is found by a second product of indicators.  Key rows
// behind the length and rows of pages that the cache lacks read as zeros instead.
//
// What bounds it.  Long prompts: the card's power and the issue of products beside exponentials (9914 tokens, 56 heads
// of 128: 2.51 to 2.64 ms by the card, 1.1 PFLOP/s, matrix cores busy 64% of the cycles, no LDS bank conflicts).
// Single tokens: the cache's bytes (131073 keys, 8 key heads of 128: 94 to 100 us and 5 us of joining, 5.5 TB/s).
// Heads of 64: the exponentials.
//
// Registers.  Tiles of 128 rows with heads of 128 use 241 to 256, all there are for two waves a SIMD.  With a cap or a
// bias 8 to 10 of them go to memory and come back inside the loop, 34 by pages of no multiple of 16 (chunks of up to
// 1024 tokens over up to 8192 keys, bias: 232 us in pages of 64, 536 in pages of 24; without the bias 182 and 251).
#pragma once

#include "attention_place.h"
#include "gemm_core.h"
#include "m5k_common.h"

namespace m5k {
namespace attn {

using gemm::v16f;
using gemm::v4i;

constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr float M_FLOOR = -3.40282347e38f;  // running maximum before any key: finite, so that no difference is NaN
constexpr float FAR = 1048576.0f;           // maximum, in base 2, from which the careful mode takes over
constexpr float LAZY = 8.0f;       // log2 of how far a tile maximum may pass the running one unadopted
constexpr float LOG2E = 1.44269504088896340736f;

struct Args {
  const uint16_t *q, *k, *v;
  int64_t q_head, q_token, k_page, k_head, k_row, v_page, v_head, v_row;  // strides in elements
  const int32_t *table, *starts, *context, *prefix;
  int64_t table_width;
  const float* slopes;
  uint16_t* out;
  float *part_o, *part_ml;
  int tokens, keys, heads, kv_heads, group, sequences, pages, page_size, window, causal, splits, slots, spread, cus;
  uint32_t page_magic, page_shift, group_magic, group_shift;
  float scale, softcap;
};

// n / d of 0 <= n < 2^31 by one multiplication: magic = ceil(2^(31 + shift) / d), shift = ceil(log2 d).  The excess
// magic * d - 2^(31 + shift) is below d <= 2^shift, so n times it stays below 2^(31 + shift) and the quotient is exact.
__device__ __forceinline__ uint32_t fast_div(uint32_t n, uint32_t magic, uint32_t shift) {
  return __umulhi(2 * n, magic) >> shift;
}

template <int DT>
__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
  if constexpr (DT == M5K_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(gemm::bf16x8, a),
                                                   __builtin_bit_cast(gemm::bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(gemm::f16x8, a),
                                                  __builtin_bit_cast(gemm::f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == M5K_BF16) return f32x2_to_bf16x2(lo, hi);
  else return f32_to_f16_bits(lo) | (f32_to_f16_bits(hi) << 16);
}

// The other half-wave's value of the same row.
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

// 16 bytes a lane from a 64-bit address straight into LDS at lds_base + 16 lane.  Inline asm for the reason given at
// gemm::dma16; it has no register outputs, and every reader waits for vmcnt and a barrier.
__device__ __forceinline__ void dma16_flat(uint32_t lds_base, const void* p) {
  __asm__ volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(p)
      : "memory", "m0");
}

static __device__ const uint4 kZeros[1] = {};

// vmcnt(0) lgkmcnt(0), as the builtin: the compiler counts it, and does not wait again for the loads before the loop
// (Q) among those in flight.
__device__ __forceinline__ void wait_all() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  __asm__ volatile("" ::: "memory");
}

// Key tile in LDS: rows of D * 2 bytes, 16-byte chunk c of row r at chunk c ^ swizzle(r).  The 16 consecutive rows of a
// ds_read_b128 phase (K) then fall on 16 different bank groups, and so do the 4 rows x 64 bytes that half a wave's
// transposed read covers (V): rows r and r + 1 (two of them share 256 bytes at D = 64) differ in the 64-byte block.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  if constexpr (D == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else return ((row & 3) << 2) | ((row >> 2) & 3);
}

// Where keys and values lie.  PAGES16: pages of a multiple of 16 keys, so that the 16 rows of a tile that one wave
// loads lie in one page and take one address; PAGES: any page size, an address a lane.
enum Keys { DENSE = 0, PAGES16 = 1, PAGES = 2 };

// Page id at a position of the table, the same for the whole wave.  SCALAR: a scalar load, which leaves vmcnt to the
// tiles in flight.  Otherwise a load per lane: a scalar one shares lgkmcnt with the LDS reads, out of order, and makes
// each of them wait.
template <bool SCALAR>
__device__ __forceinline__ int table_entry(const int32_t* table, uint32_t at) {
  if constexpr (SCALAR) {
    at = __builtin_amdgcn_readfirstlane(at);
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(table))[at];
  } else {
    __asm__("" : "+v"(at));
    return table[at];
  }
}

// Buffer window of up to `rows` rows of `stride` elements from `p`, reading 0 behind them: rows are at least D apart,
// so a row behind the last begins behind the window's end.
template <int D>
__device__ __forceinline__ v4i rows_rsrc(const uint16_t* p, int rows, int64_t stride) {
  const int64_t n = rows > 0 ? ((rows - 1) * stride + D) * 2 : 0;
  return gemm::buffer_rsrc(p, static_cast<uint32_t>(n));
}

struct RowRange {
  int lo, hi;  // visible keys; lo > hi where there are none
  int pos;     // position on the key axis, for the distance bias
};

// The interval of a row at position p of a span [s, e) of keys.
__device__ __forceinline__ RowRange row_range(int s, int e, int p, int prefix, int causal, int window) {
  int lo = s, hi = e;
  if (causal) hi = min(e, max(p + 1, s + prefix));
  if (window) {
    lo = max(lo, p - window + 1);
    if (!causal) hi = min(hi, p + window);
  }
  if (hi <= lo) { lo = 0x3FFFFFFF; hi = 0; }
  return RowRange{lo, hi, p};
}

// The last b in [0, n) with key(b) <= x, by binary search over a nondecreasing key; 0 if there is none.
template <class Key>
__device__ __forceinline__ int last_not_above(int n, int x, Key key) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (key(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = min(v, __shfl_xor(v, o));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor(v, o));
  return __builtin_amdgcn_readfirstlane(v);
}

// tanh in FP32 to a few units of its last place: the series below 1/4 (first term left out 9e-3 y^11), elsewhere
// 1 - 2 / (e^(2y) + 1), whose absolute error is 1e-7.
__device__ __forceinline__ float tanh_f32(float y) {
  const float z = y * y;
  float s = __builtin_fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f);
  s = __builtin_fmaf(z, s, 2.0f / 15.0f);
  s = __builtin_fmaf(z, s, -1.0f / 3.0f);
  s = __builtin_fmaf(y * z, s, y);
  const float e = __builtin_amdgcn_exp2f(y * (2.0f * LOG2E));
  const float f = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
  return z < 0.0625f ? s : f;
}
// Caps up to here take the second form alone, C - 2 C / (e^(2y) + 1) in five instructions: off by C 2^-22, 6e-5 at
// most (16 heads of 64, 1999 tokens: 72 us with tanh_f32, 38 us).
constexpr float CAP_SHORT = 128.0f;

// acc + sum * f, f the weight of a sum.  Infinities and NaN that a row saw stay, also where f is below FP32's range:
// times 0 an infinity would be NaN.
__device__ __forceinline__ float add_scaled(float acc, float sum, float f) {
  return fabsf(sum) < __builtin_inff() ? __builtin_fmaf(sum, f, acc) : acc + sum;
}

// Non-finite 16-bit values of a fragment: zero in `clean`; `mark` holds 1 for +inf, 128 for -inf, 16384 for NaN.
template <int DT>
__device__ __forceinline__ void split_nonfinite(v4i f, v4i& clean, v4i& mark) {
  constexpr uint32_t EXP = DT == M5K_BF16 ? 0x7F80u : 0x7C00u;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t c = 0, m = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = (static_cast<uint32_t>(f[w]) >> (16 * h)) & 0xFFFFu;
      const bool bad = (x & EXP) == EXP;
      const float code = (x & 0x7FFFu) != EXP ? 16384.0f : (x & 0x8000u) ? 128.0f : 1.0f;
      const uint32_t bits = DT == M5K_BF16 ? f32_to_bf16_bits(code) : f32_to_f16_bits(code);
      c |= (bad ? 0u : x) << (16 * h);
      m |= (bad ? bits : 0u) << (16 * h);
    }
    clean[w] = static_cast<int>(c);
    mark[w] = static_cast<int>(m);
  }
}

// What a row gets from the non-finite values that it sees: 0, an infinity or NaN, from the sum of their marks.  A tile
// has 64 keys, so that the counts of +inf (below 128) and -inf (64 * 128 < 16384) keep apart.
__device__ __forceinline__ float nonfinite_sum(float marks) {
  const uint32_t u = static_cast<uint32_t>(marks), plus = u & 127u, minus = u & (127u << 7);
  const uint32_t inf = plus ? 0x7F800000u : 0xFF800000u;
  const uint32_t bits = (u >> 14) | (plus & -static_cast<uint32_t>(minus != 0)) ? 0x7FC00000u : inf;
  return __uint_as_float(u ? bits : 0u);
}

// One workgroup's place: packed rows [row0, row0 + rows) of a sequence whose first token is `token0`.
struct Place {
  int seq, kvh, split, tile, token0, rows;  // rows: packed rows of the whole sequence
  int span, shift;                          // keys; position of token i is i + shift
};

template <int KEYS>
__device__ __forceinline__ Place place(const Args& a, int rows_per_tile) {
  Place p;
  int slot;
  if (a.spread) {
    // Tiles of unequal work, and heads that do not divide among the XCDs: in turn over the XCDs, longest first under a
    // causal mask; what a compute unit gets as its second workgroup of a grid that is resident at once is the
    // shortest left.  (6000 causal tokens, 12 query heads on 3 key heads: 189 us by XCDs, whose parts of a head differ
    // in work, 129 us.)
    const int total = gridDim.x, id = blockIdx.x;
    int item = total <= 2 * a.cus && id >= a.cus ? total - 1 - (id - a.cus) : id;
    p.kvh = item % a.kv_heads;
    item /= a.kv_heads;
    p.split = item % a.splits;
    slot = item / a.splits;
  } else {
    // One XCD after the other takes whole heads, so that a head's keys stay in its L2.
    int item = gemm::xcd_logical(blockIdx.x, gridDim.x);
    p.split = item % a.splits;
    item /= a.splits;
    p.kvh = item / a.slots;
    slot = item % a.slots;
  }
  slot = a.slots - 1 - slot;  // later tiles see more keys under a causal mask: they go first
  if constexpr (KEYS == DENSE) {
    p.seq = 0;
    p.tile = slot;
    p.token0 = 0;
    p.rows = a.tokens * a.group;
    p.span = a.keys;
    p.shift = a.keys - a.tokens;
  } else {
    const int T = a.tokens, B = a.sequences;
    const auto probes = [&](int lo, int left, int apart) {
      const int probe = static_cast<int>(threadIdx.x & 63) * apart;
      const bool below = probe < left && first_slot(a.starts, lo + probe, T, a.group, rows_per_tile) <= slot;
      return __popcll(__builtin_amdgcn_ballot_w64(below));
    };
    p.seq = __builtin_amdgcn_readfirstlane(sequence_of_slot(B + 1, probes));
    p.token0 = start_of(a.starts, p.seq, T);
    p.tile = slot - first_slot(a.starts, p.seq, T, a.group, rows_per_tile);
    const int n = tokens_of(a.starts, p.seq, B, T);
    p.rows = n * a.group;
    const int ctx = p.seq == B ? 0 : a.context[p.seq];
    p.span = min(max(ctx, 0), a.keys);
    p.shift = ctx - n;
  }
  return p;
}

// The row range, and the token and query head of packed row r (r < p.rows).
template <int KEYS>
__device__ __forceinline__ RowRange range_of(const Args& a, const Place& p, int r, int& token, int& head) {
  const int i = a.group == 1 ? r : static_cast<int>(fast_div(r, a.group_magic, a.group_shift));
  head = p.kvh * a.group + r - i * a.group;
  token = p.token0 + i;
  int s = 0, e = p.span, prefix = 0;
  if (KEYS == DENSE && a.starts) {
    const int d = last_not_above(a.sequences, i, [&](int b) { return a.starts[b]; });
    s = max(a.starts[d], 0);
    e = min(a.starts[d + 1], a.keys);
    if (i < s || i >= e) e = s = 0;
    if (a.prefix) prefix = a.prefix[d];
  } else if (a.prefix && (KEYS == DENSE || p.seq < a.sequences)) {
    prefix = a.prefix[p.seq];
  }
  prefix = min(max(prefix, 0), 0x3FFFFFFF);
  return row_range(s, e, i + p.shift, prefix, a.causal, a.window);
}

// FEW = false: the 4 waves take 32 rows each and share key tiles of 64.  FEW: they share 32 rows, for calls that have
// no more, and take every fourth tile of 32 keys each, through LDS of their own: no barrier in the loop, and the keys
// of a short row are read four tiles at a time.
//
// Tiles of K and V that a wave of FEW holds: one of each, so that two or three workgroups run on a compute unit at once
// (two of each at heads of 128, one workgroup: 64 tokens over 300 keys 36 us instead of 24).  Two of each where an
// address a lane (PAGES) makes the loads long and heads of 64 leave room for two workgroups: with one and with two, 830
// tokens of three sequences, window and cap, pages of 24, 16 heads: 27.4 and 24.2 us; 8 chunks of 64 tokens over 1564
// keys, 16 heads: 32.2 and 26.5; 63 single tokens over 1 to 4000 keys, 8 key heads: 72.6 and 57.8; single tokens over
// 1000 keys, one key head: 480 of them 28.2 and 24.7, but 508, which just fill the chip, 28.6 and 36.7.  By whole
// addresses (pages of 16, dense) two of each gained 10% in some calls and lost 3 to 12% in others.
template <int DT, int D, int KEYS, bool MODS, bool FEW>
__global__ __launch_bounds__(THREADS, 2) void attention_tile(const Args a) {
  constexpr int KT = FEW ? 32 : 64, NB = KT / 32;  // keys of a tile, 32-key blocks
  constexpr int EL = 16 * NB;                      // scores of a lane
  constexpr int CH = D / 8;                        // 16-byte chunks of a row
  constexpr int RPI = 64 / CH;                     // rows of one load instruction
  constexpr int LOADED = FEW ? KT : KT / WAVES;    // rows of a tile that one wave loads
  constexpr int GROUPS = LOADED / 16;
  constexpr int NI = LOADED / RPI;  // its load instructions, each of K and V
  constexpr int QS = D / 16, OB = D / 32;
  constexpr int AHEAD = 1;  // steps of two products between a fragment's read and its use (2: no faster)
  constexpr int ROWS = FEW ? 32 : 32 * WAVES;
  constexpr int STAGES = FEW && !(KEYS == PAGES && D == 64) ? 1 : 2;  // tiles of K, and of V, in LDS
  constexpr uint32_t ROWB = D * 2, TILE = KT * ROWB, VTILE = STAGES * TILE;
  // K stages, V stages.  FEW: those of each wave, later its sums, in rows of D + 4 floats (16 bytes a lane without bank
  // conflicts), and their maxima and totals.
  constexpr uint32_t SUMS = (D + 4) * 4, JOIN = 32 * SUMS + 256, AREA = JOIN > 2 * VTILE ? JOIN : 2 * VTILE;
  __shared__ __attribute__((aligned(256))) uint8_t lds[FEW ? WAVES * AREA : 4 * TILE];
  __shared__ int bounds[2 * WAVES];

  const Place p = place<KEYS>(a, ROWS);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  if (!tile_has_rows(p.tile, p.rows, ROWS)) return;
  const int row0 = p.tile * ROWS;
  const int row = row0 + (FEW ? 0 : 32 * wave) + (lane & 31);
  const bool live = row < p.rows;
  int token, head;
  const RowRange rr = range_of<KEYS>(a, p, min(row, p.rows - 1), token, head);

  // Key ranges: of the wave (any row, every row), and of the workgroup.
  const bool idle = !FEW && row0 + 32 * wave >= p.rows;
  const int any_lo = idle ? 0x3FFFFFFF : wave_min_i(rr.lo), any_hi = idle ? 0 : wave_max_i(rr.hi);
  const int all_lo = wave_max_i(rr.lo), all_hi = wave_min_i(rr.hi);
  int lo = any_lo, hi = any_hi;
  if constexpr (!FEW) {
    if (lane == 0) {
      bounds[wave] = any_lo;
      bounds[WAVES + wave] = any_hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      lo = min(lo, bounds[w]);
      hi = max(hi, bounds[WAVES + w]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
  }
  int t_begin = 0, t_end = 0;
  if (lo < hi) {
    t_begin = lo / KT;
    t_end = (hi + KT - 1) / KT;
    if (a.splits > 1) {
      // At least 256 keys a split: below, the partial sums cost more than the keys.
      const int per = max((t_end - t_begin + a.splits - 1) / a.splits, 256 / KT);
      t_begin = min(t_begin + p.split * per, t_end);
      t_end = min(t_begin + per, t_end);
    }
  }

  v4i qf[QS];
  {
    const uint16_t* qp = a.q + int64_t{head} * a.q_head + int64_t{token} * a.q_token + 8 * half;
#pragma unroll
    for (int s = 0; s < QS; ++s) qf[s] = *reinterpret_cast<const v4i*>(qp + 16 * s);
  }
  const float scale2 = a.scale * LOG2E;
  const float unit = MODS ? 1.0f : scale2;  // what turns finished scores into base 2, launch_unit()
  const float slope2 = MODS && a.slopes ? a.slopes[head] * LOG2E : 0.0f;

  // Loads: instruction i of a wave brings rows first_row + i * RPI + lane / CH of K and of V.
  const int first_row = FEW ? 0 : wave_s * LOADED;
  const int ld_row = first_row + lane / CH, ld_chunk = lane % CH;
  const uint16_t* kbase = a.k + int64_t{p.kvh} * a.k_head;
  const uint16_t* vbase = a.v + int64_t{p.kvh} * a.v_head;
  const int32_t* table = KEYS != DENSE && p.seq < a.sequences ? a.table + int64_t{p.seq} * a.table_width : nullptr;
  const uint32_t lds0 = gemm::lds_addr(lds) + (FEW ? wave_s * AREA : 0);
  uint32_t kofs[NI], vofs[NI];  // bytes of a lane's chunk from the window's first row
  if constexpr (KEYS != PAGES) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = KEYS == DENSE ? ld_row + i * RPI : lane / CH + i % (NI / GROUPS) * RPI;  // pages: of 16 rows
      const int chunk = (ld_chunk ^ swizzle<D>(ld_row + i * RPI)) * 8;
      kofs[i] = static_cast<uint32_t>(r * static_cast<int>(a.k_row) + chunk) * 2;
      vofs[i] = static_cast<uint32_t>(r * static_cast<int>(a.v_row) + chunk) * 2;
    }
  }
  constexpr int NIDS = KEYS == PAGES ? NI : GROUPS;
  int ids[2][NIDS] = {};  // pages of the next tile's keys, and of the tile before it, whose values come next
  bool lacking = false;

  // Unconditional, at the last key where tile t has none: a load under a condition would be waited for at the
  // condition's end, and with it everything in flight.
  auto load_ids = [&](int t, int (&to)[NIDS]) __attribute__((always_inline)) {
    if constexpr (KEYS == PAGES16) {
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const int key = min(t * KT + first_row + 16 * i, p.span - 1);
        to[i] = table_entry<FEW>(table, fast_div(key, a.page_magic, a.page_shift));
      }
    } else if constexpr (KEYS == PAGES) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int key = min(t * KT + ld_row + i * RPI, p.span - 1);
        to[i] = table[fast_div(key, a.page_magic, a.page_shift)];
      }
    }
  };
  // This wave's rows of tile t of one operand to LDS at dst.
  auto load_rows = [&](int t, const int (&id)[NIDS], const uint16_t* base, int64_t page_stride, int64_t row_stride,
                       const uint32_t (&ofs)[NI], uint32_t dst) __attribute__((always_inline)) {
    dst += FEW ? 0 : wave_s * NI * 1024;
    if constexpr (KEYS == PAGES) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = ld_row + i * RPI, key = t * KT + r;
        const int chunk = (ld_chunk ^ swizzle<D>(r)) * 8;
        const bool in = key < p.span, has = static_cast<uint32_t>(id[i]) < static_cast<uint32_t>(a.pages);
        lacking |= in && !has;
        const int slot = key - static_cast<int>(fast_div(key, a.page_magic, a.page_shift)) * a.page_size;
        const void* at = kZeros;
        if (in && has) at = base + id[i] * page_stride + slot * row_stride + chunk;
        dma16_flat(dst + i * 1024, at);
      }
    } else if constexpr (KEYS == DENSE) {
      const v4i rsrc = rows_rsrc<D>(base + int64_t{t} * KT * row_stride, min(p.span - t * KT, KT), row_stride);
#pragma unroll
      for (int i = 0; i < NI; ++i) gemm::dma16<true>(dst + i * 1024, ofs[i], rsrc);
    } else {
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int key = t * KT + first_row + 16 * g, page = __builtin_amdgcn_readfirstlane(id[g]);
        const uint16_t* at = base;
        int rows = min(p.span - key, 16);
        if (rows > 0) {
          if (static_cast<uint32_t>(page) < static_cast<uint32_t>(a.pages)) {
            const int slot = key - static_cast<int>(fast_div(key, a.page_magic, a.page_shift)) * a.page_size;
            at += page * page_stride + slot * row_stride;
          } else {
            rows = 0;
            lacking = true;
          }
        }
        const v4i rsrc = rows_rsrc<D>(at, rows, row_stride);
        constexpr int PER = NI / GROUPS;
#pragma unroll
        for (int i = 0; i < PER; ++i) gemm::dma16<true>(dst + (g * PER + i) * 1024, ofs[g * PER + i], rsrc);
      }
    }
  };

  // Fragment addresses in stage 0 (the other stage and the rows further on are instruction offsets): chunk c of a row
  // is its chunk 0 XOR 16 c, rows being aligned to their size.
  uint32_t kread[QS], vread[2][OB];
  const int g = lane >> 4, gi = lane & 15;
  const int vrow = 4 * half + (gi >> 2), vchunk = 2 * (g & 1) + ((gi & 3) >> 1);
#pragma unroll
  for (int c = 0; c < QS; ++c)
    kread[c] = (lds0 + (lane & 31) * ROWB + ((half ^ swizzle<D>(lane & 31)) << 4)) ^ (c << 5);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int b = 0; b < OB; ++b)
      vread[h][b] =
          (lds0 + (8 * h + vrow) * ROWB + ((vchunk ^ swizzle<D>(8 * h + vrow)) << 4) + (gi & 1) * 8) ^ (b << 6);

  wait_all();
  v16f o[OB], s[2][NB];
  v4i pf[2 * NB];
  float m, m2, l;  // maximum, the same in base 2, sum

  // Scores of a tile, from K at stage `st`; beside them, where `prob`, the probabilities of the tile before against the
  // running maximum, packed for the second product, and their sum.  A 32 x 32 x 16 product holds the matrix cores for
  // 32 cycles, in which the wave issues 8 VALU instructions: each step's fence keeps its share of the exponentials
  // between its products, and the next step's fragments on their way.
  auto key_frags = [&](int st, int c, v4i (&f)[NB]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
      f[b] = *reinterpret_cast<const __attribute__((address_space(3))) v4i*>(kread[c] + b * 32 * ROWB + st * TILE);
  };
  // V^T fragment of k-step c and channel block b: keys 16 c + 8 h + 4 (lane >> 5) .. + 3 for h = 0, 1.
  auto value_frag = [&](int st, int c, int b) __attribute__((always_inline)) {
    v4i f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_v4s>(vread[h][b] + 16 * c * ROWB + VTILE + st * TILE));
      const auto y = __builtin_bit_cast(m5k_u32x2, x);
      f[2 * h] = static_cast<int>(y[0]);
      f[2 * h + 1] = static_cast<int>(y[1]);
    }
    return f;
  };
  constexpr std::false_type quick{};
  constexpr std::true_type careful{};
  auto weight = [&](float x, auto with_care) __attribute__((always_inline)) {
    float t = __builtin_fmaf(x, unit, -m2);
    if constexpr (decltype(with_care)::value) t = fabsf(m2) < FAR ? t : (x - m) * unit;
    return __builtin_amdgcn_exp2f(t);
  };
  auto probabilities = [&](const v16f (&x)[NB], int from, int to, float (&sum)[2], auto with_care)
                           __attribute__((always_inline)) {
#pragma unroll
    for (int e = from; e < to; e += 2) {
      const int b = e >> 4, r = e & 15;
      const float p0 = weight(x[b][r], with_care), p1 = weight(x[b][r + 1], with_care);
      sum[0] += p0;
      sum[1] += p1;
      uint32_t w = pack2<DT>(p0, p1);
      __asm__ volatile("" : "+v"(w), "+v"(sum[0]), "+v"(sum[1]));  // made here, not where they are read
      pf[2 * b + (r >> 3)][(r & 7) >> 1] = static_cast<int>(w);
      if constexpr (decltype(with_care)::value) __builtin_amdgcn_sched_barrier(0);  // rare: few registers
    }
  };
  auto product = [&](v16f (&y)[NB], int st, const v16f (&x)[NB], bool prob) __attribute__((always_inline)) {
    v4i kf[AHEAD + 1][NB];
    float sum[2] = {};
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) key_frags(st, c, kf[c]);
#pragma unroll
    for (int c = 0; c < QS; ++c) {
      if (c + AHEAD < QS) key_frags(st, c + AHEAD, kf[(c + AHEAD) % (AHEAD + 1)]);
#pragma unroll
      for (int b = 0; b < NB; ++b) y[b] = mfma32<DT>(kf[c % (AHEAD + 1)][b], qf[c], c == 0 ? v16f{} : y[b]);
      if (prob) probabilities(x, c * EL / QS, (c + 1) * EL / QS, sum, quick);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (prob) l += sum[0] + sum[1];
  };
  // Cap, bias and mask of tile t's scores.
  auto finish = [&](v16f (&x)[NB], int t, auto with_care, uint32_t& sees_bits) __attribute__((always_inline)) {
    constexpr bool careful = decltype(with_care)::value;
    const int key0 = t * KT, kofs0 = key0 + 4 * half;
    if constexpr (MODS) {
      // Scores in base 2: capped, or scaled with the bias.  Distances are whole numbers, exact in FP32 up to 2^24.
      if (a.softcap > 0.0f) {
        const float cap2 = a.softcap * LOG2E, y = a.scale / a.softcap;
        if (a.softcap <= CAP_SHORT) {
          const float y2 = y * (2.0f * LOG2E);
#pragma unroll
          for (int e = 0; e < EL; ++e) {
            const float g = __builtin_amdgcn_exp2f(x[e >> 4][e & 15] * y2) + 1.0f;
            x[e >> 4][e & 15] = __builtin_fmaf(-2.0f * cap2, __builtin_amdgcn_rcpf(g), cap2);
            if ((e & 7) == 7) __builtin_amdgcn_sched_barrier(0);
          }
        } else {
#pragma unroll
          for (int e = 0; e < EL; ++e) {
            x[e >> 4][e & 15] = tanh_f32(x[e >> 4][e & 15] * y) * cap2;
            if ((e & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // few registers
          }
        }
      }
      if (a.slopes) {
        const float apart = static_cast<float>(rr.pos - kofs0), f = a.softcap > 0.0f ? 1.0f : scale2;
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          const float d = fabsf(apart - static_cast<float>(32 * (e >> 4) + 8 * ((e & 15) >> 2) + (e & 3)));
          x[e >> 4][e & 15] = __builtin_fmaf(x[e >> 4][e & 15], f, -slope2 * d);
        }
      }
    }
    if (careful || key0 < all_lo || key0 + KT > all_hi) {
      const uint32_t width = static_cast<uint32_t>(max(rr.hi - rr.lo, 0));
      if constexpr (careful) sees_bits = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kofs0 + 32 * b + 8 * (r >> 2) + (r & 3);
          bool sees = static_cast<uint32_t>(key - rr.lo) < width;
          if constexpr (KEYS != DENSE && careful) {
            if (sees)
              sees = static_cast<uint32_t>(table[fast_div(key, a.page_magic, a.page_shift)]) <
                     static_cast<uint32_t>(a.pages);
          }
          if constexpr (careful) sees_bits |= static_cast<uint32_t>(sees) << (16 * b + r);
          x[b][r] = sees ? x[b][r] : -__builtin_inff();
        }
    }
  };
  // O += V^T P of a tile, V at stage `st`, in steps of two products as above; beside them the maximum of the scores x.
  auto accumulate = [&](int st, const v16f (&x)[NB]) __attribute__((always_inline)) -> float {
    constexpr int STEPS = 2 * NB * OB / 2;
    v4i vf[AHEAD + 1][2];
    float t0 = x[0][0], t1 = x[0][1];
#pragma unroll
    for (int j = 0; j < 2 * AHEAD; ++j) vf[j / 2][j & 1] = value_frag(st, j / OB, j % OB);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i + AHEAD < STEPS) {
        const int n = 2 * (i + AHEAD);
#pragma unroll
        for (int j = 0; j < 2; ++j) vf[(i + AHEAD) % (AHEAD + 1)][j] = value_frag(st, n / OB, n % OB + j);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int b = 2 * i % OB + j;
        o[b] = mfma32<DT>(vf[i % (AHEAD + 1)][j], pf[2 * i / OB], o[b]);
      }
#pragma unroll
      for (int e = i * EL / STEPS; e < (i + 1) * EL / STEPS; e += 2) {
        t0 = fmaxf(t0, x[e >> 4][e & 15]);
        t1 = fmaxf(t1, x[e >> 4][(e & 15) + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return fmaxf(t0, t1);
  };
  // The same with care: non-finite values apart, for the keys in `bits`.
  auto accumulate_careful = [&](uint32_t bits) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      v16f marks = {};
#pragma unroll
      for (int c = 0; c < 2 * NB; ++c) {
        v4i clean, mark, see;
        split_nonfinite<DT>(value_frag(0, c, b), clean, mark);
        const uint32_t one = pack2<DT>(1.0f, 1.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t two = bits >> (8 * c + 2 * w);
          see[w] = static_cast<int>(((two & 1u) ? one & 0xFFFFu : 0u) | ((two & 2u) ? one & 0xFFFF0000u : 0u));
        }
        marks = mfma32<DT>(mark, see, marks);
        o[b] = mfma32<DT>(clean, pf[c], o[b]);
        __builtin_amdgcn_sched_barrier(0);  // rare: few registers rather than overlap
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] += nonfinite_sum(marks[r]);
    }
  };
  auto maximum = [&](const v16f (&x)[NB]) __attribute__((always_inline)) {
    float t0 = x[0][0];
#pragma unroll
    for (int e = 1; e < EL; ++e) t0 = fmaxf(t0, x[e >> 4][e & 15]);
    return t0;
  };
  // Adopt a tile maximum where a row's exceeds the running one by more than LAZY.
  auto adopt = [&](float tile_top, auto with_care) __attribute__((always_inline)) {
    const float t = max_halves(tile_top);
    if (__builtin_amdgcn_ballot_w64((t - m) * unit > LAZY)) {
      const float next = fmaxf(m, t), f = __builtin_amdgcn_exp2f((m - next) * unit);
      m = next;
      m2 = fmaxf(m * unit, M_FLOOR);  // finite: a masked score, -inf, stays one
      l *= f;
#pragma unroll
      for (int b = 0; b < OB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] = decltype(with_care)::value ? add_scaled(0.0f, o[b][r], f) : o[b][r] * f;
    }
  };

  const int first = max(t_begin, any_lo / KT), last = min(t_end, (any_hi + KT - 1) / KT);  // this wave's tiles
  auto start = [&]() __attribute__((always_inline)) {
    m = m2 = M_FLOOR;
    l = 0.0f;
#pragma unroll
    for (int b = 0; b < OB; ++b) o[b] = v16f{};
  };

  // Step t turns the scores of tile t into its part of O, and makes the scores of tile t + 1 meanwhile, so that the
  // matrix cores have work beside the exponentials.  The i-th step (ODD = i & 1) reads K of tile t + 1 in stage ODD and
  // V of tile t in stage EVEN; it loads V of tile t + 1 and K of tile t + 2 over what the step before was the last to
  // read.
  auto step = [&](int t, auto odd, v16f (&x)[NB], v16f (&next)[NB]) __attribute__((always_inline)) {
    constexpr int ODD = decltype(odd)::value, EVEN = 1 - ODD;
    wait_all();
    gemm::stage_barrier();
    if (t + 1 < t_end) {
      load_rows(t + 1, ids[1], vbase, a.v_page, a.v_row, vofs, lds0 + (2 + ODD) * TILE);
      if (t + 2 < t_end) load_rows(t + 2, ids[0], kbase, a.k_page, a.k_row, kofs, lds0 + EVEN * TILE);
    }
#pragma unroll
    for (int i = 0; i < NIDS; ++i) ids[1][i] = ids[0][i];
    load_ids(t + 3, ids[0]);
    uint32_t none;
    const bool now = t >= first && t < last, then = t + 1 >= first && t + 1 < last;  // the same for the whole wave
    if (now && then) {
      product(next, ODD, x, true);
      finish(next, t + 1, quick, none);
      adopt(accumulate(EVEN, next), quick);
    } else if (then) {
      product(next, ODD, x, false);
      finish(next, t + 1, quick, none);
      adopt(maximum(next), quick);
    } else if (now) {
      float sum[2] = {};
      probabilities(x, 0, EL, sum, quick);
      l += sum[0] + sum[1];
      accumulate(EVEN, x);
    }
  };
  // FEW: this wave's tile t, from stage ST.  With two stages the next one (WAVES further on) is on its way to the other
  // meanwhile.  With one the K of the next is loaded as soon as this one's has been read, V likewise, so that one of
  // the two is on its way through every phase.  Loads end in the order of their issue.
  auto own_tile = [&](int t, auto stage) __attribute__((always_inline)) {
    constexpr int ST = decltype(stage)::value;
    const bool more = t + WAVES < t_end;
    if constexpr (STAGES == 2) {
      if (more) {
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last reads of that stage
        load_rows(t + WAVES, ids[0], kbase, a.k_page, a.k_row, kofs, lds0 + (1 - ST) * TILE);
        load_rows(t + WAVES, ids[0], vbase, a.v_page, a.v_row, vofs, lds0 + VTILE + (1 - ST) * TILE);
        load_ids(t + 2 * WAVES, ids[0]);
        gemm::wait_stage<2 * NI>();
      } else {
        gemm::wait_stage<0>();
      }
      product(s[0], ST, s[0], false);
    } else {
      gemm::wait_stage<NI>();  // K, behind which V was issued
      product(s[0], ST, s[0], false);
      if (more) {
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        load_rows(t + WAVES, ids[0], kbase, a.k_page, a.k_row, kofs, lds0);
      }
    }
    uint32_t none;
    finish(s[0], t, quick, none);
    adopt(maximum(s[0]), quick);
    float sum[2] = {};
    probabilities(s[0], 0, EL, sum, quick);
    l += sum[0] + sum[1];
    if constexpr (STAGES == 1) {
      if (more) gemm::wait_stage<NI>();
      else gemm::wait_stage<0>();
    }
    accumulate(ST, s[0]);
    if constexpr (STAGES == 1) {
      if (more) {
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        load_rows(t + WAVES, ids[0], vbase, a.v_page, a.v_row, vofs, lds0 + VTILE);
        load_ids(t + 2 * WAVES, ids[0]);
      }
    }
  };
  start();
  if constexpr (FEW) {
    int t = t_begin + wave_s;
    if (t < t_end) {
      load_ids(t, ids[0]);
      load_rows(t, ids[0], kbase, a.k_page, a.k_row, kofs, lds0);
      load_rows(t, ids[0], vbase, a.v_page, a.v_row, vofs, lds0 + VTILE);
      load_ids(t + WAVES, ids[0]);
    }
    for (; t < t_end; t += STAGES * WAVES) {
      own_tile(t, std::integral_constant<int, 0>{});
      if (STAGES == 2 && t + WAVES < t_end) own_tile(t + WAVES, std::integral_constant<int, STAGES - 1>{});
    }
  } else if (t_begin < t_end) {
    load_ids(t_begin, ids[1]);
    load_rows(t_begin, ids[1], kbase, a.k_page, a.k_row, kofs, lds0);
    load_ids(t_begin + 1, ids[0]);
    for (int t = t_begin - 1; t < t_end; t += 2) {
      step(t, std::integral_constant<int, 0>{}, s[0], s[1]);
      if (t + 1 < t_end) step(t + 1, std::integral_constant<int, 1>{}, s[1], s[0]);
    }
  }
  float checks[4] = {};  // NaN from any sum that is not finite, in four chains
#pragma unroll
  for (int b = 0; b < OB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) checks[r & 3] = __builtin_fmaf(o[b][r], 0.0f, checks[r & 3]);
  const float check = (checks[0] + checks[1]) + (checks[2] + checks[3]);
  // Whether the row saw a key here: one of its tiles of this wave meets its interval.
  bool saw;
  {
    const int from = max(t_begin, rr.lo / KT), to = min(t_end, (rr.hi + KT - 1) / KT);
    saw = from + (FEW ? (wave - (from - t_begin)) & (WAVES - 1) : 0) < to;
  }
  const bool far = !MODS && m != M_FLOOR && !(fabsf(m2) < FAR);
  wait_all();
  if (__syncthreads_or(lacking || far || check != 0.0f)) {
    saw = false;
    start();
    for (int t = t_begin; t < t_end; ++t) {
      if (FEW && ((t - t_begin) & (WAVES - 1)) != wave_s) continue;
      load_ids(t, ids[0]);
      load_rows(t, ids[0], kbase, a.k_page, a.k_row, kofs, lds0);
      load_rows(t, ids[0], vbase, a.v_page, a.v_row, vofs, lds0 + VTILE);
      wait_all();
      if constexpr (!FEW) gemm::stage_barrier();
      if (t >= first && t < last) {
        uint32_t sees;
        product(s[0], 0, s[1], false);
        finish(s[0], t, careful, sees);
        adopt(maximum(s[0]), careful);
        float sum[2] = {};
        probabilities(s[0], 0, EL, sum, careful);
        l += sum[0] + sum[1];
        accumulate_careful(sees);
        saw |= sees != 0;
      }
      wait_all();
      if constexpr (!FEW) gemm::stage_barrier();
    }
    if constexpr (FEW) __syncthreads();
    saw = (__builtin_amdgcn_ballot_w64(saw) >> (lane & 31)) & 0x100000001ull;  // in either half's keys
  }

  l += other_half(l);
  if (l == 0.0f && saw) m = -__builtin_inff();
  if constexpr (FEW) {
    // The waves' sums joined in LDS, in wave order, by 8 threads a row.
    uint8_t* mine = lds + wave * AREA;
    float* ml = reinterpret_cast<float*>(mine + 32 * SUMS) + 2 * (lane & 31);
    if (half == 0) {
      ml[0] = m;
      ml[1] = l;
    }
#pragma unroll
    for (int b = 0; b < OB; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(mine + (lane & 31) * SUMS + (32 * b + 2 * r + 4 * half) * 4) =
            make_float4(o[b][r], o[b][r + 1], o[b][r + 2], o[b][r + 3]);
    __syncthreads();
    constexpr int E = D / 8;
    const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * E;
    if (row0 + r >= p.rows) return;
    float top = M_FLOOR, total = 0.0f, acc[E] = {};
    float w[WAVES];
    bool lost = false;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      w[i] = *reinterpret_cast<const float*>(lds + i * AREA + 32 * SUMS + 8 * r);
      top = fmaxf(top, w[i]);
      lost |= w[i] < M_FLOOR;
    }
    auto add_up = [&](int i, auto with_care) __attribute__((always_inline)) {
      const float* src = reinterpret_cast<const float*>(lds + i * AREA + r * SUMS) + c;
#pragma unroll
      for (int e = 0; e < E; ++e)
        acc[e] = decltype(with_care)::value ? add_scaled(acc[e], src[e], w[i]) : __builtin_fmaf(src[e], w[i], acc[e]);
    };
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      w[i] = __builtin_amdgcn_exp2f((w[i] - top) * unit);
      total = __builtin_fmaf(*reinterpret_cast<const float*>(lds + i * AREA + 32 * SUMS + 8 * r + 4), w[i], total);
      add_up(i, quick);
    }
    float odd[2] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) odd[e & 1] = __builtin_fmaf(acc[e], 0.0f, odd[e & 1]);
    if (__builtin_amdgcn_ballot_w64(odd[0] + odd[1] != 0.0f)) {  // rare: a sum is not finite
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) add_up(i, careful);
    }
    int t_out, h_out;
    range_of<KEYS>(a, p, row0 + r, t_out, h_out);
    lost = lost && total == 0.0f;
    if (a.splits > 1) {
      const int64_t at = (int64_t{p.split} * a.tokens + t_out) * a.heads + h_out;
      if (c == 0) {
        a.part_ml[2 * at] = lost ? -__builtin_inff() : top;
        a.part_ml[2 * at + 1] = total;
      }
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(a.part_o + at * D + c + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
      return;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total, none = lost ? __builtin_nanf("") : 0.0f;
    uint16_t* op = a.out + (int64_t{t_out} * a.heads + h_out) * D + c;
#pragma unroll
    for (int e = 0; e < E; e += 8) {
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = total == 0.0f ? pack2<DT>(none, none) : pack2<DT>(acc[e + 2 * i] * inv, acc[e + 2 * i + 1] * inv);
      *reinterpret_cast<uint4*>(op + e) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    return;
  }
  if (!live) return;
  if (a.splits > 1) {
    const int64_t at = (int64_t{p.split} * a.tokens + token) * a.heads + head;
    if (half == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = l;
    }
    if (l == 0.0f && m == M_FLOOR) return;  // nothing seen here: the sums are not read
#pragma unroll
    for (int b = 0; b < OB; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<float4*>(a.part_o + at * D + 32 * b + 2 * r + 4 * half) =
            make_float4(o[b][r], o[b][r + 1], o[b][r + 2], o[b][r + 3]);
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l, none = m < M_FLOOR ? __builtin_nanf("") : 0.0f;
  const uint32_t nones = pack2<DT>(none, none);
  uint16_t* op = a.out + (int64_t{token} * a.heads + head) * D + 4 * half;
#pragma unroll
  for (int b = 0; b < OB; ++b)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const uint2 w = l == 0.0f ? make_uint2(nones, nones)
                                : make_uint2(pack2<DT>(o[b][r] * inv, o[b][r + 1] * inv),
                                             pack2<DT>(o[b][r + 2] * inv, o[b][r + 3] * inv));
      *reinterpret_cast<uint2*>(op + 32 * b + 2 * r) = w;
    }
}

// unit of a launch's kernels.
__device__ __forceinline__ float launch_unit(const Args& a) {
  return a.softcap > 0.0f || a.slopes ? 1.0f : a.scale * LOG2E;
}

// Joins the key splits of a (token, head), each split's sum weighted by 2^(unit (m - max m)).  Lane i holds split i's
// maximum and total, so that the weights cost one load; the sums' loads then wait for nothing but memory.  Latency
// bound: with WAVES_ROW = 4 (many splits, so few rows) the waves take a quarter of the splits each and add up in LDS,
// in wave order (64 splits of 64 rows: 54 us with one wave and a weight at a time).
template <int DT, int D, int WAVES_ROW>
__global__ __launch_bounds__(256) void attention_join(const Args a) {
  constexpr int E = D / 64, ROWS = 4 / WAVES_ROW, BATCH = WAVES_ROW == 1 ? 4 : 16;
  __shared__ float sums[WAVES_ROW == 1 ? 1 : 4][D];
  const int64_t rows = int64_t{a.tokens} * a.heads;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t at = int64_t{blockIdx.x} * ROWS + wave / WAVES_ROW;
  if (at >= rows) return;  // whole workgroups where waves share a row
  float m = M_FLOOR, l = 0.0f;
  if (lane < a.splits) {
    const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[lane * rows + at];
    m = ml.x;
    l = ml.y;
  }
  float top = m;
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float w = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((m - top) * launch_unit(a));
  const uint64_t saw = __builtin_amdgcn_ballot_w64(l != 0.0f || m != M_FLOOR);  // splits that wrote sums
  const bool lost = __builtin_amdgcn_ballot_w64(m < M_FLOOR) != 0;
  const float total = wave_sum(l * w);
  const int per = (a.splits + WAVES_ROW - 1) / WAVES_ROW, s0 = wave % WAVES_ROW * per, s1 = min(s0 + per, a.splits);
  float acc[E];
  auto add_up = [&](auto with_care) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    for (int s = s0; s < s1; s += BATCH) {
      float v[BATCH][E];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float* src = a.part_o + (min(s + i, s1 - 1) * rows + at) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] = src[e];
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        // A split that saw nothing wrote no sums: whatever lies there is left out.
        const int from = min(s + i, s1 - 1);
        const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), from));
        const bool take = s + i < s1 && ((saw >> from) & 1);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float next =
              decltype(with_care)::value ? add_scaled(acc[e], v[i][e], f) : __builtin_fmaf(v[i][e], f, acc[e]);
          acc[e] = take ? next : acc[e];
        }
      }
    }
  };
  add_up(std::false_type{});
  float check = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) check = __builtin_fmaf(acc[e], 0.0f, check);
  if (__builtin_amdgcn_ballot_w64(check != 0.0f)) add_up(std::true_type{});  // rare: a sum is not finite
  if constexpr (WAVES_ROW > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sums[wave][lane * E + e] = acc[e];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[e] = sums[0][lane * E + e];
#pragma unroll
      for (int i = 1; i < 4; ++i) acc[e] += sums[i][lane * E + e];
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total, none = lost ? __builtin_nanf("") : 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = total == 0.0f ? none : acc[e] * inv;
  uint16_t* dst = a.out + at * D + lane * E;
  if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = pack2<DT>(acc[0], acc[1]);
  else *dst = static_cast<uint16_t>(pack2<DT>(acc[0], 0.0f) & 0xFFFFu);
}

// How a call is launched.  `few`: sequences of no more than 32 packed rows on average that are fewer, with their key
// heads, than the workgroups that run at once; or fewer tiles of 128 rows than compute units, where 32-row workgroups
// fill them better (two run on one at once), the keys are not so many that the other form's key splits cost nothing
// beside them, and not so few that a second round of workgroups costs more than it brings.  With tiles of 128 rows and
// with `few`: 128 tokens, 56 heads of 128: 8.7 and 6.5 us; 300 tokens: 12.8 and 15.8; 1024 tokens, 16 heads: 33.8 and
// 18.0; 1999 tokens, 4 key heads of 64, prefix and cap: 43.8 and 32.2; 9914 tokens, one head: 71 and 98.
//
// The first limit is no crossing of the forms.  Single tokens of 8 key heads of 128, with tiles and with `few`, over
// 300 / 1000 / 4000 keys each: 32 sequences 14, 13 / 29, 28 / 98, 98 us; 63: 20, 17 / 45, 42 / 177, 176; 64: 20, 18 /
// 46, 44 / 182, 180; 65: 26, 21 / 63, 50 / 248, 209; 128: 34, 31 / 99, 95 / 355, 352; 256: 68, 62 / 191, 184.  Two key
// heads, 256 sequences: 20, 21 / 46, 48 / 183, 205; 400: 30, 27 / 82, 82 / 289, 304.  64 of unequal lengths up to 8190,
// evenly spread: 161, 170; at random: 228, 236 and 208, 201; spread over the logarithm: 146, 105; 65 of these: 148, 97.
// Beyond the limit `few` is mostly the better one, by up to a third; tiles are where lengths are spread evenly, and
// where few key heads just fill the chip.  The limit has not been moved to what these say.
struct Plan {
  bool few;
  int slots;
};
inline Plan plan(bool paged, int64_t tokens, int group, int kv_heads, int64_t sequences, int64_t keys, int cus) {
  const int64_t rows = tokens * group, own = paged ? sequences : 1;
  const int64_t tiles = (rows / (32 * WAVES) + own) * kv_heads, thin = (rows / 32 + own) * kv_heads;
  const bool few = (rows <= 32 * own && own * kv_heads < 2 * cus) ||
                   (tiles < cus && thin <= (keys < 512 ? 2 : 4) * cus && keys <= 4096);
  const int64_t r = few ? 32 : 32 * WAVES;
  return Plan{few, static_cast<int>(paged ? rows / r + sequences + 1 : (rows + r - 1) / r)};
}

// Key splits: as many as bring the workgroups to two a compute unit, what it holds at once, each over at least 256 keys
// of the longest span; twice as many were slower (2048 tokens, 8 heads: 22 and 36 us).  Full workgroups of `few` to
// one: their waves split the keys already, and the sums of 32 rows cost as much as their keys (2000 tokens, 4 query
// heads on one key head, 250 workgroups: 19 us, 26 us in two splits).
inline int plan_splits(bool paged, int64_t tokens, int group, int kv_heads, int64_t sequences, int64_t keys,
                       int cus) {
  const Plan p = plan(paged, tokens, group, kv_heads, sequences, keys, cus);
  // Slots that have rows: of a paged launch about half a tile a sequence on top of the whole ones.
  const int64_t r = p.few ? 32 : 32 * WAVES, whole = tokens * group / r, own = tokens < sequences ? tokens : sequences;
  const int64_t tiles = !paged ? p.slots : whole + own / 2 > own ? whole + own / 2 : own;
  const int64_t busy = (tiles > 0 ? tiles : 1) * kv_heads;
  const bool full = p.few && tokens * group > 32 * (paged ? sequences : 1);
  int64_t n = (full ? 1 : 2) * int64_t{cus} / busy;
  const int64_t most = keys / 256;
  n = n < most ? n : most;
  return static_cast<int>(n < 1 ? 1 : n > 64 ? 64 : n);
}

template <int DT, int D, int KEYS>
int launch(Args& a, hipStream_t st) {
  const bool mods = a.softcap > 0.0f || a.slopes;
  const Plan p = plan(KEYS != DENSE, a.tokens, a.group, a.kv_heads, a.sequences, a.keys, device_cus());
  a.slots = p.slots;
  a.cus = device_cus();
  a.spread = a.kv_heads % 8 != 0 && (KEYS != DENSE || a.causal || a.starts);
  const int64_t blocks = int64_t{a.slots} * a.kv_heads * a.splits;
  M5K_REQUIRE(blocks <= INT32_MAX, "attention: too many tiles for one launch");
  auto kernel = p.few ? (mods ? attention_tile<DT, D, KEYS, true, true> : attention_tile<DT, D, KEYS, false, true>)
                      : (mods ? attention_tile<DT, D, KEYS, true, false> : attention_tile<DT, D, KEYS, false, false>);
  launch_kernel(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(THREADS), st, a);
  int rc = launch_status("attention");
  if (rc != M5K_OK || a.splits == 1) return rc;
  const int64_t rows = int64_t{a.tokens} * a.heads;
  if (a.splits > 8)
    launch_kernel(attention_join<DT, D, 4>, dim3(static_cast<uint32_t>(rows)), dim3(256), st, a);
  else
    launch_kernel(attention_join<DT, D, 1>, dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), st, a);
  return launch_status("attention join");
}

template <int KEYS>
int launch_typed(Args& a, int dtype, int head_dim, hipStream_t st) {
  if (dtype == M5K_BF16)
    return head_dim == 64 ? launch<M5K_BF16, 64, KEYS>(a, st) : launch<M5K_BF16, 128, KEYS>(a, st);
  return head_dim == 64 ? launch<M5K_F16, 64, KEYS>(a, st) : launch<M5K_F16, 128, KEYS>(a, st);
}

inline void magic_of(uint32_t d, uint32_t& magic, uint32_t& shift) {
  shift = 0;
  while ((uint64_t{1} << shift) < d) ++shift;
  magic = static_cast<uint32_t>(((uint64_t{1} << (31 + shift)) + d - 1) / d);
}

}  // namespace attn
}  // namespace m5k
