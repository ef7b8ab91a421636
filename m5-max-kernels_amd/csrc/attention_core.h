// Attention for gfx950: out = softmax(scores(Q K^T) + mask) V with one pass over the keys, K and V dense or in
// the pages of a cache, in 16 bits or as codes of 8 bits.
//
// Rows.  The query heads that share a key head are packed: packed row r of a sequence is token r / G, query head
// kvh * G + r % G (G = heads / kv_heads), so one K/V tile serves all of them and a single token still fills G rows.
// A workgroup has 4 waves of 32 rows; a wave keeps its Q in registers.
//
// Masks.  Every mask of these operators (causal, window, document, prefix, length) leaves a row one interval
// [lo, hi) of keys.  Key tiles outside the union of a wave's intervals are skipped, tiles inside all of them need
// no comparison, the others compare the key index.  A window that keeps a sequence's first keys (SINKS) leaves a row
// two intervals: tiles of the first keys are taken ahead of those of the windows, by the same loop, and where either
// ends inside a tile the lane's keys are bits of a word.
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
// Codes: bytes again where tokens are single (131073 keys, E4M3: 54 us, 5.0 TB/s, and 5 of joining; 64 over 4000 keys
// each 103 us, 5.1 TB/s); 64 over 0 to 6122 keys, in three bands, take 102 to 109 us in INT8 and 91 to 94 in E4M3, 3.8
// and 4.3 TB/s, the longest sequences alone at the end; 64 with lengths spread over the logarithm from 32 to 8191 71 to
// 97 us in E4M3 and 98 to 135 in INT8, where their bytes take 32 to 58.  Chunks as in 16 bits, with the expansion
// beside the products (of up to 1024 tokens over up to 8192 keys 207 us, so 182; 0.9 waves a SIMD, and one alone takes
// 3800 cycles a tile where two take 2600 each).
// First keys: 9914 causal tokens, 56 heads of 128, window 1024, 4 first keys: 363 to 373 us, 0.85 PFLOP/s over the 1090
// keys a row that are multiplied, of which 975 count; without first keys 343.  19 tiles a workgroup leave its beginning
// and end more to hide than the 155 of a call without a window.  8192 tokens in 7 documents, 32 on 8 heads of 64, FP16,
// window 256, 64 first keys: 54 to 60 us, 7 tiles a workgroup; nothing is full there (VALU 46% of the cycles, matrix
// cores 16%, 1.5 waves a SIMD, which wait for 29%).
//
// Registers.  Tiles of 128 rows with heads of 128 use 241 to 256, all there are for two waves a SIMD.  With a cap or a
// bias 8 to 10 of them go to memory and come back inside the loop, 34 by pages of no multiple of 16 (chunks of up to
// 1024 tokens over up to 8192 keys, bias: 232 us in pages of 64, 536 in pages of 24; without the bias 182 and 251).
// Codes: 7 to 22, with cap or bias 40 to 54, where the form of few rows is mostly taken instead (none spilled there).
#pragma once

#include "attention_place.h"
#include "fast_div.h"
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
  int sinks;
  int64_t reach;  // keys that a row can see, for the plan
  // Codes: exponent bytes of each block of tokens, strides in bytes.
  const uint8_t *k_exp, *v_exp;
  int64_t ke_page, ke_head, ve_page, ve_head;
  uint32_t block_magic, block_shift;
};

template <int DT>
__device__ __forceinline__ v16f mfma32(v4i a, v4i b, v16f c) {
  if constexpr (DT == M5K_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(gemm::bf16x8, a),
                                                   __builtin_bit_cast(gemm::bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(gemm::f16x8, a),
                                                  __builtin_bit_cast(gemm::f16x8, b), c, 0, 0, 0);
}

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// Two values to the inputs' type, to the nearest, by one instruction.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == M5K_BF16) return f32x2_to_bf16x2(lo, hi);
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((m5k_f32x2{lo, hi}), half2v));
}

// Two finished values to the inputs' type: in FP16 by a conversion each, which the compiler makes one instruction, and
// one rounding, with the division of the sum before it.
template <int DT>
__device__ __forceinline__ uint32_t out2(float lo, float hi) {
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
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i* lds_v2i;

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

// The same for a tile of codes, rows of D bytes: the 16 rows of a ds_read_b128 phase (K) fall on 16 bank groups, and so
// do the 8 rows x 32 bytes of half a wave's transposed read (V), rows 0 .. 3 and 8 .. 11, or 4 .. 7 and 12 .. 15, whose
// pairs of chunks therefore differ in a bit above the lowest.
template <int D>
__device__ __forceinline__ int code_swizzle(int row) {
  if constexpr (D == 64) return (row >> 2) & 3;
  else return (((row >> 3) & 1) << 2) | (((row >> 1) & 1) << 1) | ((row >> 2) & 1);
}

// Where keys and values lie.  PAGES16: pages of a multiple of 16 keys, so that the 16 rows of a tile that one wave
// loads lie in one page and take one address; PAGES: any page size, an address a lane.
enum Keys { DENSE = 0, PAGES16 = 1, PAGES = 2 };

// What a cache holds: 16-bit values, or codes of 8 bits under a block's power of two.
enum Codes { NO_CODES = 0, E4M3 = 1, INT8 = 2 };

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
template <int D, class Elem>
__device__ __forceinline__ v4i rows_rsrc(const Elem* p, int rows, int64_t stride) {
  const int64_t n = rows > 0 ? ((rows - 1) * stride + D) * static_cast<int64_t>(sizeof(Elem)) : 0;
  return gemm::buffer_rsrc(p, static_cast<uint32_t>(n));
}

constexpr int NEVER = 0x3FFFFFFF;  // behind every key

// A block's scale, 2^(e - 127), as code_pair takes it.  E4M3: e in FP32's exponent field, which is all that its
// conversion reads.  INT8: the number, which for e = 0 has no exponent field of its own; NaN for e = 255.
template <int CODES>
__device__ __forceinline__ float code_scale(int e) {
  uint32_t bits = static_cast<uint32_t>(e) << 23;
  if constexpr (CODES == INT8) bits = e == 0 ? 0x00400000u : e == 255 ? 0x7FC00000u : bits;
  return __uint_as_float(bits);
}

// Two codes, bytes 2 HI and 2 HI + 1 of a word, times their scale, as 16-bit values.  Exact in BF16, which has more
// bits than a code and FP32's range; rounded once to FP16, which only numbers below 2^-14 need.  E4M3: one conversion,
// whose results are those of an FP32 product rounded to the type, for every code and exponent (compared on MI355X).
template <int DT, int CODES, bool HI>
__device__ __forceinline__ uint32_t code_pair(int w, float scale) {
  if constexpr (CODES == E4M3 && DT == M5K_BF16) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  } else if constexpr (CODES == E4M3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  } else if constexpr (DT == M5K_BF16) {
    const int w0 = HI ? w << 8 : w << 24, w1 = HI ? w : w << 16;
    return pack2<DT>(static_cast<float>(w0 >> 24) * scale, static_cast<float>(w1 >> 24) * scale);
  } else {
    // 1024 + (code + 128) is an FP16 number with the code's bits in its mantissa; the product is FP32's, rounded once.
    const uint32_t biased = static_cast<uint32_t>(w) ^ 0x80808080u;
    const uint32_t bits = __builtin_amdgcn_perm(0x64646464u, biased, HI ? 0x07030702u : 0x07010700u);
    const half2v c = __builtin_bit_cast(half2v, bits) - half2v{1152.0f16, 1152.0f16};
    const half2v r = {static_cast<_Float16>(__builtin_fmaf(static_cast<float>(c[0]), scale, 0.0f)),
                      static_cast<_Float16>(__builtin_fmaf(static_cast<float>(c[1]), scale, 0.0f))};
    return __builtin_bit_cast(uint32_t, r);
  }
}

// 8 and 16 codes times their scale, in order, as 16-bit values.
template <int DT, int CODES>
__device__ __forceinline__ v4i expand8(int w0, int w1, float scale) {
  return v4i{static_cast<int>(code_pair<DT, CODES, false>(w0, scale)),
             static_cast<int>(code_pair<DT, CODES, true>(w0, scale)),
             static_cast<int>(code_pair<DT, CODES, false>(w1, scale)),
             static_cast<int>(code_pair<DT, CODES, true>(w1, scale))};
}
template <int DT, int CODES>
__device__ __forceinline__ void expand16(v4i c, float scale, v4i (&x)[2]) {
  x[0] = expand8<DT, CODES>(c[0], c[1], scale);
  x[1] = expand8<DT, CODES>(c[2], c[3], scale);
}

struct RowRange {
  int lo, hi;  // visible keys; lo > hi where there are none
  int pos;     // position on the key axis, for the distance bias
  int slo, shi;  // SINKS: further visible keys, before lo; slo > shi where there are none
};

// The interval of a row at position p of a span [s, e) of keys, and with SINKS the span's first keys where the window
// has left them behind.
template <bool SINKS>
__device__ __forceinline__ RowRange row_range(int s, int e, int p, int prefix, int causal, int window, int sinks) {
  int lo = s, hi = e, slo = NEVER, shi = 0;
  if (causal) hi = min(e, max(p + 1, s + prefix));
  const int kept = min(hi, s + sinks);
  if (window) {
    lo = max(lo, p - window + 1);
    if (!causal) hi = min(hi, p + window);
  }
  if constexpr (SINKS) {
    if (hi <= lo) {
      lo = s;
      hi = kept;
    } else if (kept >= lo) {
      lo = s;
      hi = max(hi, kept);
    } else if (kept > s) {
      slo = s;
      shi = kept;
    }
  }
  if (hi <= lo) { lo = NEVER; hi = 0; }
  return RowRange{lo, hi, p, slo, shi};
}

// Bits 0 .. n - 1 of a word.
__device__ __forceinline__ uint32_t bits_below(int n) {
  return n <= 0 ? 0u : 0xFFFFFFFFu >> (32 - min(n, 32));
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

// Minimum and maximum over the wave: lane movement within the rows of 16, then four scalars.  (By five shuffles through
// LDS each, the four or seven of a workgroup's beginning cost it half a microsecond.)
template <int CTRL>
__device__ __forceinline__ int moved(int v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ int wave_min_i(int v) {
  v = min(v, moved<0xB1>(v));   // quad_perm [1,0,3,2]
  v = min(v, moved<0x4E>(v));   // quad_perm [2,3,0,1]
  v = min(v, moved<0x141>(v));  // row_half_mirror
  v = min(v, moved<0x140>(v));  // row_mirror
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_max_i(int v) { return -wave_min_i(-v); }

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
template <int KEYS, bool SINKS>
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
  prefix = min(max(prefix, 0), NEVER);
  return row_range<SINKS>(s, e, i + p.shift, prefix, a.causal, a.window, a.sinks);
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
//
// SINKS: rows see their span's first keys beside their window.  The workgroup's tiles are those of the first keys, then
// those of the windows: `t` counts them, real(t) is where tile t lies.
//
// CODES: K and V are codes of 8 bits with an exponent byte a block of tokens.  They go to LDS as they are.  With FEW
// the products' fragments are made from them as they are read: two tiles of each operand then take less LDS than one of
// 16 bits, and no code is read twice (131073 keys, 8 key heads of 128, E4M3: by way of a 16-bit tile 105 us, so 64).
// Otherwise they go, times their scale, to the tile of 16-bit values that the products read: by the wave that loaded
// them, so that no barrier stands between and each code is expanded once a workgroup, not once a wave, in steps beside
// the products (chunks of up to 1024 tokens over up to 8192 keys: ahead of them 246 us, so 207; 16-bit values 182).
template <int DT, int D, int KEYS, bool MODS, bool FEW, bool SINKS, int CODES>
__global__ __launch_bounds__(THREADS, 2) void attention_tile(const Args a) {
  static_assert(CODES == NO_CODES || KEYS == PAGES16, "codes lie in pages of a multiple of 16");
  constexpr int KT = FEW ? 32 : 64, NB = KT / 32;  // keys of a tile, 32-key blocks
  constexpr int EL = 16 * NB;                      // scores of a lane
  constexpr int CH = CODES ? D / 16 : D / 8;       // 16-byte chunks of a row, as it lies in memory
  constexpr int RPI = 64 / CH;                     // rows of one load instruction
  constexpr int LOADED = FEW ? KT : KT / WAVES;    // rows of a tile that one wave loads
  constexpr int GROUPS = LOADED / 16;
  constexpr int NI = LOADED / RPI;  // its load instructions, each of K and V
  constexpr int QS = D / 16, OB = D / 32;
  constexpr int AHEAD = 1;  // steps of two products between a fragment's read and its use (2: no faster)
  constexpr int ROWS = FEW ? 32 : 32 * WAVES;
  constexpr bool DIRECT = CODES != NO_CODES && FEW;  // fragments from codes
  constexpr int STAGES = FEW && !DIRECT && !(KEYS == PAGES && D == 64) ? 1 : 2;  // tiles of K, and of V, in LDS
  constexpr uint32_t ROWB = DIRECT ? D : D * 2, TILE = KT * ROWB, VTILE = STAGES * TILE;
  // K stages, V stages.  FEW: those of each wave, later its sums, in rows of D + 4 floats (16 bytes a lane without bank
  // conflicts), and their maxima and totals.
  // CODES, not FEW: behind them a wave's codes of one tile of K and one of V.
  constexpr uint32_t RAW = CODES && !FEW ? LOADED * D : 0;
  constexpr uint32_t SUMS = (D + 4) * 4, JOIN = 32 * SUMS + 256, AREA = JOIN > 2 * VTILE ? JOIN : 2 * VTILE;
  __shared__ __attribute__((aligned(256))) uint8_t lds[FEW ? WAVES * AREA : 4 * TILE + 2 * WAVES * RAW];
  // Bounds of the waves' rows.  CODES: where the codes come later, since two workgroups' LDS fills the compute unit.
  __shared__ int bounds_own[FEW || CODES ? 1 : SINKS ? 5 * WAVES : 2 * WAVES];
  int* const bounds = CODES ? reinterpret_cast<int*>(lds) : bounds_own;

  const Place p = place<KEYS>(a, ROWS);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  if (!tile_has_rows(p.tile, p.rows, ROWS)) return;
  const int row0 = p.tile * ROWS;
  const int row = row0 + (FEW ? 0 : 32 * wave) + (lane & 31);
  const bool live = row < p.rows;
  int token, head;
  const RowRange rr = range_of<KEYS, SINKS>(a, p, min(row, p.rows - 1), token, head);

  v4i qf[QS];
  {
    const uint16_t* qp = a.q + int64_t{head} * a.q_head + int64_t{token} * a.q_token + 8 * half;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      // DIRECT: the channel order of K's fragments, two from the 16 codes of one read.
      const int channel = DIRECT ? 32 * (s >> 1) + 8 * half + 8 * (s & 1) : 16 * s;
      qf[s] = *reinterpret_cast<const v4i*>(qp + channel);
    }
  }
  // Key ranges: of the wave (any row, every row), and of the workgroup.
  const bool idle = !FEW && row0 + 32 * wave >= p.rows;
  int any_lo = idle ? NEVER : wave_min_i(rr.lo);
  const int any_hi = idle ? 0 : wave_max_i(rr.hi);
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
  // First keys that lie before the windows of all rows have tiles of their own, `kept` of them from `kept_tile` on; the
  // others (of documents that begin inside the workgroup's rows) are taken with the windows.
  int kept = 0, kept_tile = 0;
  bool with_window = true;
  if constexpr (SINKS) {
    with_window = rr.shi > lo / KT * KT;
    const bool has = rr.slo < rr.shi && !idle;
    any_lo = wave_min_i(has && with_window ? min(rr.lo, rr.slo) : idle ? NEVER : rr.lo);
    const int own_lo = wave_min_i(has && !with_window ? rr.slo : NEVER);
    int s_lo = own_lo, s_hi = wave_max_i(has && !with_window ? rr.shi : 0);
    lo = any_lo;
    if constexpr (!FEW) {
      if (lane == 0) {
        bounds[2 * WAVES + wave] = any_lo;
        bounds[3 * WAVES + wave] = s_lo;
        bounds[4 * WAVES + wave] = s_hi;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        lo = min(lo, bounds[2 * WAVES + w]);
        s_lo = min(s_lo, bounds[3 * WAVES + w]);
        s_hi = max(s_hi, bounds[4 * WAVES + w]);
      }
      lo = __builtin_amdgcn_readfirstlane(lo);
      s_lo = __builtin_amdgcn_readfirstlane(s_lo);
      s_hi = __builtin_amdgcn_readfirstlane(s_hi);
    }
    if (s_lo < s_hi) {
      kept_tile = s_lo / KT;
      kept = (s_hi + KT - 1) / KT - kept_tile;
      if (kept_tile + kept > lo / KT) {  // one stretch of tiles after all
        kept = 0;
        lo = min(lo, s_lo);
        any_lo = min(any_lo, own_lo);
        with_window = true;
      }
    }
  }
  if constexpr (CODES && !FEW) __syncthreads();  // the bounds have been read
  // Tile t lies at real(t), and a window's tile T is tile t = T - ahead.
  const int window_tile = SINKS ? lo / KT : 0, ahead = window_tile - kept;
  auto real = [&](int t) __attribute__((always_inline)) {
    if constexpr (SINKS) return t < kept ? kept_tile + t : t + ahead;
    else return t;
  };
  int t_begin = 0, t_end = 0;
  if (lo < hi) {
    t_begin = SINKS ? 0 : lo / KT;
    t_end = (hi + KT - 1) / KT - (SINKS ? ahead : 0);
    if (a.splits > 1) {
      // At least 256 keys a split: below, the partial sums cost more than the keys.
      const int per = max((t_end - t_begin + a.splits - 1) / a.splits, 256 / KT);
      t_begin = min(t_begin + p.split * per, t_end);
      t_end = min(t_begin + per, t_end);
    }
  }

  const float scale2 = a.scale * LOG2E;
  const float unit = MODS ? 1.0f : scale2;  // what turns finished scores into base 2, launch_unit()
  const float slope2 = MODS && a.slopes ? a.slopes[head] * LOG2E : 0.0f;

  // Loads: instruction i of a wave brings rows first_row + i * RPI + lane / CH of K and of V.
  const int first_row = FEW ? 0 : wave_s * LOADED;
  const int ld_row = first_row + lane / CH, ld_chunk = lane % CH;
  using Elem = std::conditional_t<CODES != NO_CODES, uint8_t, uint16_t>;
  const Elem* kbase = reinterpret_cast<const Elem*>(a.k) + int64_t{p.kvh} * a.k_head;
  const Elem* vbase = reinterpret_cast<const Elem*>(a.v) + int64_t{p.kvh} * a.v_head;
  const uint8_t* kexp = CODES ? a.k_exp + int64_t{p.kvh} * a.ke_head : nullptr;
  const uint8_t* vexp = CODES ? a.v_exp + int64_t{p.kvh} * a.ve_head : nullptr;
  const int32_t* table = KEYS != DENSE && p.seq < a.sequences ? a.table + int64_t{p.seq} * a.table_width : nullptr;
  const uint32_t lds0 = gemm::lds_addr(lds) + (FEW ? wave_s * AREA : 0);
  uint32_t kofs[NI], vofs[NI];  // bytes of a lane's chunk from the window's first row
  if constexpr (KEYS != PAGES) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = KEYS == DENSE ? ld_row + i * RPI : lane / CH + i % (NI / GROUPS) * RPI;  // pages: of 16 rows
      const int chunk = DIRECT  ? (ld_chunk ^ code_swizzle<D>(ld_row + i * RPI)) * 16
                        : CODES ? ld_chunk * 16
                                : (ld_chunk ^ swizzle<D>(ld_row + i * RPI)) * 8;
      kofs[i] = static_cast<uint32_t>(r * static_cast<int>(a.k_row) + chunk) * sizeof(Elem);
      vofs[i] = static_cast<uint32_t>(r * static_cast<int>(a.v_row) + chunk) * sizeof(Elem);
    }
  }
  constexpr int NIDS = KEYS == PAGES ? NI : GROUPS;
  int ids[2][NIDS] = {};  // pages of the next tile's keys, and of the tile before it, whose values come next
  int ek[STAGES][GROUPS] = {}, ev[STAGES][GROUPS] = {};  // CODES: exponents of the codes on their way
  bool lacking = false;

  // Unconditional, at the last key where tile t has none: a load under a condition would be waited for at the
  // condition's end, and with it everything in flight.
  auto load_ids = [&](int t, int (&to)[NIDS]) __attribute__((always_inline)) {
    if constexpr (KEYS == PAGES16) {
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        const int key = min(real(t) * KT + first_row + 16 * i, p.span - 1);
        to[i] = table_entry<FEW>(table, fast_div(key, a.page_magic, a.page_shift));
      }
    } else if constexpr (KEYS == PAGES) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int key = min(real(t) * KT + ld_row + i * RPI, p.span - 1);
        to[i] = table[fast_div(key, a.page_magic, a.page_shift)];
      }
    }
  };
  // This wave's rows of tile t of one operand to LDS at dst.
  auto load_rows = [&](int u, const int (&id)[NIDS], const Elem* base, int64_t page_stride, int64_t row_stride,
                       const uint32_t (&ofs)[NI], uint32_t dst) __attribute__((always_inline)) {
    const int t = real(u);
    dst += FEW || CODES ? 0 : wave_s * NI * 1024;
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
        const Elem* at = base;
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

  // CODES: the exponent of a key's block on page `id`, 0 where there is none.
  auto exponent_of = [&](int key, int id, const uint8_t* base, int64_t page_stride) __attribute__((always_inline)) {
    const int slot = key - static_cast<int>(fast_div(key, a.page_magic, a.page_shift)) * a.page_size;
    const bool has = key < p.span && static_cast<uint32_t>(id) < static_cast<uint32_t>(a.pages);
    const int e = base[has ? id * page_stride + fast_div(slot, a.block_magic, a.block_shift) : 0];
    return has ? e : 0;
  };
  // Pages and exponents of the tiles that this wave loads from tile t on, a group of 16 keys a lane, by vector loads
  // that it waits for once in 32 tiles (FEW) or 64.  Loads a tile would be waited for with the tiles in flight, or, as
  // scalar loads, hold up the LDS reads behind them (64 single tokens over 0 to 6122 keys, INT8: 130 us and 120).
  constexpr int HELD = 64 / GROUPS, APART = FEW ? WAVES : 1;
  int held_id = 0, held_k = 0, held_v = 0, held_at = 0;
  auto look_ahead = [&](int t) __attribute__((always_inline)) {
    if constexpr (CODES) {
      const int key = real(t + APART * (lane / GROUPS)) * KT + first_row + 16 * (lane % GROUPS);
      held_id = table[fast_div(min(key, p.span - 1), a.page_magic, a.page_shift)];
      held_k = exponent_of(key, held_id, kexp, a.ke_page);
      held_v = exponent_of(key, held_id, vexp, a.ve_page);
      held_at = 0;
    }
  };
  auto take_ids = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NIDS; ++g) ids[0][g] = __builtin_amdgcn_readlane(held_id, GROUPS * held_at + g);
  };
  auto take_exps = [&](int (&k)[GROUPS], int (&v)[GROUPS]) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      k[g] = __builtin_amdgcn_readlane(held_k, GROUPS * held_at + g);
      v[g] = __builtin_amdgcn_readlane(held_v, GROUPS * held_at + g);
    }
    ++held_at;
  };
  // The next tile's, from tile t's lookup if the last one is used up.
  auto take_next = [&](int t, int (&k)[GROUPS], int (&v)[GROUPS]) __attribute__((always_inline)) {
    if (held_at == HELD) {
      look_ahead(t);
      __asm__ volatile("" : "+v"(held_id), "+v"(held_k), "+v"(held_v));  // waited for here, not in every round
    }
    take_ids();
    take_exps(k, v);
  };
  const uint32_t raw_k = lds0 + 4 * TILE + wave_s * 2 * RAW, raw_v = raw_k + RAW;
  // This wave's codes at `raw`, times their scale, to its rows of the 16-bit tile at `dst`: step `part` of PARTS, four
  // for each 16 codes of a lane.
  constexpr int PARTS = 4 * NI;
  v4i taken;
  auto expand = [&](uint32_t raw, int exponent, uint32_t dst, int part) __attribute__((always_inline)) {
    if constexpr (CODES && !FEW) {
      const int i = part >> 2, r = ld_row + i * RPI;
      const uint32_t at = dst + r * ROWB + (((2 * ld_chunk) ^ swizzle<D>(r)) << 4);
      if ((part & 3) == 0)
        taken = *reinterpret_cast<const __attribute__((address_space(3))) v4i*>(raw + i * 1024 + lane * 16);
      if (part & 2) {
        const int h = part & 1;
        *reinterpret_cast<__attribute__((address_space(3))) v4i*>(at ^ (h << 4)) =
            expand8<DT, CODES>(taken[2 * h], taken[2 * h + 1], code_scale<CODES>(exponent));
      }
    }
  };
  auto expand_all = [&](uint32_t raw, int exponent, uint32_t dst) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) expand(raw, exponent, dst, i);
  };

  // Fragment addresses in stage 0 (the other stage and the rows further on are instruction offsets): chunk c of a row
  // is its chunk 0 XOR 16 c, rows being aligned to their size.
  constexpr int KREADS = DIRECT ? QS / 2 : QS, VREADS = DIRECT ? 1 : 2;
  uint32_t kread[KREADS], vread[VREADS][OB];
  const int g = lane >> 4, gi = lane & 15;
  const int vrow = 4 * half + (gi >> 2), vchunk = 2 * (g & 1) + ((gi & 3) >> 1);
  const int ksw = DIRECT ? code_swizzle<D>(lane & 31) : swizzle<D>(lane & 31);
#pragma unroll
  for (int c = 0; c < KREADS; ++c) kread[c] = (lds0 + (lane & 31) * ROWB + ((half ^ ksw) << 4)) ^ (c << 5);
  if constexpr (DIRECT) {
    // The 8 keys of a fragment in the accumulator's order, two lanes a key.
    const int key = 8 * (gi >> 3) + 4 * half + ((gi >> 1) & 3);
#pragma unroll
    for (int b = 0; b < OB; ++b)
      vread[0][b] = (lds0 + key * ROWB + (((g & 1) ^ code_swizzle<D>(key)) << 4) + (gi & 1) * 8) ^ (b << 5);
  } else {
#pragma unroll
    for (int h = 0; h < VREADS; ++h)
#pragma unroll
      for (int b = 0; b < OB; ++b)
        vread[h][b] =
            (lds0 + (8 * h + vrow) * ROWB + ((vchunk ^ swizzle<D>(8 * h + vrow)) << 4) + (gi & 1) * 8) ^ (b << 6);
  }

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
  // V^T fragment of k-step c and channel block b: keys 16 c + 8 h + 4 (lane >> 5) .. + 3 for h = 0, 1.  DIRECT: its
  // codes, which value_of makes a fragment of.
  auto value_frag = [&](int st, int c, int b) __attribute__((always_inline)) {
    v4i f{};
    if constexpr (DIRECT) {
      const v2i x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          reinterpret_cast<lds_v2i>(vread[0][b] + 16 * c * ROWB + VTILE + st * TILE));
      f[0] = x[0];
      f[1] = x[1];
      return f;
    }
#pragma unroll
    for (int h = 0; h < VREADS; ++h) {
      const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          reinterpret_cast<lds_v4s>(vread[h][b] + 16 * c * ROWB + VTILE + st * TILE));
      const auto y = __builtin_bit_cast(m5k_u32x2, x);
      f[2 * h] = static_cast<int>(y[0]);
      f[2 * h + 1] = static_cast<int>(y[1]);
    }
    return f;
  };
  auto value_of = [&](v4i f, int st, int c) __attribute__((always_inline)) {
    if constexpr (DIRECT) return expand8<DT, CODES>(f[0], f[1], code_scale<CODES>(ev[st][c]));
    else return f;
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
  // side(i): what else step i does.
  auto nothing = [](int) {};
  auto product = [&](v16f (&y)[NB], int st, const v16f (&x)[NB], bool prob, auto side) __attribute__((always_inline)) {
    if constexpr (DIRECT) {
      // Rows 0 .. 15 and 16 .. 31 of the tile are two groups.
      int e0 = ek[st][0], e1 = ek[st][GROUPS - 1];
      __asm__("" : "+s"(e0), "+s"(e1));  // values, not two places to choose from: those would go to memory
      const float scale = code_scale<CODES>((lane & 16) ? e1 : e0);
      v4i code[2];
      auto read = [&](int c) __attribute__((always_inline)) {
        return *reinterpret_cast<const __attribute__((address_space(3))) v4i*>(kread[c] + st * TILE);
      };
      code[0] = read(0);
#pragma unroll
      for (int c = 0; c < KREADS; ++c) {
        if (c + 1 < KREADS) code[(c + 1) & 1] = read(c + 1);
        v4i f[2];
        expand16<DT, CODES>(code[c & 1], scale, f);
        y[0] = mfma32<DT>(f[0], qf[2 * c], c == 0 ? v16f{} : y[0]);
        y[0] = mfma32<DT>(f[1], qf[2 * c + 1], y[0]);
      }
      return;
    }
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
      side(c);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (prob) l += sum[0] + sum[1];
  };
  // Cap, bias and mask of tile t's scores.
  auto finish = [&](v16f (&x)[NB], int t, auto with_care, uint32_t& sees_bits) __attribute__((always_inline)) {
    constexpr bool careful = decltype(with_care)::value;
    const int key0 = real(t) * KT, kofs0 = key0 + 4 * half;
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
    if constexpr ((SINKS || CODES) && !careful) {
      if (key0 >= all_lo && key0 + KT <= all_hi) return;
      // The lane's keys of the tile as bits, and two instructions a score.
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int at = kofs0 + 32 * b;
        uint32_t seen = bits_below(rr.hi - at) & ~bits_below(rr.lo - at);
        if constexpr (SINKS) seen |= bits_below(rr.shi - at) & ~bits_below(rr.slo - at);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t keep = __builtin_amdgcn_sbfe(seen, 8 * (r >> 2) + (r & 3), 1);
          x[b][r] = __uint_as_float((keep & __float_as_uint(x[b][r])) | (~keep & 0xFF800000u));
        }
      }
    } else if (careful || key0 < all_lo || key0 + KT > all_hi) {
      const uint32_t width = static_cast<uint32_t>(max(rr.hi - rr.lo, 0));
      const uint32_t first_keys = SINKS ? static_cast<uint32_t>(max(rr.shi - rr.slo, 0)) : 0;
      if constexpr (careful) sees_bits = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kofs0 + 32 * b + 8 * (r >> 2) + (r & 3);
          bool sees = static_cast<uint32_t>(key - rr.lo) < width;
          if constexpr (SINKS) sees |= static_cast<uint32_t>(key - rr.slo) < first_keys;
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
  auto accumulate = [&](int st, const v16f (&x)[NB], auto side) __attribute__((always_inline)) -> float {
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
        o[b] = mfma32<DT>(value_of(vf[i % (AHEAD + 1)][j], st, 2 * i / OB), pf[2 * i / OB], o[b]);
      }
#pragma unroll
      for (int e = i * EL / STEPS; e < (i + 1) * EL / STEPS; e += 2) {
        t0 = fmaxf(t0, x[e >> 4][e & 15]);
        t1 = fmaxf(t1, x[e >> 4][(e & 15) + 1]);
      }
      side(i);
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
        split_nonfinite<DT>(value_of(value_frag(0, c, b), 0, c), clean, mark);
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

  // This wave's tiles.
  const int first = max(t_begin, any_lo / KT - (SINKS ? ahead : 0));
  const int last = min(t_end, (any_hi + KT - 1) / KT - (SINKS ? ahead : 0));
  auto mine = [&](int t) __attribute__((always_inline)) {
    if constexpr (SINKS) return (t >= first && t < last) || (t >= t_begin && t < min(kept, t_end) && !idle);
    else return t >= first && t < last;
  };
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
    if constexpr (CODES) {
      // The codes of V of tile t + 1 are here, those of K of t + 2 may be on their way until the second product.
      if (t + 2 < t_end) gemm::wait_stage<NI>();
      else gemm::wait_stage<0>();
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else {
      wait_all();
    }
    gemm::stage_barrier();
    if constexpr (!CODES) {
      if (t + 1 < t_end) {
        load_rows(t + 1, ids[1], vbase, a.v_page, a.v_row, vofs, lds0 + (2 + ODD) * TILE);
        if (t + 2 < t_end) load_rows(t + 2, ids[0], kbase, a.k_page, a.k_row, kofs, lds0 + EVEN * TILE);
      }
#pragma unroll
      for (int i = 0; i < NIDS; ++i) ids[1][i] = ids[0][i];
      load_ids(t + 3, ids[0]);
    }
    // CODES: V of tile t + 1 is expanded beside the first product and K of t + 2 beside the second; then the next codes
    // of each are loaded.
    auto expand_v = [&](int i) __attribute__((always_inline)) {
      if constexpr (CODES) expand(raw_v, ev[0][0], lds0 + (2 + ODD) * TILE, i);
    };
    auto expand_k = [&](int i) __attribute__((always_inline)) {
      if constexpr (CODES) expand(raw_k, ek[0][0], lds0 + EVEN * TILE, i);
    };
    auto between = [&]() __attribute__((always_inline)) {
      if constexpr (CODES) {
        if (t + 2 < t_end) {
          ev[0][0] = ev[1][0];
          load_rows(t + 2, ids[0], vbase, a.v_page, a.v_row, vofs, raw_v);
          gemm::wait_stage<NI>();
        }
      }
    };
    auto behind = [&]() __attribute__((always_inline)) {
      if constexpr (CODES) {
        if (t + 3 < t_end) {
          take_next(t + 3, ek[0], ev[1]);
          load_rows(t + 3, ids[0], kbase, a.k_page, a.k_row, kofs, raw_k);
        }
      }
    };
    uint32_t none;
    const bool now = mine(t), then = mine(t + 1);  // the same for the whole wave
    if (now && then) {
      product(next, ODD, x, true, expand_v);
      between();
      finish(next, t + 1, quick, none);
      adopt(accumulate(EVEN, next, expand_k), quick);
      behind();
      return;
    }
    if constexpr (CODES) {
#pragma unroll
      for (int i = 0; i < PARTS; ++i) expand_v(i);
      between();
#pragma unroll
      for (int i = 0; i < PARTS; ++i) expand_k(i);
      behind();
    }
    if (then) {
      product(next, ODD, x, false, nothing);
      finish(next, t + 1, quick, none);
      adopt(maximum(next), quick);
    } else if (now) {
      float sum[2] = {};
      probabilities(x, 0, EL, sum, quick);
      l += sum[0] + sum[1];
      accumulate(EVEN, x, nothing);
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
        if constexpr (DIRECT) take_next(t + WAVES, ek[1 - ST], ev[1 - ST]);
        load_rows(t + WAVES, ids[0], kbase, a.k_page, a.k_row, kofs, lds0 + (1 - ST) * TILE);
        load_rows(t + WAVES, ids[0], vbase, a.v_page, a.v_row, vofs, lds0 + VTILE + (1 - ST) * TILE);
        if constexpr (!DIRECT) load_ids(t + 2 * WAVES, ids[0]);
        gemm::wait_stage<2 * NI>();
      } else {
        gemm::wait_stage<0>();
      }
      product(s[0], ST, s[0], false, nothing);
    } else {
      gemm::wait_stage<NI>();  // K, behind which V was issued
      product(s[0], ST, s[0], false, nothing);
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
    accumulate(ST, s[0], nothing);
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
      if constexpr (DIRECT) {
        look_ahead(t);
        take_ids();
      } else {
        load_ids(t, ids[0]);
      }
      load_rows(t, ids[0], kbase, a.k_page, a.k_row, kofs, lds0);
      load_rows(t, ids[0], vbase, a.v_page, a.v_row, vofs, lds0 + VTILE);
      if constexpr (DIRECT) take_exps(ek[0], ev[0]);
      else load_ids(t + WAVES, ids[0]);
    }
    for (; t < t_end; t += STAGES * WAVES) {
      own_tile(t, std::integral_constant<int, 0>{});
      if (STAGES == 2 && t + WAVES < t_end) own_tile(t + WAVES, std::integral_constant<int, STAGES - 1>{});
    }
  } else if (t_begin < t_end) {
    if constexpr (CODES) {
      look_ahead(t_begin);
      take_ids();
      load_rows(t_begin, ids[0], kbase, a.k_page, a.k_row, kofs, raw_k);
      load_rows(t_begin, ids[0], vbase, a.v_page, a.v_row, vofs, raw_v);
      take_exps(ek[0], ev[0]);
      gemm::wait_stage<NI>();
      expand_all(raw_k, ek[0][0], lds0);
      if (t_begin + 1 < t_end) {
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        take_next(t_begin + 1, ek[0], ev[1]);
        load_rows(t_begin + 1, ids[0], kbase, a.k_page, a.k_row, kofs, raw_k);
      }
    } else {
      load_ids(t_begin, ids[1]);
      load_rows(t_begin, ids[1], kbase, a.k_page, a.k_row, kofs, lds0);
      load_ids(t_begin + 1, ids[0]);
    }
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
    auto meets = [&](int from, int to) __attribute__((always_inline)) {
      from = max(t_begin, from);
      to = min(t_end, to);
      return from + (FEW ? (wave - (from - t_begin)) & (WAVES - 1) : 0) < to;
    };
    if constexpr (SINKS) {
      const int shift = with_window ? ahead : kept_tile;
      saw = meets(rr.lo / KT - ahead, (rr.hi + KT - 1) / KT - ahead) ||
            (rr.slo < rr.shi && meets(rr.slo / KT - shift, (rr.shi + KT - 1) / KT - shift));
    } else {
      saw = meets(rr.lo / KT, (rr.hi + KT - 1) / KT);
    }
  }
  const bool far = !MODS && m != M_FLOOR && !(fabsf(m2) < FAR);
  wait_all();
  bool again = lacking || far || check != 0.0f;
  if constexpr (CODES && !FEW) {  // in LDS of its own: the reduction's would be more than two workgroups have
    __syncthreads();
    const bool any = __builtin_amdgcn_ballot_w64(again) != 0;
    if (lane == 0) bounds[wave] = any;
    __syncthreads();
    again = (bounds[0] | bounds[1] | bounds[2] | bounds[3]) != 0;
    if (again) __syncthreads();
  } else {
    again = __syncthreads_or(again);
  }
  if (again) {
    saw = false;
    start();
    for (int t = t_begin; t < t_end; ++t) {
      if (FEW && ((t - t_begin) & (WAVES - 1)) != wave_s) continue;
      if constexpr (CODES) {
        look_ahead(t);
        take_ids();
        take_exps(ek[0], ev[0]);
      } else {
        load_ids(t, ids[0]);
      }
      load_rows(t, ids[0], kbase, a.k_page, a.k_row, kofs, CODES && !FEW ? raw_k : lds0);
      load_rows(t, ids[0], vbase, a.v_page, a.v_row, vofs, CODES && !FEW ? raw_v : lds0 + VTILE);
      wait_all();
      if constexpr (CODES && !FEW) {
        expand_all(raw_k, ek[0][0], lds0);
        expand_all(raw_v, ev[0][0], lds0 + VTILE);
        wait_all();
      }
      if constexpr (!FEW) gemm::stage_barrier();
      if (mine(t)) {
        uint32_t sees;
        product(s[0], 0, s[1], false, nothing);
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
    range_of<KEYS, SINKS>(a, p, row0 + r, t_out, h_out);
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
        v[i] = total == 0.0f ? out2<DT>(none, none) : out2<DT>(acc[e + 2 * i] * inv, acc[e + 2 * i + 1] * inv);
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
  const uint32_t nones = out2<DT>(none, none);
  uint16_t* op = a.out + (int64_t{token} * a.heads + head) * D + 4 * half;
#pragma unroll
  for (int b = 0; b < OB; ++b)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const uint2 w = l == 0.0f ? make_uint2(nones, nones)
                                : make_uint2(out2<DT>(o[b][r] * inv, o[b][r + 1] * inv),
                                             out2<DT>(o[b][r + 2] * inv, o[b][r + 3] * inv));
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
  if constexpr (E == 2) *reinterpret_cast<uint32_t*>(dst) = out2<DT>(acc[0], acc[1]);
  else *dst = static_cast<uint16_t>(out2<DT>(acc[0], 0.0f) & 0xFFFFu);
}

// How a call is launched.  `few`: sequences of no more than 32 packed rows on average that are fewer, with their key
// heads, than the workgroups that run at once; or fewer tiles of 128 rows than compute units, where 32-row workgroups
// fill them better (two run on one at once), the keys are not so many that the other form's key splits cost nothing
// beside them, and not so few that a second round of workgroups costs more than it brings.  With tiles of 128 rows and
// with `few`: 128 tokens, 56 heads of 128: 8.7 and 6.5 us; 300 tokens: 12.8 and 15.8; 1024 tokens, 16 heads: 33.8 and
// 18.0; 1999 tokens, 4 key heads of 64, prefix and cap: 43.8 and 32.2; 9914 tokens, one head: 71 and 98.
//
// The first limit is no crossing of the forms.  Single tokens, 56 query heads on 8 key heads of 128, with tiles and
// with `few`, over 300 / 1000 / 4000 keys each: 32 sequences 13, 12 / 29, 28 / 104, 104 us; 63: 19, 18 / 54, 53 / 189,
// 188; 64: 19, 19 / 58, 57 / 192, 191; 65: 25, 23 / 73, 62; 128: 37, 36 / 104, 101; 256: 75, 70 / 200, 195.  Two key
// heads, 256 sequences: 19, 19 / 55, 54 / 193, 192; 400: 31, 29 / 88, 88 / 308, 319.  64 of unequal lengths up to
// 8190, in steps: 240, 229; at random: 248, 251; spread over the logarithm: 158, 107; 65 of these: 154, 98 (one draw
// each: see slots_before for how far draws differ).  Beyond the limit `few` is mostly the better one, by up to a
// third.  The limit stays: the forms add up in another order, and calls keep the bits of their results.
//
// Codes.  `few` takes them without a detour, so it goes further, up to 64 rows on average whatever their number.  32 on
// 8 heads, tiles and `few`, E4M3 / INT8: 64 sequences of 16 tokens over 2048 keys, heads of 128 109, 85 / 127, 106 us,
// of 64 82, 53 / 88, 68; single tokens of 64 sequences, 56 heads on 8 of 128, 0 to 6122 keys, INT8 173 and 104.  INT8
// and heads of 64 pay more for expanding a code in every workgroup of 32 rows: 8 sequences of 64 tokens over 4096 keys,
// INT8, 71 and 82, heads of 64 47 and 53, but E4M3 with heads of 128 64 and 54.  With a cap or bias, heads of 128 in
// tiles have more in registers than there is room for: cap, chunks of up to 1024 tokens over up to 8192 keys 431 and
// 290 / 465 and 410, 8192 tokens 948 and 925 / 1008 and 1303.
struct Plan {
  bool few;
  int slots;
};
enum Kind { UNPAGED = 0, PAGED = 1, E4M3_PAGES = 2, INT8_PAGES = 4, WIDE_HEADS = 8, SCORE_MODS = 16 };  // bits
inline Plan plan(int kind, int64_t tokens, int group, int kv_heads, int64_t sequences, int64_t keys, int cus) {
  const bool paged = kind != UNPAGED, codes = kind & (E4M3_PAGES | INT8_PAGES);
  const bool spills = kind & SCORE_MODS && kind & WIDE_HEADS, cheap = kind & E4M3_PAGES && kind & WIDE_HEADS;
  const int64_t rows = tokens * group, own = paged ? sequences : 1;
  const int64_t tiles = (rows / (32 * WAVES) + own) * kv_heads, thin = (rows / 32 + own) * kv_heads;
  bool few = tiles < cus && thin <= (keys < 512 || (codes && !cheap) ? 2 : 4) * cus && keys <= 4096;
  if (codes) few = few || rows <= 64 * own || (spills && (cheap || tiles <= 4 * cus));
  else few = few || (rows <= 32 * own && own * kv_heads < 2 * cus);
  const int r = few ? 32 : 32 * WAVES;
  return Plan{few, static_cast<int>(paged ? slots_before(tokens, sequences + 1, group, r) : (rows + r - 1) / r)};
}

// Key splits: as many as bring the workgroups to two a compute unit, what it holds at once, each over at least 256 keys
// of the longest span; twice as many were slower (2048 tokens, 8 heads: 22 and 36 us).  Full workgroups of `few` to
// one: their waves split the keys already, and the sums of 32 rows cost as much as their keys (2000 tokens, 4 query
// heads on one key head, 250 workgroups: 19 us, 26 us in two splits).
inline int plan_splits(int kind, int64_t tokens, int group, int kv_heads, int64_t sequences, int64_t keys,
                       int cus) {
  const bool paged = kind != UNPAGED;
  const Plan p = plan(kind, tokens, group, kv_heads, sequences, keys, cus);
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

// The second launch of a call in key splits (attention.hip): a row a workgroup where there are many splits, else four.
constexpr int JOINED_TOGETHER = 8;
inline bool join_fits(const Args& a) {
  const int64_t rows = int64_t{a.tokens} * a.heads;
  return fits_launch(a.splits > JOINED_TOGETHER ? rows : (rows + 3) / 4, 256);
}
int launch_join(const Args& a, int dtype, int head_dim, hipStream_t st);

template <int DT, int D, int KEYS, bool SINKS, int CODES>
int launch(Args& a, hipStream_t st) {
  const bool mods = a.softcap > 0.0f || a.slopes;
  constexpr int KIND = KEYS == DENSE ? UNPAGED : !CODES ? PAGED : (CODES == E4M3 ? E4M3_PAGES : INT8_PAGES) |
                                                                      (D == 128 ? WIDE_HEADS : 0);
  const Plan p = plan(KIND | (CODES && mods ? SCORE_MODS : 0), a.tokens, a.group, a.kv_heads, a.sequences, a.reach,
                      device_cus());
  a.slots = p.slots;
  a.cus = device_cus();
  a.spread = a.kv_heads % 8 != 0 && (KEYS != DENSE || a.causal || a.starts);
  const int64_t blocks = int64_t{a.slots} * a.kv_heads * a.splits;
  M5K_REQUIRE(fits_launch(blocks, THREADS), "attention: too many tiles for one launch");
  M5K_REQUIRE(a.splits == 1 || join_fits(a), "attention: too many rows for one launch of their join");
  constexpr bool ALWAYS_FEW = CODES == E4M3 && D == 128;  // with MODS
  auto kernel = p.few ? (mods ? attention_tile<DT, D, KEYS, true, true, SINKS, CODES>
                              : attention_tile<DT, D, KEYS, false, true, SINKS, CODES>)
                      : (mods ? attention_tile<DT, D, KEYS, true, ALWAYS_FEW, SINKS, CODES>
                              : attention_tile<DT, D, KEYS, false, false, SINKS, CODES>);
  launch_kernel(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(THREADS), st, a);
  int rc = launch_status("attention");
  if (rc != M5K_OK || a.splits == 1) return rc;
  return launch_join(a, DT, D, st);
}

// One translation unit each (attention_*.hip), so that they compile side by side.
template <int KEYS, bool SINKS, int CODES>
int launch_typed(Args& a, int dtype, int head_dim, hipStream_t st);

#define M5K_ATTENTION_UNIT(KEYS, SINKS, CODES)                                                          \
  namespace m5k {                                                                                       \
  namespace attn {                                                                                      \
  template <>                                                                                           \
  int launch_typed<KEYS, SINKS, CODES>(Args & a, int dtype, int head_dim, hipStream_t st) {             \
    if (dtype == M5K_BF16)                                                                              \
      return head_dim == 64 ? launch<M5K_BF16, 64, KEYS, SINKS, CODES>(a, st)                           \
                            : launch<M5K_BF16, 128, KEYS, SINKS, CODES>(a, st);                         \
    return head_dim == 64 ? launch<M5K_F16, 64, KEYS, SINKS, CODES>(a, st)                              \
                          : launch<M5K_F16, 128, KEYS, SINKS, CODES>(a, st);                            \
  }                                                                                                     \
  }                                                                                                     \
  }

}  // namespace attn
}  // namespace m5k
