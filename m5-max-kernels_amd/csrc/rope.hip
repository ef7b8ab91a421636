// Rotary positions, alone and on the way into a paged cache.
//
// Pair j of a row at position p is turned by a = p f_j: (x1 c - x2 s, x2 c + x1 s).  Memory bound: each element is
// read and written once.  A thread owns a chunk of 8 channels (16 bytes of a 16-bit type) of one token and walks over
// heads with it, so that the chunk's sines and cosines, the only arithmetic of note, are made once for all of them.
// In the half layout the partner channels are R away: a second load, which the thread that owns them brings into the
// cache as well.  9914 tokens of 56 heads of 128 in BF16 take 54 us, 5.3 TB/s read and written, the rate of a copy; 64
// tokens appended 5.3 us, a chain of dependent loads (sequence, page, row).
//
// Angles.  p f_j / 2 pi is reduced to a fraction of a turn in 64 bits: at position 10^6 an FP32 angle would be off by
// 0.06 rad, the 64-bit fraction by 10^-10.  The fraction's nearest quarter turn is taken off in 64 bits too and the
// rest, |y| <= pi / 4, goes through the Taylor series of sine and cosine in FP32 (terms left out below 2e-9).
#include "m5k_common.h"

namespace m5k {
namespace {

constexpr double INV_TURN = 0.15915494309189533577;  // 1 / (2 pi)
constexpr int HEADS_MAX = 8;                         // heads one thread walks over

__device__ __forceinline__ void turn_of(int position, double frequency, float magnitude, float& c, float& s) {
  double t = static_cast<double>(position) * (frequency * INV_TURN);
  t -= rint(t);
  const double q = rint(4.0 * t);
  const float y = static_cast<float>(t - 0.25 * q) * 6.28318530717958647692f;
  const float z = y * y;
  float a = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  a = __builtin_fmaf(z, a, 1.0f / 120.0f);
  a = __builtin_fmaf(z, a, -1.0f / 6.0f);
  const float sine = __builtin_fmaf(y * z, a, y);
  float b = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  b = __builtin_fmaf(z, b, -1.0f / 720.0f);
  b = __builtin_fmaf(z, b, 1.0f / 24.0f);
  b = __builtin_fmaf(z, b, -0.5f);
  const float cosine = __builtin_fmaf(z, b, 1.0f);
  const int quarter = static_cast<int>(q) & 3;
  const bool odd = quarter & 1;
  c = (odd ? sine : cosine) * ((quarter == 1 || quarter == 2) ? -magnitude : magnitude);
  s = (odd ? cosine : sine) * (quarter >= 2 ? -magnitude : magnitude);
}

// One of a launch's tensors: read by strides, written contiguously per head and token, or into the cache's pages.
struct Part {
  const void* src;
  void* dst;
  int64_t src_head, src_token, dst_head, dst_token, dst_page;
  int heads, blocks;  // blockIdx.y values it takes
  bool turned, paged;
};

struct Args {
  Part part[3];
  const int32_t *positions, *table, *starts, *context;
  const double* frequencies;
  int64_t table_width;
  int tokens, dim, pairs, sequences, pages, page_size, walk;
  float magnitude;
};

template <int DT, int V>
__device__ __forceinline__ void load_chunk(const void* p, int64_t at, float (&x)[V]) {
  if constexpr (V == 8) {
    load8<DT>(p, at, x);
  } else {
    x[0] = load_elem<DT>(p, at);
  }
}

template <int DT, int V>
__device__ __forceinline__ void store_chunk(void* p, int64_t at, const float (&x)[V]) {
  if constexpr (V == 1) {
    store_elem<DT>(p, at, x[0]);
  } else if constexpr (DT == M5K_F32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    d[0] = make_float4(x[0], x[1], x[2], x[3]);
    d[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 w;
    uint32_t* u = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == M5K_BF16) u[i] = f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
      else u[i] = f32_to_f16_bits(x[2 * i]) | (f32_to_f16_bits(x[2 * i + 1]) << 16);
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = w;
  }
}

// V channels a thread: 8 where rows allow 16-byte accesses, else 1.  WHOLE (half layout, V = 8): pairs is a multiple of
// 8, so a chunk is turned with one other chunk or copied; otherwise the partner of each channel is read by itself.
template <int DT, int V, bool INTERLEAVED, bool WHOLE>
__global__ __launch_bounds__(256) void rope_rows(const Args a) {
  int y = blockIdx.y, which = 0;
  while (which < 2 && y >= a.part[which].blocks) y -= a.part[which++].blocks;
  const Part& part = a.part[which];
  const int chunks = a.dim / V;
  const int64_t unit = int64_t{blockIdx.x} * 256 + threadIdx.x;
  if (unit >= int64_t{a.tokens} * chunks) return;
  const int token = static_cast<int>(unit / chunks), c0 = static_cast<int>(unit - int64_t{token} * chunks) * V;
  const int head0 = y * a.walk, head1 = min(head0 + a.walk, part.heads);

  int position = 0;
  int64_t dst = int64_t{token} * part.dst_token;
  bool known = true;
  if (a.starts) {
    // The last sequence that starts at or before the token, and the token's position in it.
    int lo = 0, hi = a.sequences;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.starts[mid] <= token) lo = mid;
      else hi = mid;
    }
    const int s = a.starts[lo], e = a.starts[lo + 1];
    known = token >= s && token < e;
    position = known ? a.context[lo] - (e - token) : 0;
    if (part.paged) {
      const int page_at = position / a.page_size;
      if (!known || position < 0 || page_at >= a.table_width) return;
      const int page = a.table[lo * a.table_width + page_at];
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) return;
      dst = page * part.dst_page + (position - page_at * a.page_size) * part.dst_token;
    }
  } else if (a.positions) {
    position = a.positions[token];
  }

  const bool turned = part.turned && c0 < 2 * a.pairs;
  constexpr int NF = INTERLEAVED && V == 8 ? 4 : V;
  float cs[NF], sn[NF];
  if (turned) {
#pragma unroll
    for (int i = 0; i < NF; ++i) {
      const int d = INTERLEAVED ? c0 + (V == 8 ? 2 * i : 0) : c0 + i;
      const int j = INTERLEAVED ? d >> 1 : d < a.pairs ? d : d - a.pairs;
      cs[i] = 1.0f;
      sn[i] = 0.0f;
      if (d < 2 * a.pairs) turn_of(position, a.frequencies[j], a.magnitude, cs[i], sn[i]);
      // The first of a pair takes - s of its partner, the second + s.
      if (!(INTERLEAVED && V == 8)) {
        if (INTERLEAVED ? !(d & 1) : d < a.pairs) sn[i] = -sn[i];
      }
    }
  }
  for (int h = head0; h < head1; ++h) {
    const int64_t row = h * part.src_head + token * part.src_token;
    float x[V], out[V];
    if (known) {
      load_chunk<DT, V>(part.src, row + c0, x);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = 0.0f;
    }
    if (!turned || !known) {
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = x[i];
    } else if constexpr (INTERLEAVED && V == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool turns = c0 + 2 * i < 2 * a.pairs;  // else copied as it is: times 0, a partner's infinity is NaN
        out[2 * i] = turns ? x[2 * i] * cs[i] - x[2 * i + 1] * sn[i] : x[2 * i];
        out[2 * i + 1] = turns ? x[2 * i + 1] * cs[i] + x[2 * i] * sn[i] : x[2 * i + 1];
      }
    } else {
      float partner[V];
      if constexpr (WHOLE) {
        load_chunk<DT, V>(part.src, row + (c0 < a.pairs ? c0 + a.pairs : c0 - a.pairs), partner);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int d = c0 + i;
          const int other = INTERLEAVED ? d ^ 1 : d < a.pairs ? d + a.pairs : d - a.pairs;
          partner[i] = d < 2 * a.pairs ? load_elem<DT>(part.src, row + other) : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) out[i] = c0 + i < 2 * a.pairs ? x[i] * cs[i] + partner[i] * sn[i] : x[i];
    }
    store_chunk<DT, V>(part.dst, dst + h * part.dst_head + c0, out);
  }
}

template <int DT>
int launch(Args& a, bool vector, bool interleaved, hipStream_t st) {
  const int v = vector ? 8 : 1;
  int64_t heads = 0;
  for (const Part& p : a.part) heads += p.heads;
  const int64_t units = int64_t{a.tokens} * (a.dim / v);
  // Heads a thread: as many as leave the chip's 256 compute units 1024 threads each.
  const int64_t walk = units * heads / (256 * 1024);
  a.walk = static_cast<int>(walk < 1 ? 1 : walk > HEADS_MAX ? HEADS_MAX : walk);
  int blocks = 0;
  for (Part& p : a.part) blocks += p.blocks = (p.heads + a.walk - 1) / a.walk;
  const int64_t gx = (units + 255) / 256;
  M5K_REQUIRE(gx <= INT32_MAX && blocks <= 65535, "rope: too many rows for one launch");
  const dim3 grid(static_cast<uint32_t>(gx), static_cast<uint32_t>(blocks));
  const bool whole = a.pairs % 8 == 0;
  // With one channel a thread the partner's place is found by itself in either layout.
  auto kernel = !vector       ? (interleaved ? rope_rows<DT, 1, true, false> : rope_rows<DT, 1, false, false>)
                : interleaved ? rope_rows<DT, 8, true, false>
                : whole       ? rope_rows<DT, 8, false, true>
                              : rope_rows<DT, 8, false, false>;
  launch_kernel(kernel, grid, dim3(256), st, a);
  return launch_status("rope");
}

int launch_typed(Args& a, int dtype, bool vector, int interleaved, hipStream_t st) {
  if (dtype == M5K_BF16) return launch<M5K_BF16>(a, vector, interleaved != 0, st);
  if (dtype == M5K_F16) return launch<M5K_F16>(a, vector, interleaved != 0, st);
  return launch<M5K_F32>(a, vector, interleaved != 0, st);
}

bool vector_rows(const void* p, int64_t s0, int64_t s1, int64_t s2, int dtype) {
  const int64_t unit = dtype == M5K_F32 ? 4 : 8;  // elements of 16 bytes
  return aligned16(p) && s0 % unit == 0 && s1 % unit == 0 && s2 % unit == 0;
}

int check_rows(int dtype, int64_t tokens, int64_t head_dim, const double* frequencies, int64_t pairs) {
  M5K_REQUIRE(dtype == M5K_F32 || dtype == M5K_F16 || dtype == M5K_BF16, "rope: dtype must be f32, f16 or bf16");
  M5K_REQUIRE(tokens > 0 && tokens <= (1 << 30) && head_dim > 0 && head_dim <= (1 << 16), "rope: bad sizes");
  M5K_REQUIRE(pairs >= 0 && 2 * pairs <= head_dim && (pairs == 0 || frequencies),
              "rope: 2 * pairs must fit in head_dim");
  return M5K_OK;
}

}  // namespace
}  // namespace m5k

extern "C" int m5k_rope(const void* x, int dtype, int64_t tokens, int64_t heads, int64_t head_dim, int64_t x_head,
                        int64_t x_token, const int32_t* positions, const double* frequencies, int64_t pairs,
                        int interleaved, float magnitude, void* y, void* stream) {
  using namespace m5k;
  clear_error();
  if (int rc = check_rows(dtype, tokens, head_dim, frequencies, pairs)) return rc;
  M5K_REQUIRE(x && y && positions && pairs > 0, "rope: null pointer or no pairs");
  M5K_REQUIRE(heads > 0 && heads <= 65535, "rope: heads must be in [1, 65535]");
  Args a = {};
  a.part[0] = Part{x, y, x_head, x_token, tokens * head_dim, head_dim, 0, static_cast<int>(heads), 0, true, false};
  a.positions = positions;
  a.frequencies = frequencies;
  a.tokens = static_cast<int>(tokens);
  a.dim = static_cast<int>(head_dim);
  a.pairs = static_cast<int>(pairs);
  a.magnitude = magnitude;
  const bool vector = head_dim % 8 == 0 && vector_rows(x, x_head, x_token, 0, dtype) && aligned16(y);
  return launch_typed(a, dtype, vector, interleaved, as_stream(stream));
}

extern "C" int m5k_paged_append(const void* k, int64_t k_head, int64_t k_token, const void* v, int64_t v_head,
                                int64_t v_token, int dtype, int64_t tokens, int64_t kv_heads, int64_t head_dim,
                                void* k_cache, int64_t kc_page, int64_t kc_head, int64_t kc_slot, void* v_cache,
                                int64_t vc_page, int64_t vc_head, int64_t vc_slot, int64_t pages, int64_t page_size,
                                const int32_t* page_table, int64_t table_width, int64_t sequences,
                                const int32_t* query_starts, const int32_t* context_lengths, const void* q,
                                int64_t heads, int64_t q_head, int64_t q_token, void* q_out, const double* frequencies,
                                int64_t pairs, int interleaved, float magnitude, void* stream) {
  using namespace m5k;
  clear_error();
  if (int rc = check_rows(dtype, tokens, head_dim, frequencies, pairs)) return rc;
  M5K_REQUIRE(k && v && k_cache && v_cache && page_table && query_starts && context_lengths,
              "paged_append: null pointer");
  M5K_REQUIRE(!q || (q_out && heads > 0 && pairs > 0), "paged_append: q needs q_out, heads and a rotation");
  M5K_REQUIRE(kv_heads > 0 && kv_heads <= 16384 && (!q || heads <= 16384), "paged_append: bad number of heads");
  M5K_REQUIRE(pages > 0 && pages <= INT32_MAX && page_size > 0 && page_size <= (1 << 20) && table_width > 0 &&
                  table_width * page_size <= (1 << 30) && sequences > 0 && sequences <= (1 << 24),
              "paged_append: a sequence may have up to 2^30 keys in pages of up to 2^20");
  Args a = {};
  const int kvh = static_cast<int>(kv_heads);
  a.part[0] = Part{k, k_cache, k_head, k_token, kc_head, kc_slot, kc_page, kvh, 0, pairs > 0, true};
  a.part[1] = Part{v, v_cache, v_head, v_token, vc_head, vc_slot, vc_page, kvh, 0, false, true};
  if (q)
    a.part[2] = Part{q,       q_out, q_head, q_token, tokens * head_dim, head_dim, 0, static_cast<int>(heads), 0, true,
                     false};
  a.table = page_table;
  a.table_width = table_width;
  a.starts = query_starts;
  a.context = context_lengths;
  a.frequencies = frequencies;
  a.tokens = static_cast<int>(tokens);
  a.dim = static_cast<int>(head_dim);
  a.pairs = static_cast<int>(pairs);
  a.sequences = static_cast<int>(sequences);
  a.pages = static_cast<int>(pages);
  a.page_size = static_cast<int>(page_size);
  a.magnitude = magnitude;
  bool vector = head_dim % 8 == 0;
  for (const Part& p : a.part) {
    if (!p.heads) continue;
    vector = vector && vector_rows(p.src, p.src_head, p.src_token, 0, dtype) &&
             vector_rows(p.dst, p.dst_head, p.dst_token, p.dst_page, dtype);
  }
  return launch_typed(a, dtype, vector, interleaved, as_stream(stream));
}
