// Fresh keys and values into the paged cache, rotated on the way, and the
// 4-bit form of the pages with its read-back.
//
// Rotation at position p (r = rotary_dim; cos_p, sin_p the table's row):
//   neox    y[i] = x[i] cos_p[i] - x[i + r/2] sin_p[i]
//           y[i + r/2] = x[i + r/2] cos_p[i] + x[i] sin_p[i]          i < r/2
//   GPT-J   the same with the partners 2i and 2i + 1
// The table is read in its own type, both products and the sum are rounded to
// fp32 one by one (no contraction), and the result is rounded once to the
// element type: a row is the same bits whichever of these kernels wrote it.  (The
// relocation of cached keys rounds the table and every product to the key type.)
//
// 4-bit rows: every 64 values of a row share a lowest value and a step,
//   low = fp16(min x), step = fp16((max x - low') / 15)   (low' = the fp32 minimum)
//   code = clamp(rint((x - low) * (1 / step)), 0, 15),  value = low + step code
// fp16 (11 bits) rather than bf16 for the pair: its rounding is 2^-11 of the
// lowest value, far below a step, where bf16's 2^-8 can exceed one in a channel
// with a large offset.  Values beyond fp16's range are held at +-65504; a group
// with a NaN or an infinity gets a NaN step, so it reads as NaN.  Two codes to
// a byte, the lower dimension in the low nibble.
//
// What bounds them: HBM at long prompts, the launch at decode sizes.  Threads of
// a block run over one token's pieces first, so rows are read and written whole.
// Rows that are not 16-byte aligned go value by value: 16,384 tokens of 32 + 8 + 8
// heads 700 us (67 aligned), 20,011 tokens into 4-bit pages 79 us (40).
#include <algorithm>
#include <type_traits>

#include "cb_common.cuh"

namespace cb {
namespace append {

constexpr int kThreads = 256;  // of a block, at most
constexpr int kGroup = 64;  // values that share a step
constexpr float kHalfMax = 65504.0f;

struct Params {
  const char* key;
  const char* value;
  const char* query;  // may be null: no query heads then
  char* query_out;
  int64_t key_ts, key_hs, value_ts, value_hs, query_ts, query_hs, qo_ts, qo_hs;  // bytes
  int64_t tokens;
  int q_heads, kv_heads, head_size;
  const int64_t* positions;  // null with rotary_dim 0
  const void* table;
  int64_t max_position;
  int rotary_dim, neox;
  char* k_cache;  // 16/32-bit pages, or the codes
  char* v_cache;
  int64_t block_stride, slot_stride, head_stride;
  char* k_scales;  // 4-bit pages: (step, low) pairs
  char* v_scales;
  int64_t scale_block_stride, scale_slot_stride, scale_head_stride;
  int64_t num_slots;
  int block_size;
  const int64_t* slots;
  // thread layout: units of a token, units and tokens per block
  int units, units_block, tokens_block, threads;
};

// slot -> (block, row), with the short division wherever it does.
__device__ __forceinline__ void split_slot(int64_t slot, int block_size, int& block, int& row) {
  block = (slot >> 31) == 0 ? static_cast<int>(slot) / block_size : static_cast<int>(slot / block_size);
  row = static_cast<int>(slot - static_cast<int64_t>(block) * block_size);
}

// N consecutive elements as fp32.  WIDE: the address is aligned to the vector.
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void load_n(const T* p, float (&x)[N]) {
  if constexpr (WIDE && N > 1) {
    constexpr int kBytes = N * static_cast<int>(sizeof(T));
    constexpr int kVec = kBytes >= 16 ? 16 : kBytes;
    using V = typename Vec<kVec>::T;
    constexpr int kPer = kVec / static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
      const V v = __ldg(reinterpret_cast<const V*>(p) + i);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < kPer; ++j) x[i * kPer + j] = Elem<T>::to_f(e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = Elem<T>::to_f(p[j]);
  }
}

// N elements as they lie, in whole 16-byte vectors: loads that are issued before anything
// that depends on them, in half the registers of fp32.
template <typename T, int N>
struct Piece {
  static constexpr int kVecs = N * static_cast<int>(sizeof(T)) / 16;
  uint4 v[kVecs];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = ld_stream(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ float operator[](int j) const {
    return Elem<T>::to_f(reinterpret_cast<const T*>(v)[j]);
  }
};

template <typename T, int N, bool WIDE>
__device__ __forceinline__ void store_n(T* p, const float (&y)[N]) {
  if constexpr (WIDE && N > 1) {
    constexpr int kPer = 16 / static_cast<int>(sizeof(T));
    static_assert(N % kPer == 0, "whole 16-byte vectors");
#pragma unroll
    for (int i = 0; i < N / kPer; ++i) {
      uint4 v;
      T* e = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int j = 0; j < kPer; ++j) e[j] = Elem<T>::from_f(y[i * kPer + j]);
      reinterpret_cast<uint4*>(p)[i] = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = Elem<T>::from_f(y[j]);
  }
}

__device__ __forceinline__ float turn_first(float a, float b, float cos, float sin) {
  return __fsub_rn(__fmul_rn(a, cos), __fmul_rn(b, sin));
}
__device__ __forceinline__ float turn_second(float a, float b, float cos, float sin) {
  return __fadd_rn(__fmul_rn(b, cos), __fmul_rn(a, sin));
}

// Values d0 .. d0 + N - 1 of a row, rotated.  WIDE: d0 is a multiple of N and no
// piece of N crosses rotary_dim (neox: nor its half).
template <typename T, typename TAB, int N, bool WIDE>
__device__ __forceinline__ void rotated(const T* row, int d0, const TAB* table, int rotary, bool neox,
                                        float (&y)[N]) {
  if constexpr (WIDE) {
    load_n<T, N, true>(row + d0, y);
    if (d0 >= rotary) return;
    if (neox) {
      const int half = rotary >> 1;
      const bool first = d0 < half;
      const int i = first ? d0 : d0 - half;
      float other[N], cos[N], sin[N];
      load_n<T, N, true>(row + (first ? d0 + half : i), other);
      load_n<TAB, N, true>(table + i, cos);
      load_n<TAB, N, true>(table + half + i, sin);
#pragma unroll
      for (int j = 0; j < N; ++j)
        y[j] = first ? turn_first(y[j], other[j], cos[j], sin[j]) : turn_second(other[j], y[j], cos[j], sin[j]);
    } else {
      constexpr int kPairs = N / 2;
      float cos[kPairs], sin[kPairs];
      load_n<TAB, kPairs, true>(table + d0 / 2, cos);
      load_n<TAB, kPairs, true>(table + (rotary >> 1) + d0 / 2, sin);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float a = y[2 * j], b = y[2 * j + 1];
        y[2 * j] = turn_first(a, b, cos[j], sin[j]);
        y[2 * j + 1] = turn_second(a, b, cos[j], sin[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int d = d0 + j;
      const float x = Elem<T>::to_f(row[d]);
      if (d >= rotary) {
        y[j] = x;
        continue;
      }
      const int half = rotary >> 1;
      const int i = neox ? (d < half ? d : d - half) : d >> 1;
      const bool first = neox ? d < half : (d & 1) == 0;
      const float other = Elem<T>::to_f(row[neox ? (first ? d + half : i) : d ^ 1]);
      const float cos = Elem<TAB>::to_f(table[i]), sin = Elem<TAB>::to_f(table[half + i]);
      y[j] = first ? turn_first(x, other, cos, sin) : turn_second(other, x, cos, sin);
    }
  }
}

// Where a thread works: a token, and one piece of HPT heads of K (plane 0), V (1) or Q (2).
struct Place {
  bool real;
  int token;  // (32 bits: an address is then one short product and a sum per stride)
  int plane, head, piece;
};
template <int HPT, typename P>
__device__ __forceinline__ Place place(const P& c, int kv_heads, int q_heads, int pieces) {
  Place w;
  const int tok = threadIdx.x / c.units_block;
  const int unit = blockIdx.y * c.units_block + (threadIdx.x - tok * c.units_block);
  w.token = static_cast<int>(min(static_cast<int64_t>(blockIdx.x) * c.tokens_block + tok, c.tokens));
  w.real = tok < c.tokens_block && unit < c.units && w.token < c.tokens;
  const int bundles = unit / pieces;  // of HPT heads
  const int kv_bundles = (kv_heads + HPT - 1) / HPT;
  w.piece = unit - bundles * pieces;
  w.plane = bundles < kv_bundles ? 0 : (bundles < 2 * kv_bundles ? 1 : 2);
  w.head = (bundles - w.plane * kv_bundles) * HPT;
  return w;
}

// What a thread does with its token: where its rows go, and whether they go anywhere.
struct Target {
  bool turned;  // the position lies inside the table (or nothing is rotated)
  bool stored;  // K or V with a slot of the cache
  int64_t position;
  int block, row;
};
__device__ __forceinline__ Target target(const Params& c, const Place& w) {
  Target g{};
  if (!w.real) return g;
  const int64_t slot = w.plane < 2 ? __ldg(c.slots + w.token) : -1;
  g.turned = true;
  if (c.rotary_dim > 0) {  // V goes with its K: a bad position leaves the whole slot as it was
    g.position = __ldg(c.positions + w.token);
    g.turned = g.position >= 0 && g.position < c.max_position;
  }
  g.stored = slot >= 0 && slot < c.num_slots && g.turned;
  if (g.stored) split_slot(slot, c.block_size, g.block, g.row);
  return g;
}

// 16-byte pieces of 16/32-bit rows.  A thread takes two of them -- for neox the two
// partners of a rotation, so that each is read once and one piece of the table serves
// both -- in HPT heads, whose loads are in flight together and share the table's values.
// HPT 4 at long prompts, 1 where there are too few tokens to fill the GPU (more_heads).
// A prompt of 16,384 tokens, 32 + 8 + 8 heads of 128: 69 us, 5.9 TB/s; 137 us when the loads
// waited for slots and positions and each thread had one piece.
template <typename T, typename TAB, int HPT>
__global__ void __launch_bounds__(kThreads) append_kernel(const Params c) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));
  const Place w = place<HPT>(c, c.kv_heads, c.q_heads, c.head_size / (2 * N));
  if (!w.real) return;
  const bool is_q = w.plane == 2;
  const char* src = is_q ? c.query + w.token * c.query_ts
                         : (w.plane == 0 ? c.key + w.token * c.key_ts : c.value + w.token * c.value_ts);
  const int64_t src_hs = is_q ? c.query_hs : (w.plane == 0 ? c.key_hs : c.value_hs);
  const int heads = is_q ? c.q_heads : c.kv_heads;
  // the two pieces: partners below rotary_dim (neox), neighbours elsewhere
  const int half = c.rotary_dim >> 1;
  const bool partners = w.plane != 1 && c.neox && w.piece * N < half;
  const int d0 = partners ? w.piece * N
                          : (w.plane != 1 && c.neox ? c.rotary_dim + 2 * (w.piece * N - half) : 2 * w.piece * N);
  const int d1 = partners ? d0 + half : d0 + N;
  // padding rows are read too: the loads wait for no slot or position
  Piece<T, N> a[HPT], b[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (w.head + i < heads) {
      const T* row = reinterpret_cast<const T*>(src + (w.head + i) * src_hs);
      a[i].load(row + d0);
      b[i].load(row + d1);
    }
  const Target g = target(c, w);
  if (!is_q && !g.stored) return;
  float cos[N], sin[N];
  const bool turn = w.plane != 1 && d0 < c.rotary_dim && g.turned;
  if (turn) {
    const TAB* table = static_cast<const TAB*>(c.table) + g.position * c.rotary_dim + (partners ? d0 : d0 / 2);
    load_n<TAB, N, true>(table, cos);
    load_n<TAB, N, true>(table + half, sin);
  }
  char* dst = is_q ? c.query_out + w.token * c.qo_ts
                   : (w.plane == 0 ? c.k_cache : c.v_cache) + g.block * c.block_stride + g.row * c.slot_stride;
  const int64_t dst_hs = is_q ? c.qo_hs : c.head_stride;
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (w.head + i < heads) {
      float x[N], y[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = g.turned ? a[i][j] : 0.0f, y[j] = g.turned ? b[i][j] : 0.0f;
      if (turn && partners) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float p = x[j], q = y[j];
          x[j] = turn_first(p, q, cos[j], sin[j]);
          y[j] = turn_second(p, q, cos[j], sin[j]);
        }
      } else if (turn) {  // GPT-J: N pairs over the two pieces (rotary_dim is a multiple of both)
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          float p = x[2 * j], q = x[2 * j + 1];
          x[2 * j] = turn_first(p, q, cos[j], sin[j]);
          x[2 * j + 1] = turn_second(p, q, cos[j], sin[j]);
          p = y[2 * j], q = y[2 * j + 1];
          y[2 * j] = turn_first(p, q, cos[N / 2 + j], sin[N / 2 + j]);
          y[2 * j + 1] = turn_second(p, q, cos[N / 2 + j], sin[N / 2 + j]);
        }
      }
      T* row = reinterpret_cast<T*>(dst + (w.head + i) * dst_hs);
      store_n<T, N, true>(row + d0, x);
      store_n<T, N, true>(row + d1, y);
    }
}

// Rows that cannot go in aligned 16-byte pieces: a value per thread.
template <typename T, typename TAB>
__global__ void __launch_bounds__(kThreads) append_narrow_kernel(const Params c) {
  const Place w = place<1>(c, c.kv_heads, c.q_heads, c.head_size);
  if (!w.real) return;
  const Target g = target(c, w);
  if (w.plane < 2 && !g.stored) return;
  const TAB* table = static_cast<const TAB*>(c.table) + g.position * c.rotary_dim;
  float y[1];
  T* out;
  if (w.plane == 2) {
    out = reinterpret_cast<T*>(c.query_out + w.token * c.qo_ts + w.head * c.qo_hs);
    if (g.turned)
      rotated<T, TAB, 1, false>(reinterpret_cast<const T*>(c.query + w.token * c.query_ts + w.head * c.query_hs), w.piece,
                                table, c.rotary_dim, c.neox != 0, y);
    else
      y[0] = 0.0f;
  } else {
    out = reinterpret_cast<T*>((w.plane == 0 ? c.k_cache : c.v_cache) + g.block * c.block_stride + g.row * c.slot_stride +
                               w.head * c.head_stride);
    if (w.plane == 0)
      rotated<T, TAB, 1, false>(reinterpret_cast<const T*>(c.key + w.token * c.key_ts + w.head * c.key_hs), w.piece, table,
                                c.rotary_dim, c.neox != 0, y);
    else
      y[0] = Elem<T>::to_f(reinterpret_cast<const T*>(c.value + w.token * c.value_ts + w.head * c.value_hs)[w.piece]);
  }
  out[w.piece] = Elem<T>::from_f(y[0]);
}

// The (step, lowest) pair of a group from its extremes; `bad`: it holds a NaN or an infinity.
__device__ __forceinline__ __half2 step_of(float low, float high, bool bad) {
  low = fminf(fmaxf(low, -kHalfMax), kHalfMax);
  high = fminf(fmaxf(high, -kHalfMax), kHalfMax);
  const __half step = __float2half_rn(__fmul_rn(__fsub_rn(high, low), 1.0f / 15.0f));
  return __halves2half2(bad ? __ushort_as_half(0x7e00) : step, __float2half_rn(low));
}
// Codes of 8 values, the first in the lowest nibble.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], __half2 pair) {
  const float step = __low2float(pair), base = __high2float(pair);
  const float inverse = step > 0.0f ? __frcp_rn(step) : 0.0f;
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = fminf(fmaxf(__fmul_rn(__fsub_rn(x[j], base), inverse), 0.0f), 15.0f);
    // v + 1.5 * 2^23 has the nearest whole number (ties to even) in its low bits
    codes |= (__float_as_uint(__fadd_rn(v, 12582912.0f)) & 15u) << (4 * j);
  }
  return codes;
}

// A piece of 8 values rotated in registers: `other` holds a neox rotation's partners.
__device__ __forceinline__ void turn_piece(float (&x)[8], const float (&other)[8], int d, int rotary, bool neox,
                                           const float (&cos)[8], const float (&sin)[8]) {
  if (d >= rotary) return;
  if (neox) {
    const bool first = d < (rotary >> 1);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = first ? turn_first(x[j], other[j], cos[j], sin[j]) : turn_second(other[j], x[j], cos[j], sin[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p = x[2 * j], q = x[2 * j + 1];
      x[2 * j] = turn_first(p, q, cos[j], sin[j]);
      x[2 * j + 1] = turn_second(p, q, cos[j], sin[j]);
    }
  }
}

// Two elements of a 16-bit type in a word.
template <typename T>
struct Two;
template <>
struct Two<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 open(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {  // NaN if either is
    const __nv_bfloat162 h = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Two<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 open(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {
    const __half2 h = __hmin2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Codes of 8 values in four words.  FAR: values may lie beyond fp16's range.  Without them
// (x - low) / step is at least -1/2, since a 16-bit x in fp16's range is off its fp16 form by
// 2^-25 at most and a step is 2^-24 at least, so that the nearest whole number (the low bits of
// v + 1.5 * 2^23) can be cut to 0..15 as an integer, one instruction with the subtraction of the
// float's upper bits.
template <typename T, bool FAR>
__device__ __forceinline__ uint32_t codes_of_words(const uint32_t (&w)[4], __half2 pair) {
  const float step = __low2float(pair), base = __high2float(pair);
  const float inverse = step > 0.0f ? __frcp_rn(step) : 0.0f;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // (packed products and sums would be contracted, so only the first difference is a pair's)
    float2 v = __fadd2_rn(Two<T>::open(w[i]), make_float2(-base, -base));
    v = make_float2(__fmul_rn(v.x, inverse), __fmul_rn(v.y, inverse));
    if constexpr (FAR) v = make_float2(fminf(fmaxf(v.x, 0.0f), 15.0f), fminf(fmaxf(v.y, 0.0f), 15.0f));
    v = make_float2(__fadd_rn(v.x, 12582912.0f), __fadd_rn(v.y, 12582912.0f));
    const uint32_t x = __viaddmin_s32_relu(__float_as_int(v.x), -0x4b400000, 15);
    const uint32_t y = __viaddmin_s32_relu(__float_as_int(v.y), -0x4b400000, 15);
    codes += x * (1u << (8 * i)) + y * (16u << (8 * i));
  }
  return codes;
}

template <typename T>
__device__ __noinline__ uint32_t far_codes(uint4 w, __half2 pair) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  return codes_of_words<T, true>(words, pair);
}

// 4-bit rows of 16-bit elements, aligned.  A lane takes the 8-value pieces at 8 p and
// D / 2 + 8 p of HPT heads of K or V (and of the queries, which stay of their type): the two
// partners of a neox rotation over the whole head, so nothing is read twice, and for D 128 one
// piece of each group of 64.  The eight lanes of a D 128 row reduce both groups side by side,
// the four of a D 64 row their one.  EXTRA: neox over a part of the head, whose partners are
// read beside (they come from L1).
// Bound by its instructions before HBM: 33 a value with one float at a time (60 us for a
// prompt of 20,011 tokens and 8 heads, 1.7 TB/s), so minima and maxima, conversions and the
// arithmetic go two values at a time.
template <typename T, typename TAB, int D, bool EXTRA, int HPT>
__global__ void __launch_bounds__(kThreads) append4_kernel(const Params c) {
  const Place w = place<HPT>(c, c.kv_heads, c.q_heads, D / 16);
  const bool is_q = w.plane == 2, neox = c.neox != 0;
  const char* src = is_q ? c.query + w.token * c.query_ts
                         : (w.plane == 0 ? c.key + w.token * c.key_ts : c.value + w.token * c.value_ts);
  const int64_t src_hs = is_q ? c.query_hs : (w.plane == 0 ? c.key_hs : c.value_hs);
  const int heads = w.real ? (is_q ? c.q_heads : c.kv_heads) : 0;
  const int half = c.rotary_dim >> 1;
  const int at[2] = {8 * w.piece, D / 2 + 8 * w.piece};
  int with[2];  // partners of the two pieces
#pragma unroll
  for (int s = 0; s < 2; ++s) with[s] = at[s] >= c.rotary_dim ? at[s] : (at[s] < half ? at[s] + half : at[s] - half);
  // padding rows are read too: the loads wait for no slot or position
  Piece<T, 8> own[HPT][2], beside[EXTRA ? HPT : 1][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (w.head + i < heads) {
      const T* row = reinterpret_cast<const T*>(src + (w.head + i) * src_hs);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        own[i][s].load(row + at[s]);
        if constexpr (EXTRA) beside[i][s].load(row + with[s]);
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        own[i][s].v[0] = make_uint4(0, 0, 0, 0);
        if constexpr (EXTRA) beside[i][s].v[0] = make_uint4(0, 0, 0, 0);
      }
    }
  const Target g = target(c, w);
  const bool turn = w.plane != 1 && c.rotary_dim > 0 && g.turned;
  constexpr int kTables = EXTRA ? 2 : 1;
  float cos[kTables][8], sin[kTables][8];  // neox over the whole head: one table piece for both partners;
                                           // GPT-J: four pairs of each piece
  if (turn) {
    const TAB* table = static_cast<const TAB*>(c.table) + g.position * c.rotary_dim;
    if constexpr (EXTRA) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (at[s] >= c.rotary_dim) continue;
        const int i = min(at[s], with[s]);
        load_n<TAB, 8, true>(table + i, cos[s]);
        load_n<TAB, 8, true>(table + half + i, sin[s]);
      }
    } else if (neox) {
      load_n<TAB, 8, true>(table + at[0], cos[0]);
      load_n<TAB, 8, true>(table + half + at[0], sin[0]);
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (at[s] >= c.rotary_dim) continue;
        float few[4];
        load_n<TAB, 4, true>(table + at[s] / 2, few);
#pragma unroll
        for (int j = 0; j < 4; ++j) cos[0][4 * s + j] = few[j];
        load_n<TAB, 4, true>(table + half + at[s] / 2, few);
#pragma unroll
        for (int j = 0; j < 4; ++j) sin[0][4 * s + j] = few[j];
      }
    }
  }
  const int64_t row_at = g.block * c.block_stride + g.row * c.slot_stride;
  const int64_t scale_at = g.block * c.scale_block_stride + g.row * c.scale_slot_stride;
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    uint32_t word[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) word[s][j] = reinterpret_cast<const uint32_t*>(own[i][s].v)[j];
    if (turn) {
      if constexpr (EXTRA) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float x[8], other[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = own[i][s][j], other[j] = beside[i][s][j];
          turn_piece(x, other, at[s], c.rotary_dim, true, cos[s], sin[s]);
#pragma unroll
          for (int j = 0; j < 4; ++j) word[s][j] = Two<T>::pack(x[2 * j], x[2 * j + 1]);
        }
      } else if (neox) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // (the packed product and sum would be contracted)
          const float2 a = Two<T>::open(word[0][j]), b = Two<T>::open(word[1][j]);
          const float c0 = cos[0][2 * j], c1 = cos[0][2 * j + 1], s0 = sin[0][2 * j], s1 = sin[0][2 * j + 1];
          word[0][j] = Two<T>::pack(turn_first(a.x, b.x, c0, s0), turn_first(a.y, b.y, c1, s1));
          word[1][j] = Two<T>::pack(turn_second(a.x, b.x, c0, s0), turn_second(a.y, b.y, c1, s1));
        }
      } else {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (at[s] >= c.rotary_dim) continue;
            const float2 x = Two<T>::open(word[s][j]);
            const float co = cos[0][4 * s + j], si = sin[0][4 * s + j];
            word[s][j] = Two<T>::pack(turn_first(x.x, x.y, co, si), turn_second(x.x, x.y, co, si));
          }
      }
    }
    if (is_q && w.head + i < heads) {
      T* out = reinterpret_cast<T*>(c.query_out + w.token * c.qo_ts + (w.head + i) * c.qo_hs);
#pragma unroll
      for (int s = 0; s < 2; ++s)  // zeros at a position outside the table
        *reinterpret_cast<uint4*>(out + at[s]) =
            g.turned ? make_uint4(word[s][0], word[s][1], word[s][2], word[s][3]) : make_uint4(0, 0, 0, 0);
    }
    // (lowest, -highest) of each piece in one word; NaN where a value is
    uint32_t ends[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t low = word[s][0], high = word[s][0] ^ 0x80008000u;
#pragma unroll
      for (int j = 1; j < 4; ++j) {
        low = Two<T>::least(low, word[s][j]);
        high = Two<T>::least(high, word[s][j] ^ 0x80008000u);
      }
      // the words' two halves against each other
      ends[s] = Two<T>::least(__byte_perm(low, high, 0x5410), __byte_perm(low, high, 0x7632));
    }
    if constexpr (D == 64) ends[0] = Two<T>::least(ends[0], ends[1]);
    // every lane of the warp is here: the lanes of a row reduce with their neighbours
    constexpr int kGroups = D / kGroup;
    __half2 pair[2];
    bool far[2];
#pragma unroll
    for (int s = 0; s < kGroups; ++s) {
#pragma unroll
      for (int o = D / 32; o >= 1; o >>= 1) ends[s] = Two<T>::least(ends[s], __shfl_xor_sync(0xffffffffu, ends[s], o));
      const float2 e = Two<T>::open(ends[s]);
      far[s] = !(fmaxf(-e.x, -e.y) <= kHalfMax);
      // (each end by itself: the sum of two finite ones may pass fp32)
      pair[s] = step_of(e.x, -e.y, !(fabsf(e.x) < INFINITY && fabsf(e.y) < INFINITY));
    }
    if constexpr (D == 64) pair[1] = pair[0], far[1] = far[0];
    if (is_q || !g.stored || w.head + i >= heads) continue;
    char* dst = (w.plane == 0 ? c.k_cache : c.v_cache) + row_at + (w.head + i) * c.head_stride;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t codes = far[s] ? far_codes<T>(make_uint4(word[s][0], word[s][1], word[s][2], word[s][3]), pair[s])
                                    : codes_of_words<T, false>(word[s], pair[s]);
      *reinterpret_cast<uint32_t*>(dst + at[s] / 2) = codes;
    }
    if (w.piece == 0) {
      char* sc = (w.plane == 0 ? c.k_scales : c.v_scales) + scale_at + (w.head + i) * c.scale_head_stride;
      if constexpr (D == 64) {
        *reinterpret_cast<__half2*>(sc) = pair[0];
      } else {
        *reinterpret_cast<uint2*>(sc) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&pair[0]), *reinterpret_cast<const uint32_t*>(&pair[1]));
      }
    }
  }
}

// The same for fp32 elements, for rows that are not aligned and for a rotary_dim that cuts a
// piece of 8: value by value, one head per thread.
template <typename T, typename TAB, int D>
__global__ void __launch_bounds__(kThreads) append4_narrow_kernel(const Params c) {
  const Place w = place<1>(c, c.kv_heads, c.q_heads, D / 16);
  const bool is_q = w.plane == 2;
  const char* src = is_q ? c.query + w.token * c.query_ts + w.head * c.query_hs
                         : (w.plane == 0 ? c.key + w.token * c.key_ts + w.head * c.key_hs
                                         : c.value + w.token * c.value_ts + w.head * c.value_hs);
  const Target g = target(c, w);
  const int at[2] = {8 * w.piece, D / 2 + 8 * w.piece};
  const bool here = w.real && g.turned && (is_q || g.stored);
  float x[2][8], low[2], high[2], odd[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (here) {
      rotated<T, TAB, 8, false>(reinterpret_cast<const T*>(src), at[s],
                                static_cast<const TAB*>(c.table) + g.position * c.rotary_dim,
                                w.plane == 1 ? 0 : c.rotary_dim, c.neox != 0, x[s]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[s][j] = 0.0f;
    }
    low[s] = INFINITY, high[s] = -INFINITY, odd[s] = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[s][j] = rnd<T>(x[s][j]);  // the row as the element type holds it
      low[s] = fminf(low[s], x[s][j]);
      high[s] = fmaxf(high[s], x[s][j]);
      odd[s] = fmaf(x[s][j], 0.0f, odd[s]);  // NaN once a value is NaN or infinite
    }
  }
  if (is_q && w.real) {
    T* out = reinterpret_cast<T*>(c.query_out + w.token * c.qo_ts + w.head * c.qo_hs);
#pragma unroll
    for (int s = 0; s < 2; ++s) store_n<T, 8, false>(out + at[s], x[s]);
  }
  if constexpr (D == 64) low[0] = fminf(low[0], low[1]), high[0] = fmaxf(high[0], high[1]), odd[0] += odd[1];
  constexpr int kGroups = D / kGroup;
  __half2 pair[2];
#pragma unroll
  for (int s = 0; s < kGroups; ++s) {
#pragma unroll
    for (int o = D / 32; o >= 1; o >>= 1) {
      low[s] = fminf(low[s], __shfl_xor_sync(0xffffffffu, low[s], o));
      high[s] = fmaxf(high[s], __shfl_xor_sync(0xffffffffu, high[s], o));
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, odd[s] != 0.0f);  // unequal also when NaN
    constexpr uint32_t kLanes = D / 16;
    pair[s] = step_of(low[s], high[s], (votes >> (threadIdx.x & (32u - kLanes))) & ((1u << kLanes) - 1u));
  }
  if constexpr (D == 64) pair[1] = pair[0];
  if (!here || is_q) return;
  char* dst = (w.plane == 0 ? c.k_cache : c.v_cache) + g.block * c.block_stride + g.row * c.slot_stride + w.head * c.head_stride;
#pragma unroll
  for (int s = 0; s < 2; ++s) *reinterpret_cast<uint32_t*>(dst + at[s] / 2) = codes_of(x[s], pair[s]);
  if (w.piece == 0) {
    __half2* sc = reinterpret_cast<__half2*>((w.plane == 0 ? c.k_scales : c.v_scales) + g.block * c.scale_block_stride +
                                             g.row * c.scale_slot_stride + w.head * c.scale_head_stride);
#pragma unroll
    for (int s = 0; s < kGroups; ++s) sc[s] = pair[s];
  }
}

struct GatherParams {
  const char* k_codes;
  const char* v_codes;
  const char* k_scales;
  const char* v_scales;
  int64_t block_stride, slot_stride, head_stride;
  int64_t scale_block_stride, scale_slot_stride, scale_head_stride;
  int64_t num_slots;
  int block_size;
  int heads, head_size;
  const int64_t* slots;
  int64_t tokens;
  char* out;
  int64_t out_plane_stride, out_token_stride, out_head_stride;
  int units, units_block, tokens_block, threads;
};

// 16 values of HPT heads of K or V per thread; a slot outside the cache reads as zeros.  Values past fp16's
// end are held there in fp16.
template <typename T, bool WIDE, int HPT>
__global__ void __launch_bounds__(kThreads) gather4_kernel(const GatherParams c) {
  const Place w = place<HPT>(c, c.heads, 0, c.head_size / 16);
  if (!w.real) return;
  const int64_t slot = __ldg(c.slots + w.token);
  const int d0 = w.piece * 16;
  uint2 codes[HPT];
  float2 pair[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) codes[i] = make_uint2(0, 0), pair[i] = make_float2(0.0f, 0.0f);
  if (slot >= 0 && slot < c.num_slots) {
    int block, row;
    split_slot(slot, c.block_size, block, row);
    const char* src = (w.plane ? c.v_codes : c.k_codes) + block * c.block_stride + row * c.slot_stride + d0 / 2;
    const char* sc = (w.plane ? c.v_scales : c.k_scales) + block * c.scale_block_stride + row * c.scale_slot_stride +
                     d0 / kGroup * static_cast<int>(sizeof(__half2));
#pragma unroll
    for (int i = 0; i < HPT; ++i)
      if (w.head + i < c.heads) {
        codes[i] = __ldg(reinterpret_cast<const uint2*>(src + (w.head + i) * c.head_stride));
        pair[i] = __half22float2(__ldg(reinterpret_cast<const __half2*>(sc + (w.head + i) * c.scale_head_stride)));
      }
  }
  T* out = reinterpret_cast<T*>(c.out + w.plane * c.out_plane_stride + w.token * c.out_token_stride) + d0;
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (w.head + i < c.heads) {
      T* row = reinterpret_cast<T*>(reinterpret_cast<char*>(out) + (w.head + i) * c.out_head_stride);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t word = s ? codes[i].y : codes[i].x;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = fmaf(static_cast<float>((word >> (4 * j)) & 15u), pair[i].x, pair[i].y);
        if constexpr (std::is_same<T, __half>::value) {
          // the step's rounding may take the highest code past fp16's end, which would read as an infinity
          if (fabsf(pair[i].y) + 15.0f * fabsf(pair[i].x) > kHalfMax) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (fabsf(y[j]) < INFINITY) y[j] = fminf(fmaxf(y[j], -kHalfMax), kHalfMax);
          }
        }
        store_n<T, 8, WIDE>(row + 8 * s, y);
      }
    }
}

// Threads of a block: the units of one token, or of several tokens side by side, and no idle
// ones behind them (32 + 8 + 8 heads: 96 units, 192 threads; 256 with 64 idle took 77 us, not 69).
template <typename P>
dim3 lay_out(P& c, int64_t units, int64_t tokens) {
  c.units = static_cast<int>(units);
  c.units_block = static_cast<int>(std::min<int64_t>(units, kThreads));
  c.tokens_block = kThreads / c.units_block;
  c.threads = (c.units_block * c.tokens_block + 31) / 32 * 32;
  return dim3(static_cast<unsigned>((tokens + c.tokens_block - 1) / c.tokens_block),
              static_cast<unsigned>((units + c.units_block - 1) / c.units_block));
}

// Units of a token: pieces of bundles of `hpt` heads.
inline int64_t units_of(int64_t kv_heads, int64_t q_heads, int64_t pieces, int64_t hpt) {
  return (2 * ((kv_heads + hpt - 1) / hpt) + (q_heads + hpt - 1) / hpt) * pieces;
}

// Whether a thread takes several heads: once one head per thread would fill the GPU's resident
// threads anyway.  Four of them for 16/32-bit pages and the read-back; two for 4-bit pages, which
// want the registers (20,011 tokens: 74 us with four).
inline bool more_heads(int64_t units, int64_t tokens) { return units * tokens >= int64_t(kSmCount) * 2048; }

int check_units(int64_t units) {
  CB_REQUIRE(units < (int64_t(1) << 23), "row too wide (%lld pieces)", (long long)units);
  return CB_OK;
}

template <typename T, typename TAB, int D>
void launch4(const Params& c, dim3 grid, bool wide, bool more, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    const bool extra = c.neox && c.rotary_dim > 0 && c.rotary_dim < D;
    if (wide) {
      if (extra)
        more ? append4_kernel<T, TAB, D, true, 2><<<grid, c.threads, 0, s>>>(c)
             : append4_kernel<T, TAB, D, true, 1><<<grid, c.threads, 0, s>>>(c);
      else
        more ? append4_kernel<T, TAB, D, false, 2><<<grid, c.threads, 0, s>>>(c)
             : append4_kernel<T, TAB, D, false, 1><<<grid, c.threads, 0, s>>>(c);
      return;
    }
  }
  append4_narrow_kernel<T, TAB, D><<<grid, c.threads, 0, s>>>(c);
}

template <bool FOUR, typename T, typename TAB>
int launch(Params& c, bool wide, cudaStream_t s) {
  constexpr int kPiece = FOUR ? 16 : 32 / static_cast<int>(sizeof(T));
  const int64_t pieces = FOUR || wide ? c.head_size / kPiece : c.head_size;
  const int64_t units = units_of(c.kv_heads, c.q_heads, pieces, 1);
  const int rc = check_units(units);
  if (rc != CB_OK) return rc;
  const bool more = wide && more_heads(units, c.tokens);
  const dim3 grid = lay_out(c, more ? units_of(c.kv_heads, c.q_heads, pieces, FOUR ? 2 : 4) : units, c.tokens);
  if constexpr (FOUR) {
    if (c.head_size == 64)
      launch4<T, TAB, 64>(c, grid, wide, more, s);
    else
      launch4<T, TAB, 128>(c, grid, wide, more, s);
  } else {
    if (!wide)
      append_narrow_kernel<T, TAB><<<grid, c.threads, 0, s>>>(c);
    else if (more)
      append_kernel<T, TAB, 4><<<grid, c.threads, 0, s>>>(c);
    else
      append_kernel<T, TAB, 1><<<grid, c.threads, 0, s>>>(c);
  }
  return launch_status(FOUR ? "cb_append_paged_kv4" : "cb_append_paged_kv");
}

template <bool FOUR>
int dispatch(Params& c, int dtype, int table_dtype, bool wide, cudaStream_t s) {
  const bool f32_table = table_dtype == CB_DTYPE_FP32;
  switch (dtype) {
    case CB_DTYPE_BF16:
      return f32_table ? launch<FOUR, __nv_bfloat16, float>(c, wide, s) : launch<FOUR, __nv_bfloat16, __nv_bfloat16>(c, wide, s);
    case CB_DTYPE_FP16:
      return f32_table ? launch<FOUR, __half, float>(c, wide, s) : launch<FOUR, __half, __half>(c, wide, s);
    default:
      return launch<FOUR, float, float>(c, wide, s);
  }
}

template <typename T>
void launch_gather4(GatherParams& c, bool wide, cudaStream_t s) {
  const int64_t pieces = c.head_size / 16, units = units_of(c.heads, 0, pieces, 1);
  const bool four = wide && more_heads(units, c.tokens);
  const dim3 grid = lay_out(c, four ? units_of(c.heads, 0, pieces, 4) : units, c.tokens);
  if (!wide)
    gather4_kernel<T, false, 1><<<grid, c.threads, 0, s>>>(c);
  else if (four)
    gather4_kernel<T, true, 4><<<grid, c.threads, 0, s>>>(c);
  else
    gather4_kernel<T, true, 1><<<grid, c.threads, 0, s>>>(c);
}

// What both appends check of their rows and of the rotation.
int check_rows(const Params& c, int dtype, int table_dtype, int64_t num_blocks) {
  CB_SUPPORTED(dtype_bytes(dtype) != 0, "unsupported element type code %d", dtype);
  CB_REQUIRE(c.tokens >= 0 && c.kv_heads > 0 && c.head_size > 0 && num_blocks >= 0 && c.block_size > 0 && c.q_heads >= 0,
             "negative or zero size");
  CB_REQUIRE(c.tokens < (int64_t(1) << 31) && num_blocks < (int64_t(1) << 31) && c.block_size < (int64_t(1) << 22),
             "size out of range");
  CB_REQUIRE(c.rotary_dim >= 0 && c.rotary_dim <= c.head_size && c.rotary_dim % 2 == 0,
             "rotary_dim %d does not fit the head size %d", c.rotary_dim, c.head_size);
  if (c.rotary_dim > 0)
    CB_SUPPORTED(table_dtype == CB_DTYPE_FP32 || table_dtype == dtype, "the cos/sin table must be fp32 or of the keys' type");
  if (c.tokens == 0) return CB_OK;
  CB_REQUIRE(c.key && c.value && c.k_cache && c.v_cache && c.slots, "null pointer argument");
  CB_REQUIRE(c.q_heads == 0 || (c.query && c.query_out), "null query pointer");
  CB_REQUIRE(c.rotary_dim == 0 || (c.positions && c.table && c.max_position >= 0), "rotation needs positions and a table");
  const uint64_t esize = static_cast<uint64_t>(dtype_bytes(dtype));
  const uint64_t acc = reinterpret_cast<uint64_t>(c.key) | reinterpret_cast<uint64_t>(c.value) |
                       reinterpret_cast<uint64_t>(c.query) | reinterpret_cast<uint64_t>(c.query_out) | (uint64_t)c.key_ts |
                       (uint64_t)c.key_hs | (uint64_t)c.value_ts | (uint64_t)c.value_hs | (uint64_t)c.query_ts |
                       (uint64_t)c.query_hs | (uint64_t)c.qo_ts | (uint64_t)c.qo_hs;
  CB_REQUIRE((acc & (esize - 1)) == 0, "rows must be aligned to their element size");
  if (c.rotary_dim > 0)
    CB_REQUIRE((reinterpret_cast<uint64_t>(c.table) & (uint64_t)(dtype_bytes(table_dtype) - 1)) == 0,
               "the cos/sin table must be aligned to its element size");
  return CB_OK;
}

// Whether rows go in whole aligned pieces: `n` values a piece, `row` values a multiple of
// which a head holds, and no piece across rotary_dim or (neox) its half.
bool wide_rows(const Params& c, int n, int row, uint64_t more) {
  const uint64_t acc = more | reinterpret_cast<uint64_t>(c.key) | reinterpret_cast<uint64_t>(c.value) |
                       reinterpret_cast<uint64_t>(c.query) | reinterpret_cast<uint64_t>(c.query_out) | (uint64_t)c.key_ts |
                       (uint64_t)c.key_hs | (uint64_t)c.value_ts | (uint64_t)c.value_hs | (uint64_t)c.query_ts |
                       (uint64_t)c.query_hs | (uint64_t)c.qo_ts | (uint64_t)c.qo_hs | reinterpret_cast<uint64_t>(c.table);
  if ((acc & 15u) != 0 || c.head_size % row != 0) return false;
  return c.neox ? c.rotary_dim % (2 * n) == 0 : c.rotary_dim % n == 0 && (c.rotary_dim / 2) % n == 0;
}

int check_pages4(int64_t block_stride, int64_t slot_stride, int64_t head_stride, int64_t scale_block_stride,
                 int64_t scale_slot_stride, int64_t scale_head_stride, const void* k_codes, const void* v_codes,
                 const void* k_scales, const void* v_scales, int64_t head_size) {
  CB_SUPPORTED(head_size == 64 || head_size == 128, "4-bit pages hold heads of 64 or 128 values (got %lld)",
               (long long)head_size);
  CB_REQUIRE(k_codes && v_codes && k_scales && v_scales, "null page pointer");
  const uint64_t codes = reinterpret_cast<uint64_t>(k_codes) | reinterpret_cast<uint64_t>(v_codes) |
                         (uint64_t)block_stride | (uint64_t)slot_stride | (uint64_t)head_stride;
  CB_REQUIRE((codes & 15u) == 0, "4-bit rows must be 16-byte aligned");
  const uint64_t scales = reinterpret_cast<uint64_t>(k_scales) | reinterpret_cast<uint64_t>(v_scales) |
                          (uint64_t)scale_block_stride | (uint64_t)scale_slot_stride | (uint64_t)scale_head_stride;
  CB_REQUIRE((scales & (uint64_t)(head_size / 16 - 1)) == 0, "the steps of a 4-bit row must be %lld-byte aligned",
             (long long)(head_size / 16));
  return CB_OK;
}

}  // namespace append
}  // namespace cb

using namespace cb;

extern "C" int cb_append_paged_kv(const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                                  int64_t value_token_stride, int64_t value_head_stride, const void* query,
                                  int64_t query_token_stride, int64_t query_head_stride, void* query_out,
                                  int64_t query_out_token_stride, int64_t query_out_head_stride, int64_t num_tokens,
                                  int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size, int dtype,
                                  const int64_t* positions, const void* cos_sin, int cos_sin_dtype, int64_t max_position,
                                  int64_t rotary_dim, int is_neox, void* k_cache, void* v_cache, int64_t block_stride,
                                  int64_t slot_stride, int64_t head_stride, int64_t num_blocks, int64_t block_size,
                                  const int64_t* slots, void* stream) {
  CB_BIND(stream, k_cache);
  CB_REQUIRE(num_kv_heads < 65536 && num_q_heads < 65536 && head_size <= 65536 && rotary_dim <= 65536 &&
                 block_size < (int64_t(1) << 22),
             "size out of range");
  append::Params c{};
  c.key = static_cast<const char*>(key), c.value = static_cast<const char*>(value);
  c.query = static_cast<const char*>(query), c.query_out = static_cast<char*>(query_out);
  c.key_ts = key_token_stride, c.key_hs = key_head_stride, c.value_ts = value_token_stride, c.value_hs = value_head_stride;
  c.query_ts = query_token_stride, c.query_hs = query_head_stride;
  c.qo_ts = query_out_token_stride, c.qo_hs = query_out_head_stride;
  c.tokens = num_tokens;
  c.q_heads = static_cast<int>(num_q_heads), c.kv_heads = static_cast<int>(num_kv_heads);
  c.head_size = static_cast<int>(head_size);
  c.positions = positions, c.table = cos_sin, c.max_position = max_position;
  c.rotary_dim = static_cast<int>(rotary_dim), c.neox = is_neox;
  c.k_cache = static_cast<char*>(k_cache), c.v_cache = static_cast<char*>(v_cache);
  c.block_stride = block_stride, c.slot_stride = slot_stride, c.head_stride = head_stride;
  c.num_slots = num_blocks * block_size, c.block_size = static_cast<int>(block_size), c.slots = slots;
  int rc = append::check_rows(c, dtype, cos_sin_dtype, num_blocks);
  if (rc != CB_OK || num_tokens == 0) return rc;
  const uint64_t pages = reinterpret_cast<uint64_t>(k_cache) | reinterpret_cast<uint64_t>(v_cache) | (uint64_t)block_stride |
                         (uint64_t)slot_stride | (uint64_t)head_stride;
  CB_REQUIRE((pages & (uint64_t)(dtype_bytes(dtype) - 1)) == 0, "pages must be aligned to their element size");
  const int piece = 16 / dtype_bytes(dtype);
  const bool wide = append::wide_rows(c, piece, 2 * piece, pages);
  return append::dispatch<false>(c, dtype, cos_sin_dtype, wide, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int cb_append_paged_kv4(const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                                   int64_t value_token_stride, int64_t value_head_stride, const void* query,
                                   int64_t query_token_stride, int64_t query_head_stride, void* query_out,
                                   int64_t query_out_token_stride, int64_t query_out_head_stride, int64_t num_tokens,
                                   int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size, int dtype,
                                   const int64_t* positions, const void* cos_sin, int cos_sin_dtype, int64_t max_position,
                                   int64_t rotary_dim, int is_neox, void* k_codes, void* v_codes, int64_t block_stride,
                                   int64_t slot_stride, int64_t head_stride, void* k_scales, void* v_scales,
                                   int64_t scale_block_stride, int64_t scale_slot_stride, int64_t scale_head_stride,
                                   int64_t num_blocks, int64_t block_size, const int64_t* slots, void* stream) {
  CB_BIND(stream, k_codes);
  CB_REQUIRE(num_kv_heads < 65536 && num_q_heads < 65536 && head_size <= 65536 && rotary_dim <= 65536 &&
                 block_size < (int64_t(1) << 22),
             "size out of range");
  append::Params c{};
  c.key = static_cast<const char*>(key), c.value = static_cast<const char*>(value);
  c.query = static_cast<const char*>(query), c.query_out = static_cast<char*>(query_out);
  c.key_ts = key_token_stride, c.key_hs = key_head_stride, c.value_ts = value_token_stride, c.value_hs = value_head_stride;
  c.query_ts = query_token_stride, c.query_hs = query_head_stride;
  c.qo_ts = query_out_token_stride, c.qo_hs = query_out_head_stride;
  c.tokens = num_tokens;
  c.q_heads = static_cast<int>(num_q_heads), c.kv_heads = static_cast<int>(num_kv_heads);
  c.head_size = static_cast<int>(head_size);
  c.positions = positions, c.table = cos_sin, c.max_position = max_position;
  c.rotary_dim = static_cast<int>(rotary_dim), c.neox = is_neox;
  c.k_cache = static_cast<char*>(k_codes), c.v_cache = static_cast<char*>(v_codes);
  c.block_stride = block_stride, c.slot_stride = slot_stride, c.head_stride = head_stride;
  c.k_scales = static_cast<char*>(k_scales), c.v_scales = static_cast<char*>(v_scales);
  c.scale_block_stride = scale_block_stride, c.scale_slot_stride = scale_slot_stride;
  c.scale_head_stride = scale_head_stride;
  c.num_slots = num_blocks * block_size, c.block_size = static_cast<int>(block_size), c.slots = slots;
  int rc = append::check_rows(c, dtype, cos_sin_dtype, num_blocks);
  if (rc != CB_OK || num_tokens == 0) return rc;
  rc = append::check_pages4(block_stride, slot_stride, head_stride, scale_block_stride, scale_slot_stride,
                            scale_head_stride, k_codes, v_codes, k_scales, v_scales, head_size);
  if (rc != CB_OK) return rc;
  return append::dispatch<true>(c, dtype, cos_sin_dtype, dtype != CB_DTYPE_FP32 && append::wide_rows(c, 8, 16, 0),
                                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int cb_gather_paged_kv4(const void* k_codes, const void* v_codes, int64_t block_stride, int64_t slot_stride,
                                   int64_t head_stride, const void* k_scales, const void* v_scales,
                                   int64_t scale_block_stride, int64_t scale_slot_stride, int64_t scale_head_stride,
                                   int64_t num_blocks, int64_t block_size, int64_t num_heads, int64_t head_size,
                                   const int64_t* slots, int64_t num_tokens, void* out, int64_t out_plane_stride,
                                   int64_t out_token_stride, int64_t out_head_stride, int dtype, void* stream) {
  CB_BIND(stream, out);
  CB_SUPPORTED(dtype_bytes(dtype) != 0, "unsupported element type code %d", dtype);
  CB_REQUIRE(num_tokens >= 0 && num_blocks >= 0 && block_size > 0 && num_heads > 0, "negative or zero size");
  CB_REQUIRE(num_tokens < (int64_t(1) << 31) && num_blocks < (int64_t(1) << 31) && block_size < (int64_t(1) << 22) &&
                 num_heads < 65536,
             "size out of range");
  if (num_tokens == 0) return CB_OK;
  CB_REQUIRE(slots && out, "null pointer argument");
  int rc = append::check_pages4(block_stride, slot_stride, head_stride, scale_block_stride, scale_slot_stride,
                                scale_head_stride, k_codes, v_codes, k_scales, v_scales, head_size);
  if (rc != CB_OK) return rc;
  const uint64_t acc = reinterpret_cast<uint64_t>(out) | (uint64_t)out_plane_stride | (uint64_t)out_token_stride |
                       (uint64_t)out_head_stride;
  CB_REQUIRE((acc & (uint64_t)(dtype_bytes(dtype) - 1)) == 0, "output rows must be aligned to their element size");
  append::GatherParams c{};
  c.k_codes = static_cast<const char*>(k_codes), c.v_codes = static_cast<const char*>(v_codes);
  c.k_scales = static_cast<const char*>(k_scales), c.v_scales = static_cast<const char*>(v_scales);
  c.block_stride = block_stride, c.slot_stride = slot_stride, c.head_stride = head_stride;
  c.scale_block_stride = scale_block_stride, c.scale_slot_stride = scale_slot_stride;
  c.scale_head_stride = scale_head_stride;
  c.num_slots = num_blocks * block_size, c.block_size = static_cast<int>(block_size);
  c.heads = static_cast<int>(num_heads), c.head_size = static_cast<int>(head_size);
  c.slots = slots, c.tokens = num_tokens, c.out = static_cast<char*>(out);
  c.out_plane_stride = out_plane_stride, c.out_token_stride = out_token_stride, c.out_head_stride = out_head_stride;
  rc = append::check_units(append::units_of(num_heads, 0, head_size / 16, 1));
  if (rc != CB_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = (acc & 15u) == 0;
  if (dtype == CB_DTYPE_BF16)
    append::launch_gather4<__nv_bfloat16>(c, wide, s);
  else if (dtype == CB_DTYPE_FP16)
    append::launch_gather4<__half>(c, wide, s);
  else
    append::launch_gather4<float>(c, wide, s);
  return launch_status("cb_gather_paged_kv4");
}
