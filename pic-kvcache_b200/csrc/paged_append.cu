// Fresh keys and values into the paged cache, rotated on the way, and the
// 4-bit form of the pages with its read-back.
//
// Rotation at position p (r = rotary_dim; cos_p, sin_p the table's row):
//   neox    y[i] = x[i] cos_p[i] - x[i + r/2] sin_p[i]
//           y[i + r/2] = x[i + r/2] cos_p[i] + x[i] sin_p[i]          i < r/2
//   GPT-J   the same with the partners 2i and 2i + 1
// The table is read in its own type, both products and the sum are rounded to
// fp32 one by one (no contraction), and the result is rounded once to the
// element type: a cached row is the same bits whatever launch wrote it.
//
// 4-bit rows: every 64 values of a row share a lowest value and a step,
//   low = fp16(min x), step = fp16((max x - low') / 15)   (low' = the fp32 minimum)
//   code = clamp(rint((x - low) * (1 / step)), 0, 15),  value = low + step code
// fp16 (11 bits) rather than bf16 for the pair: its rounding is 2^-12 of the
// lowest value, far below a step, where bf16's 2^-9 can exceed one in a channel
// with a large offset.  Values beyond fp16's range are held at +-65504; a group
// with a NaN or an infinity gets a NaN step, so it reads as NaN.  Two codes to
// a byte, the lower dimension in the low nibble.
//
// What bounds them: HBM at long prompts, the launch at decode sizes.  One
// thread holds one 16-byte piece of an output row (8 values of a 4-bit row) and
// reads the partner piece through L1; threads of a block run over one token's
// pieces first, so rows are read and written whole.
#include <algorithm>
#include <type_traits>

#include "cb_common.cuh"

namespace cb {
namespace append {

constexpr int kThreads = 256;
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
  int64_t num_slots, block_size;
  const int64_t* slots;
  // thread layout: units of a token, units and tokens per block
  int units, units_block, tokens_block;
};

// slot -> (block, row), with the short division wherever it does.
__device__ __forceinline__ void split_slot(int64_t slot, int64_t block_size, int64_t& block, int64_t& row) {
  if ((slot | block_size) >> 31) {
    block = slot / block_size;
    row = slot - block * block_size;
  } else {
    const uint32_t b = static_cast<uint32_t>(slot) / static_cast<uint32_t>(block_size);
    block = b;
    row = static_cast<uint32_t>(slot) - b * static_cast<uint32_t>(block_size);
  }
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

// 8 values of a 4-bit row: the eight lanes of a group agree on its lowest value and step.
// Every lane of the warp calls this.
__device__ __forceinline__ uint32_t encode8(const float (&y)[8], __half2& pair) {
  float low = INFINITY, high = -INFINITY;
  bool bad = false;
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    bad |= (__float_as_uint(y[j]) & 0x7f800000u) == 0x7f800000u;
    x[j] = fminf(fmaxf(y[j], -kHalfMax), kHalfMax);
    low = fminf(low, x[j]);
    high = fmaxf(high, x[j]);
  }
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const uint32_t votes = __ballot_sync(0xffffffffu, bad);
  const __half step_h = __float2half_rn(__fmul_rn(__fsub_rn(high, low), 1.0f / 15.0f));
  const __half low_h = __float2half_rn(low);
  const float step = __half2float(step_h);
  const float inverse = step > 0.0f ? __frcp_rn(step) : 0.0f;
  const float base = __half2float(low_h);
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[j], base), inverse)), 0.0f), 15.0f);
    codes |= static_cast<uint32_t>(c) << (4 * j);
  }
  const bool group_bad = (votes >> (threadIdx.x & 24u)) & 0xffu;
  pair = __halves2half2(group_bad ? __ushort_as_half(0x7e00) : step_h, low_h);
  return codes;
}

// One piece (N values) of one row of K, V or Q per thread.
template <typename T, typename TAB, int N, bool WIDE, bool FOUR>
__global__ void __launch_bounds__(kThreads) append_kernel(const Params c) {
  const int tok = threadIdx.x / c.units_block;
  const int unit = blockIdx.y * c.units_block + (threadIdx.x - tok * c.units_block);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * c.tokens_block + tok;
  const bool real = tok < c.tokens_block && unit < c.units && t < c.tokens;
  const int pieces = c.head_size / N;
  const int kv_units = c.kv_heads * pieces;
  // plane 0: K, 1: V, 2: Q
  const int plane = unit < kv_units ? 0 : (unit < 2 * kv_units ? 1 : 2);
  const int in_plane = unit - plane * kv_units;
  const int head = in_plane / pieces;
  const int d0 = (in_plane - head * pieces) * N;

  int64_t slot = -1;
  bool turned = true;  // the position lies inside the table
  const TAB* table = nullptr;
  if (real) {
    if (plane < 2) slot = c.slots[t];
    if (plane != 1 && c.rotary_dim > 0) {
      const int64_t pos = c.positions[t];
      turned = pos >= 0 && pos < c.max_position;
      table = static_cast<const TAB*>(c.table) + pos * c.rotary_dim;
    }
  }
  // V goes with its K: a position outside the table leaves the whole slot as it was
  if (real && plane == 1 && c.rotary_dim > 0) {
    const int64_t pos = c.positions[t];
    turned = pos >= 0 && pos < c.max_position;
  }
  const bool stored = real && plane < 2 && slot >= 0 && slot < c.num_slots && turned;
  float y[N];
  if (real && plane == 2) {
    T* out = reinterpret_cast<T*>(c.query_out + t * c.qo_ts + head * c.qo_hs) + d0;
    if (turned) {
      rotated<T, TAB, N, WIDE>(reinterpret_cast<const T*>(c.query + t * c.query_ts + head * c.query_hs), d0, table,
                               c.rotary_dim, c.neox != 0, y);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = 0.0f;
    }
    store_n<T, N, WIDE>(out, y);
  } else if (stored) {
    if (plane == 0)
      rotated<T, TAB, N, WIDE>(reinterpret_cast<const T*>(c.key + t * c.key_ts + head * c.key_hs), d0, table,
                               c.rotary_dim, c.neox != 0, y);
    else
      load_n<T, N, WIDE>(reinterpret_cast<const T*>(c.value + t * c.value_ts + head * c.value_hs) + d0, y);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = 0.0f;
  }
  if constexpr (!FOUR) {
    if (!stored) return;
    int64_t block, row;
    split_slot(slot, c.block_size, block, row);
    char* dst = (plane == 0 ? c.k_cache : c.v_cache) + block * c.block_stride + row * c.slot_stride + head * c.head_stride;
    store_n<T, N, WIDE>(reinterpret_cast<T*>(dst) + d0, y);
  } else {
    static_assert(N == 8, "eight lanes to a group of 64");
    // the row as the element type holds it: the 4-bit pages hold what 16-bit pages would
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = rnd<T>(y[j]);
    __half2 pair;
    const uint32_t codes = encode8(y, pair);
    if (!stored) return;
    int64_t block, row;
    split_slot(slot, c.block_size, block, row);
    char* dst = (plane == 0 ? c.k_cache : c.v_cache) + block * c.block_stride + row * c.slot_stride + head * c.head_stride;
    *reinterpret_cast<uint32_t*>(dst + d0 / 2) = codes;
    if ((d0 & (kGroup - 1)) == 0) {
      char* sc = (plane == 0 ? c.k_scales : c.v_scales) + block * c.scale_block_stride + row * c.scale_slot_stride +
                 head * c.scale_head_stride;
      *(reinterpret_cast<__half2*>(sc) + d0 / kGroup) = pair;
    }
  }
}

struct GatherParams {
  const char* k_codes;
  const char* v_codes;
  const char* k_scales;
  const char* v_scales;
  int64_t block_stride, slot_stride, head_stride;
  int64_t scale_block_stride, scale_slot_stride, scale_head_stride;
  int64_t num_slots, block_size;
  int heads, head_size;
  const int64_t* slots;
  int64_t tokens;
  char* out;
  int64_t out_plane_stride, out_token_stride, out_head_stride;
  int units, units_block, tokens_block;
};

// 8 values of one row of K or V per thread; a slot outside the cache reads as zeros.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) gather4_kernel(const GatherParams c) {
  const int tok = threadIdx.x / c.units_block;
  const int unit = blockIdx.y * c.units_block + (threadIdx.x - tok * c.units_block);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * c.tokens_block + tok;
  if (tok >= c.tokens_block || unit >= c.units || t >= c.tokens) return;
  const int pieces = c.head_size / 8;
  const int row_piece = unit / pieces;
  const int d0 = (unit - row_piece * pieces) * 8;
  const int plane = row_piece >= c.heads;
  const int head = row_piece - plane * c.heads;
  const int64_t slot = c.slots[t];
  float y[8];
  if (slot >= 0 && slot < c.num_slots) {
    int64_t block, row;
    split_slot(slot, c.block_size, block, row);
    const char* src = (plane ? c.v_codes : c.k_codes) + block * c.block_stride + row * c.slot_stride + head * c.head_stride;
    const char* sc = (plane ? c.v_scales : c.k_scales) + block * c.scale_block_stride + row * c.scale_slot_stride +
                     head * c.scale_head_stride;
    const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>(src + d0 / 2));
    const float2 pair = __half22float2(__ldg(reinterpret_cast<const __half2*>(sc) + d0 / kGroup));
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = fmaf(static_cast<float>((codes >> (4 * j)) & 15u), pair.x, pair.y);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = 0.0f;
  }
  store_n<T, 8, WIDE>(
      reinterpret_cast<T*>(c.out + plane * c.out_plane_stride + t * c.out_token_stride + head * c.out_head_stride) + d0, y);
}

// Threads of a block: the units of one token, or of several tokens side by side.
template <typename P>
dim3 lay_out(P& c, int64_t units, int64_t tokens) {
  c.units = static_cast<int>(units);
  c.units_block = static_cast<int>(std::min<int64_t>(units, kThreads));
  c.tokens_block = kThreads / c.units_block;
  return dim3(static_cast<unsigned>((tokens + c.tokens_block - 1) / c.tokens_block),
              static_cast<unsigned>((units + c.units_block - 1) / c.units_block));
}

template <bool FOUR, typename T, typename TAB>
int launch(Params& c, bool wide, cudaStream_t s) {
  constexpr int kWide = FOUR ? 8 : 16 / static_cast<int>(sizeof(T));
  constexpr int kNarrow = FOUR ? 8 : 1;
  const int64_t n = wide ? kWide : kNarrow;
  const int64_t units = (2 * static_cast<int64_t>(c.kv_heads) + c.q_heads) * (c.head_size / n);
  CB_REQUIRE(units < (int64_t(1) << 23), "row too wide (%lld pieces)", (long long)units);
  const dim3 grid = lay_out(c, units, c.tokens);
  if (wide)
    append_kernel<T, TAB, kWide, true, FOUR><<<grid, kThreads, 0, s>>>(c);
  else
    append_kernel<T, TAB, kNarrow, false, FOUR><<<grid, kThreads, 0, s>>>(c);
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

// What both appends check of their rows and of the rotation.
int check_rows(const Params& c, int dtype, int table_dtype, int64_t num_blocks) {
  CB_SUPPORTED(dtype_bytes(dtype) != 0, "unsupported element type code %d", dtype);
  CB_REQUIRE(c.tokens >= 0 && c.kv_heads > 0 && c.head_size > 0 && num_blocks >= 0 && c.block_size > 0 && c.q_heads >= 0,
             "negative or zero size");
  CB_REQUIRE(c.tokens < (int64_t(1) << 31) && num_blocks < (int64_t(1) << 40) && c.block_size < (int64_t(1) << 22),
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

// Whether pieces of `n` values can be read whole: aligned rows, and no piece across
// rotary_dim or (neox) its half.  Rows that cannot go value by value; measured for one
// 8,192-token prompt of 8 KV heads beside the wide form: see below the launch.
bool wide_rows(const Params& c, int n, uint64_t more) {
  const uint64_t acc = more | reinterpret_cast<uint64_t>(c.key) | reinterpret_cast<uint64_t>(c.value) |
                       reinterpret_cast<uint64_t>(c.query) | reinterpret_cast<uint64_t>(c.query_out) | (uint64_t)c.key_ts |
                       (uint64_t)c.key_hs | (uint64_t)c.value_ts | (uint64_t)c.value_hs | (uint64_t)c.query_ts |
                       (uint64_t)c.query_hs | (uint64_t)c.qo_ts | (uint64_t)c.qo_hs | reinterpret_cast<uint64_t>(c.table);
  if ((acc & 15u) != 0 || c.head_size % n != 0) return false;
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
  CB_REQUIRE(num_kv_heads < 65536 && num_q_heads < 65536 && head_size <= 65536 && rotary_dim <= 65536, "size out of range");
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
  c.num_slots = num_blocks * block_size, c.block_size = block_size, c.slots = slots;
  int rc = append::check_rows(c, dtype, cos_sin_dtype, num_blocks);
  if (rc != CB_OK || num_tokens == 0) return rc;
  const uint64_t pages = reinterpret_cast<uint64_t>(k_cache) | reinterpret_cast<uint64_t>(v_cache) | (uint64_t)block_stride |
                         (uint64_t)slot_stride | (uint64_t)head_stride;
  CB_REQUIRE((pages & (uint64_t)(dtype_bytes(dtype) - 1)) == 0, "pages must be aligned to their element size");
  const bool wide = append::wide_rows(c, 16 / dtype_bytes(dtype), pages);
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
  CB_REQUIRE(num_kv_heads < 65536 && num_q_heads < 65536 && head_size <= 65536 && rotary_dim <= 65536, "size out of range");
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
  c.num_slots = num_blocks * block_size, c.block_size = block_size, c.slots = slots;
  int rc = append::check_rows(c, dtype, cos_sin_dtype, num_blocks);
  if (rc != CB_OK || num_tokens == 0) return rc;
  rc = append::check_pages4(block_stride, slot_stride, head_stride, scale_block_stride, scale_slot_stride,
                            scale_head_stride, k_codes, v_codes, k_scales, v_scales, head_size);
  if (rc != CB_OK) return rc;
  return append::dispatch<true>(c, dtype, cos_sin_dtype, append::wide_rows(c, 8, 0), reinterpret_cast<cudaStream_t>(stream));
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
  CB_REQUIRE(num_tokens < (int64_t(1) << 31) && num_blocks < (int64_t(1) << 40) && block_size < (int64_t(1) << 22) &&
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
  c.num_slots = num_blocks * block_size, c.block_size = block_size;
  c.heads = static_cast<int>(num_heads), c.head_size = static_cast<int>(head_size);
  c.slots = slots, c.tokens = num_tokens, c.out = static_cast<char*>(out);
  c.out_plane_stride = out_plane_stride, c.out_token_stride = out_token_stride, c.out_head_stride = out_head_stride;
  const dim3 grid = append::lay_out(c, 2 * num_heads * (head_size / 8), num_tokens);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = (acc & 15u) == 0;
  switch (dtype) {
    case CB_DTYPE_BF16:
      wide ? append::gather4_kernel<__nv_bfloat16, true><<<grid, append::kThreads, 0, s>>>(c)
           : append::gather4_kernel<__nv_bfloat16, false><<<grid, append::kThreads, 0, s>>>(c);
      break;
    case CB_DTYPE_FP16:
      wide ? append::gather4_kernel<__half, true><<<grid, append::kThreads, 0, s>>>(c)
           : append::gather4_kernel<__half, false><<<grid, append::kThreads, 0, s>>>(c);
      break;
    default:
      wide ? append::gather4_kernel<float, true><<<grid, append::kThreads, 0, s>>>(c)
           : append::gather4_kernel<float, false><<<grid, append::kThreads, 0, s>>>(c);
      break;
  }
  return launch_status("cb_gather_paged_kv4");
}
