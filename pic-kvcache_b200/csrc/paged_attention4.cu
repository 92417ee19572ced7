// Attention of single tokens (or a few per sequence) over 4-bit pages.
//
// A row of the pages holds, per group G of 64 dimensions, codes c and a pair
// (step, low); its values are low_G + step_G c.  For a query q of KV head h and
// the key at position j, with everything in the log2 domain,
//   w_j  = scale log2e (sum_G step_jG (q . c_j)_G + sum_G low_jG (sum q)_G)
//   p_j  = 2^(w_j - M)                             M: a running reference per row
//   out  = (sum_j p_j step'_jG c'_j + sum_j p_j low'_jG) / sum_j p_j
// so no value is ever built: the products are of codes, which are exact in fp16,
// and the steps and lowest values enter as one factor and one term per key.
//
// Products: mma.sync m16n8k16 in fp16 with fp32 sums, operands in registers.
// The work is bound by reading the pages (0.56 bytes for 2 x 8 products of a
// row's value), and tcgen05 would want every code widened and stored to shared
// memory first: 46 codes a clock and SM at the memory's rate are 92 bytes of its
// 128, before any is read.  From registers a code costs under one instruction:
//   * a masked word is two fp16 at once: a nibble at bits 0-3 of a half is the
//     subnormal c 2^-24, at bits 4-7 c 2^-20, both exact in the tensor core.  The
//     factor 2^24 goes into the row's factor, the odd nibbles' 16 into q (K) or
//     into the output row (V).
//   * K: the 16 keys of a tile are the M rows, the query rows the N columns
//     (8: a whole group of query heads usually fits), the dimensions of one group
//     the K steps.  q is scaled per row by a power of two so that its largest
//     value is in [2^14, 2^15): bf16 and fp16 values are exact in fp16 down to
//     2^-28 of it.
//   * V: the dimensions are the M rows, the keys the K steps, P the B operand; a
//     byte permute pairs the same nibble of two keys.  P step'_G is rounded to
//     fp16 (11 bits: 2^-12 relative, against the 2^-9 of a bf16 output) once per
//     group and transposed by movmatrix.  M also carries the exponent of the
//     largest step' so that a factor stays in fp16's range whatever the values'
//     size: at most 2^15, 2^10 when M is set.
// Sums, maxima, steps and the low terms are fp32.
//
// Memory: a warp takes tiles of 32 keys of one KV head through a ring of its
// own, filled by cp.async (16 bytes of a row per lane; a page's rows may lie
// anywhere and end anywhere in a tile), so no barrier joins the warps inside a
// piece of work.  Rows are swizzled (32-byte halves by row) and the tile's rows
// permuted (pi) so that neither product's fragment loads conflict.
//
// Split: all (sequence, KV head, row block) pieces form one line of tiles, cut
// into equal shares, one per CTA, whatever the lengths are; the cut is found on
// the device from the lengths.  The first and last piece of a share may be
// parts; parts go to the workspace and a second launch joins them in order, so a
// result does not depend on timing.
#include <algorithm>

#include "cb_common.cuh"

namespace cb {
namespace att4 {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTileKeys = 32;    // keys of a warp's stage
constexpr int kMinShare = 8;     // tiles: one per warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSetRoom = 10.0f;   // a factor p step' is at most 2^10 when M is set,
constexpr float kMostRoom = 15.0f;  // and 2^15 before M moves

struct Params {
  const char* query;
  int64_t query_ts, query_hs;  // bytes
  char* out;
  int64_t out_ts, out_hs;
  int64_t tokens;
  const int32_t* start;  // null: one token per sequence
  const int32_t* lens;
  const int32_t* table;
  int64_t table_stride;  // entries
  int num_seqs, width, heads_kv, groups;
  const char* codes[2];
  const char* scales[2];
  int64_t block_stride, slot_stride, head_stride;
  int64_t scale_block_stride, scale_slot_stride, scale_head_stride;
  int64_t num_blocks;
  int block_size;
  float scale_log2;  // scale * log2(e)
  bool aligned;      // query rows in whole 16-byte vectors
  float* parts;      // [ctas][2][rows][D + 2]
  int4* meta;        // [ctas]: (parts that follow, sequence, KV head, row block); x < 0: none
};

// One sequence's share of the line.
struct Seq {
  int first_token, tokens, len;
  int row_blocks, tiles;  // per piece
  int64_t work;           // tiles of all its pieces
};
template <int ROWS>
__device__ __forceinline__ Seq sequence(const Params& c, int i) {
  Seq s;
  int64_t a = i, b = i + 1;
  if (c.start != nullptr) a = __ldg(c.start + i), b = __ldg(c.start + i + 1);
  a = min(max(a, int64_t(0)), c.tokens);
  b = min(max(b, a), c.tokens);
  s.first_token = static_cast<int>(a);
  s.tokens = static_cast<int>(b - a);
  const int64_t most = static_cast<int64_t>(c.width) * c.block_size;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(__ldg(c.lens + i), 0)), most));
  s.row_blocks = static_cast<int>((static_cast<int64_t>(s.tokens) * c.groups + ROWS - 1) / ROWS);
  s.tiles = max(1, (s.len + kTileKeys - 1) / kTileKeys);
  s.work = static_cast<int64_t>(s.row_blocks) * c.heads_kv * s.tiles;
  return s;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src, bool real) {
  const int size = real ? BYTES : 0;  // 0: zeros, nothing read
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(size) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;

// Row m of a 16-key tile holds key pi(m): with the halves of a row swizzled by row bit 1, the
// rows of {0..3}, {4..7}, the even and the odd m's all lie in different banks.
__device__ __forceinline__ int pi(int m) { return m ^ ((m >> 2) & 1); }

template <int D>
struct Tile {
  static constexpr int kRow = D / 2;        // bytes of a row's codes
  static constexpr int kPairs = D / 16;     // bytes of its (step, low) pairs
  static constexpr int kGroups = D / 64;
  static constexpr int kCodes = kTileKeys * kRow;
  static constexpr int kBytes = 2 * (kCodes + kTileKeys * kPairs);
  // byte `at` of row `key` of the codes
  static __device__ __forceinline__ int where(int key, int at) {
    return D == 128 ? key * kRow + (at ^ ((key & 2) << 4)) : key * kRow + at;
  }
};

template <int D, int NT>
constexpr int stages() {
  return NT == 1 ? 3 : 6;  // two CTAs an SM, or one with more registers
}
template <int D, int NT>
constexpr size_t ring_bytes() {
  return static_cast<size_t>(kWarps) * stages<D, NT>() * Tile<D>::kBytes;
}
template <int D, int NT>
constexpr size_t smem_bytes() {
  constexpr size_t join = static_cast<size_t>(kWarps) * 8 * NT * (D + 8) * sizeof(float);
  return ring_bytes<D, NT>() > join ? ring_bytes<D, NT>() : join;
}

template <int D, int NT, typename QT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) attention4_kernel(const Params c) {
  using L = Tile<D>;
  constexpr int kRows = 8 * NT, kGroups = L::kGroups, kStages = stages<D, NT>();
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ uint32_t live[kWarps][kStages];  // keys of a stage that exist
  __shared__ float row_m[kWarps][kRows], row_l[kWarps][kRows];
  __shared__ float low_sum[kWarps][kRows][kGroups];
  __shared__ int64_t scan[kWarps];
  __shared__ int64_t found_offset;
  __shared__ int found_seq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;

  // ---- this CTA's share of the line of tiles
  int64_t total, begin, end, share;
  {
    const int per = (c.num_seqs + kThreads - 1) / kThreads;
    const int lo = min(static_cast<int>(threadIdx.x) * per, c.num_seqs), hi = min(lo + per, c.num_seqs);
    int64_t mine = 0;
    for (int i = lo; i < hi; ++i) mine += sequence<kRows>(c, i).work;
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) scan[warp] = before;
    if (threadIdx.x == 0) found_seq = -1;
    __syncthreads();
    total = 0;
    int64_t base = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += scan[w];
      total += scan[w];
    }
    before += base - mine;  // tiles before this thread's sequences
    share = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(kMinShare));
    begin = share * blockIdx.x;
    end = min(begin + share, total);
    if (begin < end && before <= begin && begin < before + mine) {
      int64_t left = begin - before;
      int i = lo;
      for (; i < hi; ++i) {
        const int64_t work = sequence<kRows>(c, i).work;
        if (left < work) break;
        left -= work;
      }
      found_seq = i;
      found_offset = left;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) c.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (begin >= end) return;

  int seq_index = found_seq;
  int64_t offset = found_offset;
  Seq s = sequence<kRows>(c, seq_index);
  unsigned char* ring = dyn + warp * kStages * L::kBytes;
  const uint32_t ring_at = smem_u32(ring);

  for (int64_t at = begin; at < end;) {
    while (offset >= s.work) {  // the next sequence that has any
      offset -= s.work;
      s = sequence<kRows>(c, ++seq_index);
    }
    const int piece = static_cast<int>(offset / s.tiles);
    const int tile0 = static_cast<int>(offset - static_cast<int64_t>(piece) * s.tiles);
    const int tile1 = static_cast<int>(min(static_cast<int64_t>(s.tiles), tile0 + (end - at)));
    const int head = piece / s.row_blocks;
    const int row0 = (piece - head * s.row_blocks) * kRows;
    const int rows = min(kRows, s.tokens * c.groups - row0);
    const int before_tokens = s.len - s.tokens;  // the last key of the first token, less itself
    // the fewest keys that any row of the piece sees
    const int all_see = before_tokens + row0 / c.groups + 1;

    // ---- the pipeline of this warp's tiles: the next table entry is always on its way
    const int32_t* table = c.table + static_cast<int64_t>(seq_index) * c.table_stride;
    const int64_t head_at = static_cast<int64_t>(head) * c.head_stride;
    const int64_t scale_head_at = static_cast<int64_t>(head) * c.scale_head_stride;
    auto entry_of = [&](int tile) -> int {
      const int key = tile * kTileKeys + lane;
      return tile < tile1 && key < s.len ? __ldg(table + static_cast<uint32_t>(key) / static_cast<uint32_t>(c.block_size)) : -1;
    };
    auto issue = [&](int tile, int stage, int entry) {
      if (tile < tile1) {
        const bool real = entry >= 0 && entry < c.num_blocks;
        const uint32_t slot = static_cast<uint32_t>(tile * kTileKeys + lane) % static_cast<uint32_t>(c.block_size);
        const uint32_t mask = __ballot_sync(0xffffffffu, real);
        if (lane == 0) live[warp][stage] = mask;
        const int64_t codes_at = real ? entry * c.block_stride + slot * c.slot_stride + head_at : 0;
        const int64_t pairs_at = real ? entry * c.scale_block_stride + slot * c.scale_slot_stride + scale_head_at : 0;
        const uint32_t base = ring_at + stage * L::kBytes;
        constexpr int kChunks = L::kRow / 16;         // 16-byte chunks of a row
        constexpr int kRowsAtOnce = 32 / kChunks;
#pragma unroll
        for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
          const int key = i * kRowsAtOnce + lane / kChunks, chunk = lane % kChunks;
          const int64_t from = __shfl_sync(0xffffffffu, codes_at, key) + chunk * 16;
          const bool here = (mask >> key) & 1u;
          const uint32_t to = base + L::where(key, chunk * 16);
          copy_async<16>(to, c.codes[0] + from, here);
          copy_async<16>(to + L::kCodes, c.codes[1] + from, here);
        }
        const uint32_t pairs = base + 2 * L::kCodes + lane * L::kPairs;
        copy_async<L::kPairs>(pairs, c.scales[0] + pairs_at, real);
        copy_async<L::kPairs>(pairs + kTileKeys * L::kPairs, c.scales[1] + pairs_at, real);
      }
      copy_commit();
    };
    int next = tile0 + warp;  // the next tile to issue
    int entry = entry_of(next);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      const int here = entry;
      entry = entry_of(next + kWarps);
      issue(next, i, here);
      next += kWarps;
    }

    // ---- the query rows as B operands, and per row its factor and the sums of its groups
    uint32_t q[NT][kGroups][4][2];
    float factor[NT][2], sums[NT][kGroups][2];
    int last[NT][2];  // the last key of the two rows that this lane's scores belong to
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + n * 8 + g;
      const int token = row / c.groups;
      const bool real = row < s.tokens * c.groups;
      const QT* src = reinterpret_cast<const QT*>(c.query + (s.first_token + static_cast<int64_t>(real ? token : 0)) * c.query_ts +
                                                  static_cast<int64_t>(head * c.groups + (real ? row - token * c.groups : 0)) * c.query_hs);
      float x[kGroups][16], most = 0.0f, sum[kGroups];
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        const QT* from = src + G * 64 + t * 16;
        if (c.aligned) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(from) + i);
            const QT* e = reinterpret_cast<const QT*>(&v);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[G][i * 8 + j] = real ? Elem<QT>::to_f(e[j]) : 0.0f;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) x[G][j] = real ? Elem<QT>::to_f(from[j]) : 0.0f;
        }
        sum[G] = 0.0f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          most = fmaxf(most, fabsf(x[G][j]));
          sum[G] += x[G][j];
        }
      }
#pragma unroll
      for (int o = 1; o <= 2; o <<= 1) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
#pragma unroll
        for (int G = 0; G < kGroups; ++G) sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], o);
      }
      int e = most > 0.0f ? 14 - (static_cast<int>(__float_as_uint(most) >> 23) - 127) : 0;
      e = min(max(e, -110), 110);
      const float up = __int_as_float((e + 127) << 23);  // 2^e
#pragma unroll
      for (int G = 0; G < kGroups; ++G)
#pragma unroll
        for (int j = 0; j < 2; ++j)  // a word of 8 codes: dimensions (0, 4) (1, 5) (2, 6) (3, 7)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* w = &x[G][j * 8 + h * 2];
            q[n][G][j * 2 + h][0] = pack(w[0] * up, w[4] * up);
            q[n][G][j * 2 + h][1] = pack(w[1] * up * 0.0625f, w[5] * up * 0.0625f);
          }
      // 2^24 of the codes, less the row's own power of two
      const float f = c.scale_log2 * __int_as_float((127 - e) << 23) * 16777216.0f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = 2 * t + j;
        factor[n][j] = __shfl_sync(0xffffffffu, f, col * 4);
#pragma unroll
        for (int G = 0; G < kGroups; ++G) sums[n][G][j] = __shfl_sync(0xffffffffu, sum[G], col * 4) * c.scale_log2;
        last[n][j] = before_tokens + min(row0 + n * 8 + col, s.tokens * c.groups - 1) / c.groups;
      }
    }

    float o[NT][kGroups][4][4], low[NT][kGroups][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int G = 0; G < kGroups; ++G) {
        low[n][G][0] = low[n][G][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[n][G][i][j] = 0.0f;
      }
    }

    int stage = 0;
    for (int tile = tile0 + warp; tile < tile1; tile += kWarps) {
      {
        const int here = entry;
        entry = entry_of(next + kWarps);
        const int into = stage == 0 ? kStages - 1 : stage - 1;
        issue(next, into, here);
        next += kWarps;
      }
      copy_wait<kStages - 1>();
      __syncwarp();
      const unsigned char* buf = ring + stage * L::kBytes;
      const uint32_t mask = live[warp][stage];
      const int key0 = tile * kTileKeys;
      const bool cut = mask != 0xffffffffu || key0 + kTileKeys > all_see;  // some row does not see some key

      // ---- scores of 2 x 16 keys
      float w[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int ka = mt * 16 + pi(g), kb = ka + 8;
        float step[2][kGroups], base[2][kGroups];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const __half2* p = reinterpret_cast<const __half2*>(buf + 2 * L::kCodes + (r ? kb : ka) * L::kPairs);
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            const float2 f = __half22float2(p[G]);
            step[r][G] = f.x, base[r][G] = f.y;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) w[mt][n][j] = 0.0f;
        float acc[NT][kGroups][4];
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          const uint2 va = *reinterpret_cast<const uint2*>(buf + L::where(ka, G * 32 + t * 8));
          const uint2 vb = *reinterpret_cast<const uint2*>(buf + L::where(kb, G * 32 + t * 8));
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][G][j] = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t a = j < 2 ? va.x : va.y, b = j < 2 ? vb.x : vb.y;
            if (j & 1) a >>= 8, b >>= 8;
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma(acc[n][G], a & kEven, b & kEven, a & kOdd, b & kOdd, q[n][G][j][0], q[n][G][j][1]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j >> 1;
            float dot = step[r][0] * acc[n][0][j], rest = base[r][0] * sums[n][0][j & 1];
            if constexpr (kGroups == 2) {
              dot = fmaf(step[r][1], acc[n][1][j], dot);
              rest = fmaf(base[r][1], sums[n][1][j & 1], rest);
            }
            w[mt][n][j] = fmaf(dot, factor[n][j & 1], rest);
          }
        if (cut) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = j < 2 ? ka : kb;
              if (key0 + key > last[n][j & 1] || !((mask >> key) & 1u)) w[mt][n][j] = -INFINITY;
            }
        }
      }

      // ---- steps and lowest values of the V rows, and the exponent of the largest step
      float vstep[2][2][kGroups], vlow[2][2][kGroups], largest = 0.0f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = mt * 16 + pi(g) + r * 8;
          const __half2* p = reinterpret_cast<const __half2*>(buf + 2 * L::kCodes + (kTileKeys + key) * L::kPairs);
          const bool dead = cut && (!((mask >> key) & 1u));
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            const float2 f = __half22float2(p[G]);
            vstep[mt][r][G] = f.x, vlow[mt][r][G] = f.y;
            largest = fmaxf(largest, dead ? 0.0f : fminf(fabsf(f.x), 65504.0f));
          }
        }
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(largest));
      // 2^room_e is above the largest step; steps below 2^-24 do not exist in fp16
      const float room_e = static_cast<float>(max(static_cast<int>(bits >> 23) - 126, -24));

      // ---- the reference M moves only when a factor would pass 2^15
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top[2];
        bool move = false;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[j] = fmaxf(fmaxf(w[0][n][j], w[0][n][j + 2]), fmaxf(w[1][n][j], w[1][n][j + 2]));
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], x));
          top[j] += room_e;
          move |= top[j] > m[n][j] + kMostRoom;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (top[j] > m[n][j] + kMostRoom) {
              const float now = top[j] - kSetRoom;
              const float keep = m[n][j] == -INFINITY ? 0.0f : ex2(m[n][j] - now);
              m[n][j] = now;
              l[n][j] *= keep;
#pragma unroll
              for (int G = 0; G < kGroups; ++G) {
                low[n][G][j] *= keep;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][G][i][j] *= keep, o[n][G][i][j + 2] *= keep;
              }
            }
          }
        }
      }

      // ---- P and the products with V
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t b[NT][kGroups][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float ref = m[n][j & 1] == -INFINITY ? 0.0f : m[n][j & 1];
            p[j] = ex2(w[mt][n][j] - ref);
            l[n][j & 1] += p[j];
          }
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              f[j] = p[j] * vstep[mt][j >> 1][G];
              float term = p[j] * vlow[mt][j >> 1][G];
              if (cut && w[mt][n][j] == -INFINITY) f[j] = term = 0.0f;  // whatever an unseen row holds
              low[n][G][j & 1] += term;
            }
            b[n][G][0] = transposed(pack(f[0], f[1]));
            b[n][G][1] = transposed(pack(f[2], f[3]));
          }
        }
        const unsigned char* v = buf + L::kCodes;
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          uint32_t x[4];  // 8 dimensions of keys pi(2 t), pi(2 t + 1), and of those 8 further
#pragma unroll
          for (int k = 0; k < 4; ++k)
            x[k] = *reinterpret_cast<const uint32_t*>(v + L::where(mt * 16 + (k >> 1) * 8 + pi(2 * t + (k & 1)), G * 32 + g * 4));
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // dimensions 0-3, 4-7
            uint32_t near = __byte_perm(x[0], x[1], half ? 0x7632 : 0x5410);
            uint32_t far = __byte_perm(x[2], x[3], half ? 0x7632 : 0x5410);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (i) near >>= 8, far >>= 8;
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma(o[n][G][half * 2 + i], near & kEven, near & kOdd, far & kEven, far & kOdd, b[n][G][0], b[n][G][1]);
            }
          }
        }
      }
      __syncwarp();  // the stage may be filled again
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    copy_wait<0>();

    // ---- the warps' parts meet
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], x);
#pragma unroll
          for (int G = 0; G < kGroups; ++G) low[n][G][j] += __shfl_xor_sync(0xffffffffu, low[n][G][j], x);
        }
        if (g == 0) {
          const int row = n * 8 + 2 * t + j;
          row_m[warp][row] = m[n][j];
          row_l[warp][row] = l[n][j];
#pragma unroll
          for (int G = 0; G < kGroups; ++G) low_sum[warp][row][G] = low[n][G][j];
        }
      }
    __syncthreads();  // every warp is done with its ring as well
    float* join = reinterpret_cast<float*>(dyn);  // [warp][row][D + 8], dimensions as the fragments hold them
    constexpr int kJoinRow = D + 8;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float* dst = join + (warp * kRows + n * 8 + 2 * t + j) * kJoinRow + g * 2;
#pragma unroll
        for (int G = 0; G < kGroups; ++G)
#pragma unroll
          for (int i = 0; i < 4; ++i)  // the codes' 2^24, and 2^20 for the odd nibbles
            *reinterpret_cast<float2*>(dst + (G * 4 + i) * 16) =
                make_float2(o[n][G][i][j] * 16777216.0f, o[n][G][i][j + 2] * 1048576.0f);
      }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == s.tiles;
    float* part = c.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (tile0 == 0)) * kRows * (D + 2);
    for (int x = threadIdx.x; x < rows * (D / 2); x += kThreads) {
      const int row = x / (D / 2), pair = x - row * (D / 2);  // two neighbouring dimensions
      const int G = pair / 32, i = (pair / 8) & 3, dim = G * 64 + (pair & 7) * 8 + i * 2;
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < kWarps; ++u) top = fmaxf(top, row_m[u][row]);
      float sum = 0.0f;
      float2 value = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int u = 0; u < kWarps; ++u) {
        const float um = row_m[u][row];
        const float by = um == -INFINITY ? 0.0f : ex2(um - top);
        const float2 y = *reinterpret_cast<const float2*>(join + (u * kRows + row) * kJoinRow + pair * 2);
        const float add = low_sum[u][row][G];
        sum = fmaf(row_l[u][row], by, sum);
        value.x = fmaf(y.x + add, by, value.x);
        value.y = fmaf(y.y + add, by, value.y);
      }
      if (whole) {
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees no key is zeros
        const int r = row0 + row, token = r / c.groups;
        QT* dst = reinterpret_cast<QT*>(c.out + (s.first_token + static_cast<int64_t>(token)) * c.out_ts +
                                        static_cast<int64_t>(head * c.groups + r - token * c.groups) * c.out_hs) + dim;
        dst[0] = Elem<QT>::from_f(value.x * inverse);
        dst[1] = Elem<QT>::from_f(value.y * inverse);
      } else {
        float* dst = part + row * (D + 2);
        dst[2 + dim] = value.x;
        dst[3 + dim] = value.y;
        if (pair == 0) dst[0] = top, dst[1] = sum;
      }
    }
    if (threadIdx.x == 0 && tile0 == 0 && tile1 < s.tiles)
      c.meta[blockIdx.x] = make_int4(static_cast<int>((s.tiles - tile1 + share - 1) / share), seq_index, head, row0);
    __syncthreads();  // the ring and the row values may be written again
    at += tile1 - tile0;
    offset += tile1 - tile0;
  }
}

// Joins the parts of one row of a piece that was cut: part 1 of its first CTA, then part 0 of
// the CTAs that follow, always in that order.  A warp takes every eighth part.
template <int D, int NT, typename QT>
__global__ void __launch_bounds__(kThreads) join4_kernel(const Params c) {
  constexpr int kRows = 8 * NT, kPer = D / 32;
  const int4 meta = c.meta[blockIdx.x];
  if (meta.x < 0) return;
  const Seq s = sequence<kRows>(c, meta.y);
  const int row = blockIdx.y, r = meta.w + row;
  if (r >= s.tokens * c.groups) return;
  __shared__ float tops[kWarps], sums[kWarps], values[kWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto part_of = [&](int i) -> const float* {
    return c.parts + ((static_cast<int64_t>(blockIdx.x) + i) * 2 + (i == 0)) * kRows * (D + 2) + row * (D + 2);
  };
  float top = -INFINITY, sum = 0.0f, value[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) value[j] = 0.0f;
  for (int i = warp; i <= meta.x; i += kWarps) {
    const float* p = part_of(i);
    const float pm = p[0], pl = p[1];
    float v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = p[2 + j * 32 + lane];
    const float now = fmaxf(top, pm);
    const float keep = top == -INFINITY ? 0.0f : ex2(top - now), by = pm == -INFINITY ? 0.0f : ex2(pm - now);
    top = now;
    sum = sum * keep + pl * by;
#pragma unroll
    for (int j = 0; j < kPer; ++j) value[j] = value[j] * keep + v[j] * by;
  }
  if (lane == 0) tops[warp] = top, sums[warp] = sum;
#pragma unroll
  for (int j = 0; j < kPer; ++j) values[warp][j * 32 + lane] = value[j];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float all = -INFINITY;
#pragma unroll
    for (int u = 0; u < kWarps; ++u) all = fmaxf(all, tops[u]);
    float l = 0.0f, v = 0.0f;
#pragma unroll
    for (int u = 0; u < kWarps; ++u) {
      const float by = tops[u] == -INFINITY ? 0.0f : ex2(tops[u] - all);
      l = fmaf(sums[u], by, l);
      v = fmaf(values[u][d], by, v);
    }
    const int token = r / c.groups;
    QT* dst = reinterpret_cast<QT*>(c.out + (s.first_token + static_cast<int64_t>(token)) * c.out_ts +
                                    static_cast<int64_t>(meta.z * c.groups + r - token * c.groups) * c.out_hs) + d;
    *dst = Elem<QT>::from_f(l == 0.0f ? 0.0f : v / l);
  }
}

// ---------------------------------------------------------------- host side
// Rows of a row block: 8 while a sequence's rows of a KV head (on average) fit, else 16, which
// reads the pages half as often.
int tiles_n(int64_t num_tokens, int64_t num_seqs, int64_t groups) {
  return groups * ((num_tokens + num_seqs - 1) / num_seqs) > 8 ? 2 : 1;
}
int ctas(int nt) { return kSmCount * (nt == 1 ? 2 : 1); }

size_t workspace(int nt, int64_t head_size) {
  const size_t meta = (static_cast<size_t>(ctas(nt)) * sizeof(int4) + 255) / 256 * 256;
  return meta + static_cast<size_t>(ctas(nt)) * 2 * 8 * nt * (head_size + 2) * sizeof(float);
}

template <int D, int NT, typename QT>
int launch(const Params& c, cudaStream_t s) {
  constexpr size_t kBytes = smem_bytes<D, NT>();
  int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(attention4_kernel<D, NT, QT>), kBytes);
  if (rc != CB_OK) return rc;
  attention4_kernel<D, NT, QT><<<ctas(NT), kThreads, kBytes, s>>>(c);
  rc = launch_status("cb_paged_attention4");
  if (rc != CB_OK) return rc;
  join4_kernel<D, NT, QT><<<dim3(ctas(NT), 8 * NT), kThreads, 0, s>>>(c);
  return launch_status("cb_paged_attention4 (join)");
}

template <typename QT>
int dispatch(const Params& c, int64_t head_size, int nt, cudaStream_t s) {
  if (head_size == 128) return nt == 1 ? launch<128, 1, QT>(c, s) : launch<128, 2, QT>(c, s);
  return nt == 1 ? launch<64, 1, QT>(c, s) : launch<64, 2, QT>(c, s);
}

int check_shape(int64_t num_tokens, int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size) {
  CB_SUPPORTED(head_size == 64 || head_size == 128, "4-bit pages hold heads of 64 or 128 values (got %lld)",
               (long long)head_size);
  CB_REQUIRE(num_tokens >= 0 && num_seqs >= 0, "negative size");
  CB_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
             "query heads must be a multiple of KV heads");
  CB_REQUIRE(num_seqs < (int64_t(1) << 24) && num_q_heads < (int64_t(1) << 16) &&
                 num_tokens < (int64_t(1) << 30) / num_q_heads,
             "size out of range");
  CB_REQUIRE(num_seqs > 0 || num_tokens == 0, "tokens without sequences");
  return CB_OK;
}

}  // namespace att4
}  // namespace cb

using namespace cb;

extern "C" int cb_paged_attention4_workspace_size(int64_t num_tokens, int64_t num_seqs, int64_t num_q_heads,
                                                  int64_t num_kv_heads, int64_t head_size, int64_t* bytes) {
  clear_error();
  CB_REQUIRE(bytes != nullptr, "null output");
  const int rc = att4::check_shape(num_tokens, num_seqs, num_q_heads, num_kv_heads, head_size);
  if (rc != CB_OK) return rc;
  *bytes = num_tokens == 0 ? 0
                           : static_cast<int64_t>(att4::workspace(
                                 att4::tiles_n(num_tokens, num_seqs, num_q_heads / num_kv_heads), head_size));
  return CB_OK;
}

extern "C" int cb_paged_attention4(const void* query, int64_t query_token_stride, int64_t query_head_stride,
                                   int64_t num_tokens, int64_t num_q_heads, int dtype, const int32_t* query_start,
                                   const void* k_codes, const void* v_codes, int64_t block_stride, int64_t slot_stride,
                                   int64_t head_stride, const void* k_scales, const void* v_scales,
                                   int64_t scale_block_stride, int64_t scale_slot_stride, int64_t scale_head_stride,
                                   int64_t num_blocks, int64_t block_size, int64_t num_kv_heads, int64_t head_size,
                                   const int32_t* block_table, int64_t table_stride, int64_t table_width,
                                   const int32_t* seq_lens, int64_t num_seqs, float scale, void* out,
                                   int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  CB_BIND(stream, out);
  CB_SUPPORTED(dtype == CB_DTYPE_BF16 || dtype == CB_DTYPE_FP16, "queries must be bf16 or fp16");
  const int rc = att4::check_shape(num_tokens, num_seqs, num_q_heads, num_kv_heads, head_size);
  if (rc != CB_OK) return rc;
  if (num_tokens == 0) return CB_OK;
  CB_REQUIRE(query_start != nullptr || num_tokens == num_seqs, "one token per sequence, or query_start");
  CB_REQUIRE(num_blocks >= 0 && num_blocks < (int64_t(1) << 31) && block_size > 0 && block_size < (int64_t(1) << 22) &&
                 table_width >= 0 && table_width * block_size < (int64_t(1) << 31),
             "page sizes out of range");
  CB_REQUIRE(query && out && seq_lens && workspace && (block_table || table_width == 0), "null pointer argument");
  CB_REQUIRE(k_codes && v_codes && k_scales && v_scales, "null page pointer");
  const uint64_t codes = reinterpret_cast<uint64_t>(k_codes) | reinterpret_cast<uint64_t>(v_codes) | (uint64_t)block_stride |
                         (uint64_t)slot_stride | (uint64_t)head_stride;
  CB_REQUIRE((codes & 15u) == 0, "4-bit rows must be 16-byte aligned");
  const uint64_t scales = reinterpret_cast<uint64_t>(k_scales) | reinterpret_cast<uint64_t>(v_scales) |
                          (uint64_t)scale_block_stride | (uint64_t)scale_slot_stride | (uint64_t)scale_head_stride;
  CB_REQUIRE((scales & (uint64_t)(head_size / 16 - 1)) == 0, "the steps of a 4-bit row must be %lld-byte aligned",
             (long long)(head_size / 16));
  const uint64_t rows = reinterpret_cast<uint64_t>(query) | (uint64_t)query_token_stride | (uint64_t)query_head_stride;
  CB_REQUIRE(((rows | reinterpret_cast<uint64_t>(out) | (uint64_t)out_token_stride | (uint64_t)out_head_stride) & 1u) == 0,
             "rows must be aligned to their element size");
  const int64_t groups = num_q_heads / num_kv_heads;
  const int nt = att4::tiles_n(num_tokens, num_seqs, groups);
  CB_REQUIRE((reinterpret_cast<uint64_t>(workspace) & 15u) == 0, "the workspace must be 16-byte aligned");
  CB_REQUIRE(workspace_bytes >= static_cast<int64_t>(att4::workspace(nt, head_size)), "workspace too small (%lld < %zu)",
             (long long)workspace_bytes, att4::workspace(nt, head_size));
  att4::Params c{};
  c.query = static_cast<const char*>(query), c.query_ts = query_token_stride, c.query_hs = query_head_stride;
  c.out = static_cast<char*>(out), c.out_ts = out_token_stride, c.out_hs = out_head_stride;
  c.tokens = num_tokens, c.start = query_start, c.lens = seq_lens, c.table = block_table, c.table_stride = table_stride;
  c.num_seqs = static_cast<int>(num_seqs), c.width = static_cast<int>(table_width);
  c.heads_kv = static_cast<int>(num_kv_heads), c.groups = static_cast<int>(groups);
  c.codes[0] = static_cast<const char*>(k_codes), c.codes[1] = static_cast<const char*>(v_codes);
  c.scales[0] = static_cast<const char*>(k_scales), c.scales[1] = static_cast<const char*>(v_scales);
  c.block_stride = block_stride, c.slot_stride = slot_stride, c.head_stride = head_stride;
  c.scale_block_stride = scale_block_stride, c.scale_slot_stride = scale_slot_stride;
  c.scale_head_stride = scale_head_stride;
  c.num_blocks = num_blocks, c.block_size = static_cast<int>(block_size);
  c.scale_log2 = scale * att4::kLog2e;
  c.aligned = (rows & 15u) == 0;
  c.meta = static_cast<int4*>(workspace);
  c.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                     (static_cast<size_t>(att4::ctas(nt)) * sizeof(int4) + 255) / 256 * 256);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == CB_DTYPE_BF16 ? att4::dispatch<__nv_bfloat16>(c, head_size, nt, s) : att4::dispatch<__half>(c, head_size, nt, s);
}
