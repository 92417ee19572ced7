// Attention of single tokens (or a few per sequence) over 4-bit pages.
//
// A row of the pages holds, per group G of 64 dimensions, codes c and a pair
// (step, low); its values are low_G + step_G c.  For a query q of KV head h and
// the key at position j, with everything in the log2 domain,
//   w_j  = scale log2e (sum_G step_jG (q . c_j)_G + sum_G low_jG (sum_G q))
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
//     subnormal c 2^-24, at bits 4-7 c 2^-20, both exact operands.  The factor 2^24
//     goes into the row's factor, the odd nibbles' 16 into q (K) or into the output row
//     (V).  A product lines its terms up by the operands' exponents, a subnormal's being
//     2^-14, so that its sum is cut at about 2^-14 of a factor (measured: 2^-18.6 of 8
//     factors): coarser than fp32, but an eighth of what rounding the factor may cost.
//   * K: the 16 keys of a tile are the M rows, the query rows the N columns, the
//     dimensions of one group the K steps.  Eight columns: a whole group of query
//     heads usually fits, and 16 at once, which share the masked words, ran with half
//     the warps and up to 1.3 times as long.  q is scaled per row by a power of two so
//     that its largest value is in [2^14, 2^15): bf16 and fp16 values are exact in
//     fp16 down to 2^-28 of it.  The low terms are one more product, of the lowest
//     values as they lie with q's group sums in three fp16 limbs.
//   * V: the dimensions are the M rows, the keys the K steps, P the B operand; a
//     transposing ldmatrix of 16-bit units (four codes of a key) pairs the same
//     codes of two keys.  P step'_G is rounded to fp16 (11 bits: 2^-11 relative,
//     against the 2^-8 of a bf16 output) once per group and transposed by
//     movmatrix.  The roundings weigh with codes less 8, not with codes: 8 times the
//     sum of the rounded factors (one more product, of ones) is taken off again and
//     the low terms are taken at code 8, so that a row's offset does not multiply them
//     (fp16 outputs of rows around 0: 3.4e-4 off without, 2.5e-4 with, 2.1e-4 for the
//     rounding of the result alone).  M is taken over p step' of the keys that a
//     row sees, so that a factor stays in fp16's range whatever the values' size: at most
//     2^15, and the largest 2^10 when M is set.  M moves only when a factor would pass that,
//     which each lane bounds for itself: the common tile needs no maximum over the warp.
// Sums, maxima, steps and the low terms are fp32.
//
// Memory: a warp takes tiles of 32 keys of one KV head through a ring of its
// own, filled by cp.async (16 bytes of a row per lane; a page's rows may lie
// anywhere and end anywhere in a tile), so no barrier joins the warps inside a
// piece of work.  The 16-byte chunks of a row are swizzled by row so that the
// eight rows of an ldmatrix lie in different banks.
//
// Split: all (sequence, KV head, row block) pieces form one line, each as long as
// its rounds (a tile per warp) and a fixed cost, cut into equal shares, one per
// CTA, whatever the lengths are; the cut is found on the device from the lengths.
// Without the fixed cost the CTAs that got many short sequences ran twice as long
// as the rest (64 sequences of 1 to 8,192 keys: 130 us against 74 then).  The first
// and last piece of a share may be parts; parts go to the workspace and a second
// launch joins them in order, so a result does not depend on timing.
//
// What bounds it (6 sequences of up to 98,304 keys, 32 query heads on 4: 40 us, 3.8
// TB/s, replayed from a graph; 41 to 51 us call by call): about 500 instructions a
// tile, 160 of them the codes' masks and shifts, at 55 % of the issue slots and 46 % of
// the ALU pipe with 16 warps an SM, beside some 10 us of launch, first loads and the
// join.  The memory side alone takes 33 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cb_common.cuh"

namespace cb {
namespace att4 {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;         // query rows of a piece: the columns of a product
constexpr int kTileKeys = 32;    // keys of a warp's stage
constexpr int kStages = 2;       // of a warp's ring; three measured 3 % slower
constexpr int kCtas = 2 * kSmCount;
constexpr int kRound = kWarps;   // tiles of a CTA's round: one per warp
// What a piece costs besides its rounds, in rounds: its first loads, the query operands and
// the warps' meeting.
constexpr int kPieceCost = 3;
// Tables of at most this many keys are not cut: the join's launch costs more than the rounds
// that a second CTA would take over.
constexpr int kUncutKeys = 2 * kRound * kTileKeys;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSetRoom = 10.0f;   // a factor p step' is at most 2^10 when M is set,
constexpr float kMostRoom = 15.0f;  // and 2^15 before M moves
// Logits below this count as this when M is set: a row that sees a key has a finite M, so that one of
// which no weight is left (fp32 does not hold its logits) ends as 0 / 0 and not as a row without keys.
constexpr float kLeast = -3e38f;

// A piece that a CTA began and others go on with.
struct alignas(32) Cut {
  int followers;  // CTAs that go on; negative: no such piece
  int head, row0, rows, first_token;  // rows: of the sequence and KV head
};

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
  // 16-byte units for the codes, 4-byte units for the scales: offsets fit 32 bits
  uint32_t block_stride, slot_stride, head_stride;
  uint32_t scale_block_stride, scale_slot_stride, scale_head_stride;
  uint32_t num_blocks;
  int block_size;
  int step_pages, step_rows;  // kRound * kTileKeys keys further: pages and rows
  float scale_log2;  // scale * log2(e)
  bool aligned;      // query rows in whole 16-byte vectors
  bool uncut;        // every piece whole in one CTA: nothing to join
  float* parts;      // [ctas][2][rows][D + 2]
  Cut* meta;         // [ctas]
};

// One sequence's share of the line.
struct Seq {
  int first_token, tokens;
  int len, before;                // keys that the table has room for; those before the query tokens, past it or not
  int row_blocks, tiles, rounds;  // tiles and rounds per piece
  int64_t work;                   // of all its pieces
};
__device__ __forceinline__ Seq sequence(const Params& c, int i) {
  Seq s;
  int64_t a = i, b = i + 1;
  if (c.start != nullptr) a = __ldg(c.start + i), b = __ldg(c.start + i + 1);
  a = min(max(a, int64_t(0)), c.tokens);
  b = min(max(b, a), c.tokens);
  s.first_token = static_cast<int>(a);
  s.tokens = static_cast<int>(b - a);
  const int64_t most = static_cast<int64_t>(c.width) * c.block_size;
  const int all = max(__ldg(c.lens + i), 0);
  s.len = static_cast<int>(min(static_cast<int64_t>(all), most));
  s.before = all - s.tokens;
  s.row_blocks = static_cast<int>((static_cast<int64_t>(s.tokens) * c.groups + kRows - 1) / kRows);
  s.tiles = max(1, (s.len + kTileKeys - 1) / kTileKeys);
  s.rounds = (s.tiles + kRound - 1) / kRound;
  s.work = static_cast<int64_t>(s.row_blocks) * c.heads_kv * (s.rounds + kPieceCost);
  return s;
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const char* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// Four 8 x 8 matrices of 16-bit units, a row address per lane.
__device__ __forceinline__ void load_rows(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_columns(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same onto zeros.
__device__ __forceinline__ void mma_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u, kEight = 0x00080008u;

template <int D>
struct Tile {
  static constexpr int kRow = D / 2;        // bytes of a row's codes
  static constexpr int kPairs = D / 16;     // bytes of its (step, low) pairs
  static constexpr int kGroups = D / 64;
  static constexpr int kCodes = kTileKeys * kRow;
  static constexpr int kBytes = 2 * (kCodes + kTileKeys * kPairs);
  // 16-byte chunk of row `key` of the codes
  static __device__ __forceinline__ int where(int key, int chunk) {
    return key * kRow + 16 * (D == 128 ? chunk ^ ((key >> 1) & 3) : chunk ^ ((key >> 2) & 1));
  }
};

// The (step, low) pairs of a key's K row and V row.
template <int GROUPS>
__device__ __forceinline__ void load_pairs(uint32_t (&k)[GROUPS], uint32_t (&v)[GROUPS], uint32_t at) {
  if constexpr (GROUPS == 2)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(k[0]), "=r"(k[1]), "=r"(v[0]), "=r"(v[1]) : "r"(at) : "memory");
  else
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(k[0]), "=r"(v[0]) : "r"(at) : "memory");
}

template <int D>
constexpr size_t smem_bytes() {
  constexpr size_t ring = static_cast<size_t>(kWarps) * kStages * Tile<D>::kBytes;
  constexpr size_t join = static_cast<size_t>(kWarps) * kRows * (D + 8) * sizeof(float);
  return ring > join ? ring : join;
}

// A CTA's place on the line, and the work that it finds there.
struct Walk {
  int64_t at, end, offset, share;  // offset: in the sequence's part of the line
  int seq;
};
struct Piece {
  int seq, head, row0, tile0, tile1, len, tokens, first_token;  // tile1 < 0: the share is done
  int before;
  bool whole;
};
__device__ __noinline__ void next_piece(const Params& c, Walk& walk, Piece& piece) {
  piece.tile1 = -1;
  while (walk.at < walk.end) {
    const Seq s = sequence(c, walk.seq);
    if (walk.offset >= s.work) {  // the next sequence that has any
      walk.offset -= s.work;
      ++walk.seq;
      continue;
    }
    const int length = s.rounds + kPieceCost;  // a piece's place on the line: its cost, then its rounds
    const int number = (walk.offset >> 31) == 0 ? static_cast<int>(walk.offset) / length : static_cast<int>(walk.offset / length);
    const int from = static_cast<int>(walk.offset - static_cast<int64_t>(number) * length);
    // uncut pieces belong to the share that they begin in
    const int to = c.uncut ? length : static_cast<int>(min(static_cast<int64_t>(length), from + (walk.end - walk.at)));
    walk.at += to - from;
    walk.offset += to - from;
    if (c.uncut && from > 0) continue;
    if (to <= kPieceCost) continue;  // the share ends before the piece's first round: the next CTA begins it
    piece.seq = walk.seq;
    piece.head = number / s.row_blocks;
    piece.row0 = (number - piece.head * s.row_blocks) * kRows;
    piece.tile0 = max(from - kPieceCost, 0) * kRound;
    piece.tile1 = min((to - kPieceCost) * kRound, s.tiles);
    piece.len = s.len, piece.tokens = s.tokens, piece.first_token = s.first_token;
    piece.before = s.before;
    piece.whole = piece.tile0 == 0 && piece.tile1 == s.tiles;
    if (piece.tile0 == 0 && !piece.whole)
      c.meta[blockIdx.x] = Cut{static_cast<int>((length - to + walk.share - 1) / walk.share), piece.head, piece.row0,
                               s.tokens * c.groups, s.first_token};
    return;
  }
}

template <int D, typename QT>
__global__ void __launch_bounds__(kThreads, 2) attention4_kernel(const __grid_constant__ Params c) {
  using L = Tile<D>;
  constexpr int kGroups = L::kGroups, kChunks = D / 32;
  // (ldmatrix: lane l names row l & 15 of a 16-key tile, chunk l >> 4 of a group's two)
  extern __shared__ __align__(128) unsigned char dyn[];
  __shared__ uint32_t live[kWarps][kStages];  // keys of a stage that exist
  __shared__ float row_m[kWarps][kRows], row_l[kWarps][kRows];
  __shared__ float low_sum[kWarps][kRows][kGroups];
  __shared__ int64_t scan[kWarps];
  __shared__ Walk walk;    // thread 0's place on the line,
  __shared__ Piece piece;  // and what it found there: kept out of the registers
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;

  // ---- this CTA's share of the line
  {
    const int per = (c.num_seqs + kThreads - 1) / kThreads;
    const int lo = min(static_cast<int>(threadIdx.x) * per, c.num_seqs), hi = min(lo + per, c.num_seqs);
    int64_t mine = 0;
    for (int i = lo; i < hi; ++i) mine += sequence(c, i).work;
    int64_t before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) scan[warp] = before;
    __syncthreads();
    int64_t total = 0, base = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += scan[w];
      total += scan[w];
    }
    before += base - mine;  // the line before this thread's sequences
    const int64_t share = (total + gridDim.x - 1) / gridDim.x, begin = share * blockIdx.x;
    if (begin >= total) {
      if (threadIdx.x == 0) c.meta[blockIdx.x].followers = -1;
      return;
    }
    if (before <= begin && begin < before + mine) {
      int64_t left = begin - before;
      int i = lo;
      for (; i < hi; ++i) {
        const int64_t work = sequence(c, i).work;
        if (left < work) break;
        left -= work;
      }
      c.meta[blockIdx.x].followers = -1;  // until a cut piece replaces it
      walk = Walk{begin, min(begin + share, total), left, share, i};
      next_piece(c, walk, piece);
    }
  }
  const uint32_t ring_at = smem_u32(dyn) + warp * kStages * L::kBytes;

  for (bool first = true;; first = false) {
    __syncthreads();  // the first piece is known; the ring and the row values may be written again
    if (!first) {
      if (threadIdx.x == 0) next_piece(c, walk, piece);
      __syncthreads();
    }
    const int tile0 = piece.tile0, tile1 = piece.tile1;
    if (tile1 < 0) break;
    const int head = piece.head, row0 = piece.row0;
    // the fewest keys that any row of the piece sees
    const int all_see = piece.before + row0 / c.groups + 1;

    // ---- the pipeline of this warp's tiles: the next table entry is always on its way
    const int32_t* table = c.table + static_cast<int64_t>(piece.seq) * c.table_stride;
    const int len = piece.len;
    const uint32_t head_at = head * c.head_stride, scale_head_at = head * c.scale_head_stride;
    int next = tile0 + warp;  // the tile that is issued next, and this lane's key of the tile after it
    int key_after = next * kTileKeys + lane;
    int page_after = key_after / c.block_size, slot_after = key_after - page_after * c.block_size;
    int entry = -1, slot = 0;
    auto look_up = [&](int tile) {  // entry and row of this lane's key of `tile`, then a round further
      slot = slot_after;
      entry = tile < tile1 && key_after < len ? __ldg(table + page_after) : -1;
      key_after += kRound * kTileKeys;
      page_after += c.step_pages;
      slot_after += c.step_rows;
      if (slot_after >= c.block_size) slot_after -= c.block_size, ++page_after;
    };
    auto issue = [&](int stage) {
      const int row = slot;
      const uint32_t page = static_cast<uint32_t>(entry);
      const int tile = next;
      next += kRound;
      look_up(next);
      if (tile < tile1) {
        // a key that does not exist copies the cache's first row; its score and factors are
        // replaced, whatever it holds
        const bool real = page < c.num_blocks;
        const uint32_t mask = __ballot_sync(0xffffffffu, real);
        if (lane == 0) live[warp][stage] = mask;
        const uint32_t at = real ? page * c.block_stride + row * c.slot_stride + head_at : 0u;
        const uint32_t pairs_at = real ? page * c.scale_block_stride + row * c.scale_slot_stride + scale_head_at : 0u;
        const uint32_t base = ring_at + stage * L::kBytes;
        constexpr int kChunks = L::kRow / 16;  // 16-byte chunks of a row
        constexpr int kRowsAtOnce = 32 / kChunks;
        if (mask != 0) {  // (an empty cache has no first row)
#pragma unroll
          for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
            const int key = i * kRowsAtOnce + lane / kChunks, chunk = lane % kChunks;
            const uint64_t from = static_cast<uint64_t>(__shfl_sync(0xffffffffu, at, key)) * 16u + chunk * 16u;
            const uint32_t into = base + L::where(key, chunk);
            copy_async<16>(into, c.codes[0] + from);
            copy_async<16>(into + L::kCodes, c.codes[1] + from);
          }
          const uint32_t pairs = base + 2 * L::kCodes + lane * 2 * L::kPairs;  // a key's K pairs, then its V pairs
          copy_async<L::kPairs>(pairs, c.scales[0] + static_cast<uint64_t>(pairs_at) * 4u);
          copy_async<L::kPairs>(pairs + L::kPairs, c.scales[1] + static_cast<uint64_t>(pairs_at) * 4u);
        }
      }
      copy_commit();
    };
    look_up(next);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // ---- the query rows as B operands, and per row its factor and the sums of its groups
    uint32_t q[kGroups][4][2];
    uint32_t sums;
    float factor[2];
    int last[2];  // the last key of the two rows that this lane's scores belong to
    const int row = row0 + g;
    const int token = row / c.groups;
    const bool real = row < piece.tokens * c.groups;
    const QT* src = reinterpret_cast<const QT*>(c.query + (piece.first_token + static_cast<int64_t>(real ? token : 0)) * c.query_ts +
                                                static_cast<int64_t>(head * c.groups + (real ? row - token * c.groups : 0)) * c.query_hs);
    float x[kGroups][16], most = 0.0f, sum[kGroups];
#pragma unroll
    for (int G = 0; G < kGroups; ++G) {
      const QT* from = src + G * 64 + t * 8;  // 8 dimensions of each 32
      if (c.aligned) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(from + i * 32));
          const QT* e = reinterpret_cast<const QT*>(&v);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[G][i * 8 + j] = real ? Elem<QT>::to_f(e[j]) : 0.0f;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[G][j] = real ? Elem<QT>::to_f(from[(j >> 3) * 32 + (j & 7)]) : 0.0f;
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
    // 2^e, with the scale's sign: the factors that come after are positive
    const float up = copysignf(__int_as_float((e + 127) << 23), c.scale_log2);
#pragma unroll
    for (int G = 0; G < kGroups; ++G)
#pragma unroll
      for (int j = 0; j < 2; ++j)  // a word of 8 codes: dimensions (0, 4) (1, 5) (2, 6) (3, 7)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* w = &x[G][j * 8 + h * 2];
          q[G][j * 2 + h][0] = pack(w[0] * up, w[4] * up);
          q[G][j * 2 + h][1] = pack(w[1] * up * 0.0625f, w[5] * up * 0.0625f);
        }
    // the sums of the groups in the codes' unit 2^-24, as three fp16 limbs (at most 2^-3, to
    // 2^-25): K steps 2 t and 2 t + 1 of the lane's t hold both groups' limb t
    float limb[kGroups];
#pragma unroll
    for (int G = 0; G < kGroups; ++G) {
      float left = sum[G] * up * 5.9604645e-8f;
      limb[G] = 0.0f;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const float part = __half2float(__float2half_rn(left));
        if (t == i) limb[G] = part;
        left -= part;
      }
    }
    sums = pack(limb[0], kGroups == 2 ? limb[kGroups - 1] : 0.0f);
    // 2^24 of the codes, less the row's own power of two; not 0, so that a logit of -inf stays one
    const float f = fmaxf(fabsf(c.scale_log2) * __int_as_float((127 - e) << 23) * 16777216.0f, 1e-30f);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = 2 * t + j;
      factor[j] = __shfl_sync(0xffffffffu, f, col * 4);
      last[j] = piece.before + min(row0 + col, piece.tokens * c.groups - 1) / c.groups;
    }

    float o[kChunks][2][4], eights[4], low[kGroups][2], m[2], l[2];
    eights[0] = eights[1] = eights[2] = eights[3] = 0.0f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.0f;
#pragma unroll
    for (int G = 0; G < kGroups; ++G) low[G][0] = low[G][1] = 0.0f;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[ch][i][j] = 0.0f;

    // a tile; CUT: some row does not see some key of it, or a step is not finite, which without CUT
    // is found before anything has changed (false)
    auto consume = [&](auto cut_tag, int key0, uint32_t buf, uint32_t mask) -> bool {
      constexpr bool CUT = decltype(cut_tag)::value;
      const uint32_t rows_at = buf + L::where(lane & 15, lane >> 4);
      const uint32_t pairs_at = buf + 2 * L::kCodes + g * 2 * L::kPairs;

      // ---- products of 2 x 16 keys (rows g and g + 8 of each), in the unit of `factor`, and
      // the pairs of the V rows with the largest step among this lane's
      float w[2][4];
      uint32_t vpair[2][2][kGroups];
      __half2 most = __half2half2(__ushort_as_half(0));
      uint32_t rows_of[2][kGroups][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int G = 0; G < kGroups; ++G) load_rows(rows_of[mt][G], (rows_at ^ (G * 32)) + mt * 16 * L::kRow);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t pair[2][kGroups], lows[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          load_pairs<kGroups>(pair[r], vpair[mt][r], pairs_at + (mt * 16 + r * 8) * 2 * L::kPairs);
          lows[r] = kGroups == 2 ? __byte_perm(pair[r][0], pair[r][kGroups - 1], 0x7632) : pair[r][0] >> 16;
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            if constexpr (CUT) {
              if (!((mask >> (mt * 16 + r * 8 + g)) & 1u)) vpair[mt][r][G] = 0;
              // A group whose step is not finite goes by its lowest value alone, made NaN: a factor of NaN
              // would meet the other group's zeros in the sums of factors, an infinite one would set M.
              if ((vpair[mt][r][G] & 0x7c00u) == 0x7c00u) vpair[mt][r][G] = 0x7e000000u;
            }
            most = __hmax2_nan(most, __habs2(*reinterpret_cast<const __half2*>(&vpair[mt][r][G])));
          }
        }
        float acc[kGroups][4];
        mma_new(w[mt], lows[0], lows[1], 0u, 0u, sums, 0u);
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          const uint32_t (&x)[4] = rows_of[mt][G];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a = x[j & 2] >> (8 * (j & 1)), b = x[(j & 2) + 1] >> (8 * (j & 1));
            if (j == 0)
              mma_new(acc[G], a & kEven, b & kEven, a & kOdd, b & kOdd, q[G][j][0], q[G][j][1]);
            else
              mma(acc[G], a & kEven, b & kEven, a & kOdd, b & kOdd, q[G][j][0], q[G][j][1]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            const float step = __low2float(*reinterpret_cast<const __half2*>(&pair[r][G]));
#pragma unroll
            for (int j = 0; j < 2; ++j) w[mt][r * 2 + j] = fmaf(step, acc[G][r * 2 + j], w[mt][r * 2 + j]);
          }
        if constexpr (CUT) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = mt * 16 + (j >> 1) * 8 + g;
            if (key0 + key > last[j & 1] || !((mask >> key) & 1u)) w[mt][j] = -INFINITY;
          }
        }
      }
      // steps below 2^-24 do not exist in fp16, but rows of step 0 do
      const float room = lg2(max_nan(__low2float(most), 5.9604645e-8f));

      // ---- the reference M moves only when a factor would pass 2^15: the largest logit with the largest
      // step is a bound on them (NaN where a step is, which counts as passed, as -inf does while there is no M)
      bool stay = true;
#pragma unroll
      for (int j = 0; j < 2; ++j)
        stay &= fmaf(fmaxf(fmaxf(w[0][j], w[0][j + 2]), fmaxf(w[1][j], w[1][j + 2])), factor[j], room) < m[j] + kMostRoom;
      if (!__all_sync(0xffffffffu, stay)) {
        if constexpr (!CUT)
          if (!__all_sync(0xffffffffu, room < INFINITY)) return false;
        // M goes by the factors themselves: set by the bound, a large step of a key that hardly weighs, or
        // that the row does not see, would take the bits of those that do
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            __half2 step = __habs2(*reinterpret_cast<const __half2*>(&vpair[mt][r][0]));
            if constexpr (kGroups == 2) step = __hmax2(step, __habs2(*reinterpret_cast<const __half2*>(&vpair[mt][r][kGroups - 1])));
            const float own = lg2(fmaxf(__low2float(step), 5.9604645e-8f));
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (!CUT || w[mt][r * 2 + j] != -INFINITY) top[j] = fmaxf(top[j], fmaxf(fmaf(w[mt][r * 2 + j], factor[j], own), kLeast));
          }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float high = top[j];
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
          if (high > m[j] + kMostRoom) {
            const float now = high - kSetRoom;
            const float keep = m[j] == -INFINITY ? 0.0f : ex2(m[j] - now);
            m[j] = now;
            l[j] *= keep;
#pragma unroll
            for (int G = 0; G < kGroups; ++G) low[G][j] *= keep;
            eights[j] *= keep, eights[j + 2] *= keep;
#pragma unroll
            for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
              for (int i = 0; i < 2; ++i) o[ch][i][j] *= keep, o[ch][i][j + 2] *= keep;
          }
        }
      }
      float ref[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) ref[j] = CUT && m[j] == -INFINITY ? 0.0f : -m[j];

      // ---- P and the products with V
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        uint32_t b[kGroups][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float p[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            p[j] = ex2(fmaf(w[mt][r * 2 + j], factor[j], ref[j]));
            l[j] += p[j];
          }
#pragma unroll
          for (int G = 0; G < kGroups; ++G) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&vpair[mt][r][G]));
            const float middle = fmaf(8.0f, f.x, f.y);  // of a row's values: what code 8 stands for
            float by[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // an unseen row gives nothing whatever it holds
              const bool none = CUT && w[mt][r * 2 + j] == -INFINITY;
              by[j] = none ? 0.0f : p[j] * f.x;
              low[G][j] = none ? low[G][j] : fmaf(p[j], middle, low[G][j]);
            }
            b[G][r] = transposed(pack(by[0], by[1]));
          }
        }
#pragma unroll
        for (int G = 0; G < kGroups; ++G) {
          uint32_t x[4];  // four codes of keys 2 t and 2 t + 1, of 2 t + 8 and 2 t + 9; the next chunk's
          load_columns(x, (rows_at ^ (G * 32)) + L::kCodes + mt * 16 * L::kRow);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t near = x[j & 2] >> (8 * (j & 1)), far = x[(j & 2) + 1] >> (8 * (j & 1));
            mma(o[G * 2 + (j >> 1)][j & 1], near & kEven, near & kOdd, far & kEven, far & kOdd, b[G][0], b[G][1]);
          }
          // 8 times the sums of the rounded factors, the first group's in rows 0-7
          mma(eights, G == 0 ? kEight : 0u, G == 0 ? 0u : kEight, G == 0 ? kEight : 0u, G == 0 ? 0u : kEight, b[G][0], b[G][1]);
        }
      }
      return true;
    };

    int stage = 0;
    for (int tile = tile0 + warp; tile < tile1; tile += kRound) {
      issue(stage == 0 ? kStages - 1 : stage - 1);
      copy_wait<kStages - 1>();
      __syncwarp();
      const uint32_t buf = ring_at + stage * L::kBytes;
      const uint32_t mask = live[warp][stage];
      const int key0 = tile * kTileKeys;
      if (mask != 0xffffffffu || key0 + kTileKeys > all_see || !consume(std::false_type{}, key0, buf, mask))
        consume(std::true_type{}, key0, buf, mask);
      __syncwarp();  // the stage may be filled again
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    copy_wait<0>();

    // ---- the warps' parts meet
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
#pragma unroll
        for (int G = 0; G < kGroups; ++G) low[G][j] += __shfl_xor_sync(0xffffffffu, low[G][j], x);
      }
      if (g == 0) {
        const int row = 2 * t + j;
        row_m[warp][row] = m[j];
        row_l[warp][row] = l[j];
#pragma unroll
        for (int G = 0; G < kGroups; ++G) low_sum[warp][row][G] = low[G][j] - eights[2 * G + j] * 16777216.0f;
      }
    }
    __syncthreads();  // every warp is done with its ring as well
    float* join = reinterpret_cast<float*>(dyn);  // [warp][row][D + 8], dimensions as the fragments hold them
    constexpr int kJoinRow = D + 8;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float* dst = join + (warp * kRows + 2 * t + j) * kJoinRow + g * 2;
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
        for (int i = 0; i < 2; ++i)  // the codes' 2^24, and 2^20 for the odd nibbles
          *reinterpret_cast<float2*>(dst + (ch * 2 + i) * 16) =
              make_float2(o[ch][i][j] * 16777216.0f, o[ch][i][j + 2] * 1048576.0f);
    }
    __syncthreads();
    const bool whole = piece.whole;
    const int rows = min(kRows, piece.tokens * c.groups - row0);
    float* part = c.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (tile0 == 0)) * kRows * (D + 2);
    for (int x = threadIdx.x; x < rows * (D / 2); x += kThreads) {
      const int row = x / (D / 2), pair = x - row * (D / 2);  // two neighbouring dimensions
      const int G = pair / 32, dim = pair / 16 * 32 + (pair & 7) * 4 + ((pair >> 3) & 1) * 2;
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
        const float inverse = top == -INFINITY ? 0.0f : 1.0f / sum;  // a row that sees no key is zeros
        const int r = row0 + row, token = r / c.groups;
        QT* dst = reinterpret_cast<QT*>(c.out + (piece.first_token + static_cast<int64_t>(token)) * c.out_ts +
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
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Joins the parts of one row of a piece that was cut: part 1 of its first CTA, then part 0 of
// the CTAs that follow, always in that order.  A warp takes every eighth part.
template <int D, typename QT>
__global__ void __launch_bounds__(kThreads) join4_kernel(const Params c) {
  constexpr int kPer = D / 32;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the parts are still written
  const Cut cut = c.meta[blockIdx.x];
  if (cut.followers < 0) return;
  const int row = blockIdx.y, r = cut.row0 + row;
  if (r >= cut.rows) return;
  __shared__ float tops[kWarps], sums[kWarps], values[kWarps][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* const mine = c.parts + (static_cast<int64_t>(blockIdx.x) * 2 + 1) * kRows * (D + 2) + row * (D + 2);
  auto part_of = [&](int i) -> const float* {  // part 1 of this CTA, part 0 of the i-th after it
    return mine + (i == 0 ? int64_t(0) : (2 * static_cast<int64_t>(i) - 1) * kRows * (D + 2));
  };
  float top = -INFINITY, sum = 0.0f, value[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) value[j] = 0.0f;
  constexpr int kAtOnce = 4;  // parts whose loads are in flight together
  for (int i0 = warp; i0 <= cut.followers; i0 += kAtOnce * kWarps) {
    float pm[kAtOnce], pl[kAtOnce], v[kAtOnce][kPer];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * kWarps;
      pm[u] = -INFINITY, pl[u] = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[u][j] = 0.0f;
      if (i <= cut.followers) {
        const float* p = part_of(i);
        pm[u] = p[0], pl[u] = p[1];
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[u][j] = p[2 + j * 32 + lane];
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float now = fmaxf(top, pm[u]);
      const float keep = top == -INFINITY ? 0.0f : ex2(top - now), by = pm[u] == -INFINITY ? 0.0f : ex2(pm[u] - now);
      top = now;
      sum = sum * keep + pl[u] * by;
#pragma unroll
      for (int j = 0; j < kPer; ++j) value[j] = value[j] * keep + v[u][j] * by;
    }
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
    QT* dst = reinterpret_cast<QT*>(c.out + (cut.first_token + static_cast<int64_t>(token)) * c.out_ts +
                                    static_cast<int64_t>(cut.head * c.groups + r - token * c.groups) * c.out_hs) + d;
    *dst = Elem<QT>::from_f(all == -INFINITY ? 0.0f : v / l);
  }
}

// ---------------------------------------------------------------- host side
constexpr size_t kMetaBytes = (kCtas * sizeof(Cut) + 255) / 256 * 256;
size_t workspace(int64_t head_size) {
  return kMetaBytes + static_cast<size_t>(kCtas) * 2 * kRows * (head_size + 2) * sizeof(float);
}

template <int D, typename QT>
int launch(const Params& c, cudaStream_t s) {
  // rows that a piece can have: a group's, where each sequence has one token
  const int rows = c.start == nullptr ? std::min(kRows, c.groups) : kRows;
  constexpr size_t kBytes = smem_bytes<D>();
  int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(attention4_kernel<D, QT>), kBytes);
  if (rc != CB_OK) return rc;
  attention4_kernel<D, QT><<<kCtas, kThreads, kBytes, s>>>(c);
  rc = launch_status("cb_paged_attention4");
  if (rc != CB_OK) return rc;
  if (c.uncut) return CB_OK;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(kCtas, rows), config.blockDim = dim3(kThreads), config.stream = s;
  cudaLaunchAttribute attribute;  // the join's CTAs may come up before the parts are there; they wait
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute, config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, join4_kernel<D, QT>, c);
  if (e != cudaSuccess) {
    set_error("cb_paged_attention4 (join) launch failed: %s", cudaGetErrorString(e));
    return CB_ERR_CUDA;
  }
  return launch_status("cb_paged_attention4 (join)");
}

template <typename QT>
int dispatch(const Params& c, int64_t head_size, cudaStream_t s) {
  return head_size == 128 ? launch<128, QT>(c, s) : launch<64, QT>(c, s);
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
  *bytes = num_tokens == 0 ? 0 : static_cast<int64_t>(att4::workspace(head_size));
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
  CB_REQUIRE(std::isfinite(scale * att4::kLog2e), "the scale must be finite (got %g)", static_cast<double>(scale));
  if (num_tokens == 0) return CB_OK;
  CB_REQUIRE(query_start != nullptr || num_tokens == num_seqs, "one token per sequence, or query_start");
  CB_REQUIRE(num_blocks >= 0 && num_blocks < (int64_t(1) << 31) && block_size > 0 && block_size < (int64_t(1) << 22) &&
                 table_width >= 0 && table_width * block_size < (int64_t(1) << 30),
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
  CB_REQUIRE((reinterpret_cast<uint64_t>(workspace) & 31u) == 0, "the workspace must be 32-byte aligned");
  CB_REQUIRE(workspace_bytes >= static_cast<int64_t>(att4::workspace(head_size)), "workspace too small (%lld < %zu)",
             (long long)workspace_bytes, att4::workspace(head_size));
  att4::Params c{};
  c.query = static_cast<const char*>(query), c.query_ts = query_token_stride, c.query_hs = query_head_stride;
  c.out = static_cast<char*>(out), c.out_ts = out_token_stride, c.out_hs = out_head_stride;
  c.tokens = num_tokens, c.start = query_start, c.lens = seq_lens, c.table = block_table, c.table_stride = table_stride;
  c.num_seqs = static_cast<int>(num_seqs), c.width = num_blocks > 0 ? static_cast<int>(table_width) : 0;
  c.heads_kv = static_cast<int>(num_kv_heads), c.groups = static_cast<int>(groups);
  c.codes[0] = static_cast<const char*>(k_codes), c.codes[1] = static_cast<const char*>(v_codes);
  c.scales[0] = static_cast<const char*>(k_scales), c.scales[1] = static_cast<const char*>(v_scales);
  CB_REQUIRE(block_stride >= 0 && slot_stride >= 0 && head_stride >= 0 && scale_block_stride >= 0 && scale_slot_stride >= 0 &&
                 scale_head_stride >= 0,
             "negative stride");
  const auto reach = [&](int64_t block, int64_t slot, int64_t head) {
    return static_cast<double>(num_blocks) * block + static_cast<double>(block_size) * slot +
           static_cast<double>(num_kv_heads) * head;
  };
  CB_SUPPORTED(reach(block_stride, slot_stride, head_stride) < 68719476736.0 &&
                   reach(scale_block_stride, scale_slot_stride, scale_head_stride) < 17179869184.0,
               "pages of one plane span 64 GiB of codes or 16 GiB of steps");
  c.block_stride = static_cast<uint32_t>(block_stride / 16), c.slot_stride = static_cast<uint32_t>(slot_stride / 16);
  c.head_stride = static_cast<uint32_t>(head_stride / 16);
  c.scale_block_stride = static_cast<uint32_t>(scale_block_stride / 4);
  c.scale_slot_stride = static_cast<uint32_t>(scale_slot_stride / 4);
  c.scale_head_stride = static_cast<uint32_t>(scale_head_stride / 4);
  c.num_blocks = static_cast<uint32_t>(num_blocks), c.block_size = static_cast<int>(block_size);
  c.step_pages = att4::kRound * att4::kTileKeys / c.block_size;
  c.step_rows = att4::kRound * att4::kTileKeys % c.block_size;
  c.scale_log2 = scale * att4::kLog2e;
  c.aligned = (rows & 15u) == 0;
  c.uncut = c.width * block_size <= att4::kUncutKeys;
  c.meta = static_cast<att4::Cut*>(workspace);
  c.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + att4::kMetaBytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == CB_DTYPE_BF16 ? att4::dispatch<__nv_bfloat16>(c, head_size, s) : att4::dispatch<__half>(c, head_size, s);
}
