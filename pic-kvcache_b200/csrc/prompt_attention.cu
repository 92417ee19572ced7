// Causal attention of a packed batch of prompts, on the 5th-generation tensor
// cores.
//
// Sequence i owns the query rows query_start[i] .. and the key rows key_start[i]
// ..; its n queries are the last n of its k keys, so query j sees the keys at or
// before k - n + j of its own sequence:
//   out = softmax(scale q k^T over the seen keys) v,  head h on KV head h / groups
// Logits, softmax and sums are fp32; the unnormalized probabilities are rounded
// to the element type for the second product (2^-8 bf16, 2^-11 fp16, relative,
// each its own: about what rounding the output costs; an fp16 one below 2^-21 of the
// largest is off by 2^-32 of that instead), and O is divided by the fp32 row sum at the end.
//
// Rows are (query, group) pairs of one KV head, so a K / V tile serves the whole
// group; a tile is 128 / groups queries (the last rows of a tile whose group
// count does not divide 128 are idle).  An item is one KV head and a pair of
// query tiles A and B.  Where there are more of them than SMs, a first launch lists
// the items of all sequences, the longest first (a counting sort), and the persistent CTAs take the next one of the
// list as they come to their last two K tiles (dealt out beforehand, the slowest of 148
// CTAs took 9 % longer than the median).  Per CTA, 12 warps:
//   warp 0   takes items; Q per item, K tiles through a ring of two (TMA)
//   warp 3   V tiles through a ring of three, see below (with two, P V waited for V:
//            it is given back only once the next S is seen)
//   warp 1   tcgen05.mma: P_A V (t), S_A (t + 1), P_B V (t), S_B (t + 1), ..., from
//            an item's last tile straight into the next item's first S
//   warp 2   TMEM: S_A, S_B, O_A, O_B, all 512 columns
//   warps 4-7 / 8-11   softmax of A / B, a row per thread
// P goes back to TMEM over the columns of its own S and is the A operand of P V
// from there: with P in shared memory the products would read A and B of both
// (8 KiB per 64 cycles and product, all of shared memory's 128 bytes a clock) and
// P's stores and the TMA's would come on top, 3,072 cycles a tile pair against
// 2,048 of the tensor cores; from TMEM it is 2,048.  The price is that S (t + 1)
// of a tile waits for its P V (t), so A and B take turns: while one is in its
// softmax the tensor cores have the other's two products.  P is handed over in
// two halves, and P V begins on the first.
// O is rescaled only when a row's maximum grows by more than 2^8 (until then the
// stale one keeps every exp2 <= 2^8, or 2^15 in fp16); that P V (t - 1) is finished is known from
// S (t), which was issued behind it.
//
// Masked places: a logit that a row does not see is replaced, whatever it is.  A
// value row that some row of the item does not see meets a probability of 0, and
// 0 x NaN is NaN: the V warp looks through the tiles at the diagonal and at the
// end of a sequence, puts 0 in the place of NaN and infinities there, and the
// epilogue of such an item (rare) adds them to the rows that do see them.
// Every mbarrier wait is bounded (2 s): a wait that runs out records a code in
// *device_error, the CTA drains its MMAs and loads, frees TMEM and returns.
//
// What bounds it (16,384 tokens, 32 heads on 8, D 128: 1,635 us, 1,345 TFLOP/s; 1,850 to
// 1,900 us once the power cap holds the clocks): the chain S, P, P V, S of one tile, 2,880
// cycles even where it runs alone, in a pair's period of 3,150; the tensor cores and the
// MUFU (16 exp2 a clock) need 2,048 each.
// The softmax warps' code is kept short: what runs once per item is fetched anew each
// time (about 4 cycles an instruction).  One copy of the tile's code for whole and
// masked tiles and rolled loops in the epilogue took 9 prompts of 8,500 tokens from
// 152 to 144 us.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cb_common.cuh"
#include "cb_tcgen05.cuh"

namespace cb {
namespace prompt {
using namespace ::cb::tc;

constexpr int kPair = 2;     // query tiles per item, one softmax warpgroup each
constexpr int kKStages = 2;
constexpr int kVStages = 3;
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;  // S_A [0,128) S_B [128,256) O_A [256,384) O_B [384,512)
constexpr uint32_t kTmemO = 256;
// 128 control threads x 56 + 256 softmax threads x 224 = 64512 = 384 x 168 at launch
constexpr int kRegsControl = 56;
constexpr int kRegsSoftmax = 224;
static_assert(4 * 32 * kRegsControl + 8 * 32 * kRegsSoftmax <= kThreads * 168, "register split");
constexpr float kRescaleLog2 = 8.0f;
// Where the reference is set, below the row's maximum: an fp16 probability is then 2^7 there (2^15 at most
// before the reference moves), so that fp16's subnormals, 2^-25 off, are 2^-32 of the largest and not
// 2^-25, which over the keys of a long context would be more than the rounding of the result.
template <typename T>
constexpr float kSetLog2 = std::is_same<T, __half>::value ? 7.0f : 0.0f;
constexpr float kLog2e = 1.4426950408889634f;

// One pair of query tiles of one sequence (for every KV head).
struct alignas(16) Item {
  int q_row;    // its first query row
  int queries;  // valid queries, at most kPair * queries per tile
  int k_row;    // the sequence's first key row
  int pos;      // the last key (of the sequence) that the first query sees; may be negative
};

struct Params {
  int kv_heads, groups, tile_queries;  // queries per tile: 128 / groups
  float scale_log2;                    // scale * log2(e)
  const Item* items;  // null: an item per CTA, found from the sequences' starts
  int* num_items;  // and behind it how many were taken beyond the first of each CTA
  const int32_t* query_start;  // without a list
  const int32_t* key_start;
  int num_seqs, num_queries, num_keys;
  const char* value;  // for the epilogue of items with values that are not finite
  int64_t value_ts, value_hs;
  char* out;
  int64_t out_ts, out_hs;  // bytes
  int32_t* error;
};

struct Shared {
  uint64_t q_full[kPair], q_empty[kPair];
  uint64_t k_full[kKStages], k_empty[kKStages];
  uint64_t v_landed[kVStages], v_full[kVStages], v_empty[kVStages];
  uint64_t s_full[kPair], p_full[kPair][2];
  uint64_t o_full[kPair], o_empty[kPair];
  uint64_t work_full, work_empty;
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
  int pairs;  // pairs of query tiles of all sequences
  Item work;  // the CTA's current item, and its KV head; -1: no more
  int work_head;
  int odd_values;  // a boundary tile held values that are not finite (stays set)
};

__device__ __forceinline__ void report(const Params& c, Shared& sh, int code) {
  if (c.error != nullptr) atomicCAS(c.error, 0, code);
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
}
__device__ __forceinline__ bool aborted(Shared& sh) { return *reinterpret_cast<volatile int*>(&sh.abort) != 0; }

__device__ __forceinline__ Item load_item(const Params& c, int pair) {
  const int4 v = *reinterpret_cast<const int4*>(c.items + pair);
  return Item{v.x, v.y, v.z, v.w};
}
// The k-th item of the CTA, as the thread that loads Q and K publishes it (the first before the
// CTA's barrier).  False: the wait ran out.
template <bool WARP>
__device__ __forceinline__ bool take(Shared& sh, int k, Item& w, int& head) {
  if (k > 0 && !(WARP ? wait_warp(&sh.work_full, (k - 1) & 1) : wait1(&sh.work_full, (k - 1) & 1))) return false;
  w = sh.work, head = sh.work_head;
  if constexpr (WARP) __syncwarp();
  if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(&sh.work_empty);
  return true;
}
// A sequence's rows: starts are clamped to the rows there are.
__device__ __forceinline__ void span(const int32_t* start, int i, int most, int& first, int& length) {
  first = min(max(start[i], 0), most);
  length = min(max(start[i + 1], first), most) - first;
}
// Valid queries of tile x of an item, and its key tiles: up to the last key its last query sees.
__device__ __forceinline__ int tile_valid(const Params& c, const Item& w, int x) {
  return min(max(w.queries - x * c.tile_queries, 0), c.tile_queries);
}
__device__ __forceinline__ int tile_count(const Params& c, const Item& w, int x) {
  const int valid = tile_valid(c, w, x), last = w.pos + x * c.tile_queries + valid - 1;
  return valid > 0 && last >= 0 ? last / kTile + 1 : 0;
}

// An item for a CTA that will soon be done with its last: the longest that is left.
__device__ __forceinline__ int claim(const Params& c) {
  return static_cast<int>(gridDim.x) + (c.items != nullptr ? atomicAdd(c.num_items + 1, 1) : 0);
}
__device__ __forceinline__ void publish(const Params& c, Shared& sh, int item) {
  const int pair = item / c.kv_heads;
  const bool there = c.items != nullptr && pair < sh.pairs;  // without a list a CTA has one item
  sh.work_head = there ? item - pair * c.kv_heads : -1;
  if (there) sh.work = load_item(c, pair);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 32 lanes x 16 consecutive columns of this warp's TMEM sub-partition, stored.
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// 16 rows of 16-byte pieces: lane 4 g + t holds word t of each piece of row g (even registers) and of
// row g + 8 (odd ones).
__device__ __forceinline__ void tmem_ld_rows(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x128b.x8.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15"
      "}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_rows(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x128b.x16.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31"
      "}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
template <typename T, int N>
__host__ __device__ constexpr uint32_t instr_desc() {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// Four K steps (64 dims) of S = Q K^T, both operands 128-row K-major halves in shared memory
// (descriptors' low words).  One asm block: the issuing thread keeps no descriptor in registers.
__device__ __forceinline__ void product_s(uint32_t tmem_d, uint32_t q_lo, uint32_t k_lo, uint32_t idesc, bool onto) {
  static_assert(kstep_lo(1) == 2, "K-step offsets baked into product_s");
  asm volatile(
      "{\n\t.reg .b64 da, db;\n\t.reg .b32 a, b;\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t"
      "add.u32 a, %1, 2;\n\tadd.u32 b, %2, 2;\n\t"
      "mov.b64 da, {a, %5};\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, 1;\n\t"
      "add.u32 a, %1, 4;\n\tadd.u32 b, %2, 4;\n\t"
      "mov.b64 da, {a, %5};\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, 1;\n\t"
      "add.u32 a, %1, 6;\n\tadd.u32 b, %2, 6;\n\t"
      "mov.b64 da, {a, %5};\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, 1;\n\t}" ::"r"(tmem_d),
      "r"(q_lo), "r"(k_lo), "r"(idesc), "r"(onto ? 1u : 0u), "n"(kDescHi));
}
// O += P V over 64 keys: P from TMEM (two elements a column, 8 columns a K step), V [keys][D]
// MN-major in shared memory (16 keys further: 2 KiB).
__device__ __forceinline__ void product_pv(uint32_t tmem_d, uint32_t tmem_p, uint32_t v_lo, uint32_t idesc, bool onto) {
  asm volatile(
      "{\n\t.reg .b64 db;\n\t.reg .b32 a, b;\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t"
      "add.u32 a, %1, 8;\n\tadd.u32 b, %2, 128;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, 1;\n\t"
      "add.u32 a, %1, 16;\n\tadd.u32 b, %2, 256;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, 1;\n\t"
      "add.u32 a, %1, 24;\n\tadd.u32 b, %2, 384;\n\tmov.b64 db, {b, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [a], db, %3, 1;\n\t}" ::"r"(tmem_d),
      "r"(tmem_p), "r"(v_lo), "r"(idesc), "r"(onto ? 1u : 0u), "n"(kDescHi));
}

// Values that are not finite, to a row that sees them: 32 dimensions of the sum over the item's
// boundary tiles, where the product had zeros instead.
template <typename T>
__device__ __forceinline__ void add_odd(uint32_t (&o)[32], const Params& c, const Item& w, int h, int q, int pos) {
#pragma unroll 1
  for (int key = max(w.pos + 1, 0); key <= pos; ++key) {
    const T* row = reinterpret_cast<const T*>(c.value + (static_cast<int64_t>(w.k_row) + key) * c.value_ts + h * c.value_hs);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const float y = Elem<T>::to_f(row[q * 32 + j]);
      if (!(fabsf(y) <= 3.4e38f)) o[j] = __float_as_uint(__uint_as_float(o[j]) + y);
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map, const __grid_constant__ Params c) {
  constexpr int kHalves = D / 64;
  constexpr int kBytes = kHalves * kHalfBytes;  // a full operand tile
  extern __shared__ __align__(1024) unsigned char dyn[];
  __shared__ Shared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~static_cast<uintptr_t>(1023));
  unsigned char* q_buf = base;
  unsigned char* k_buf = base + kPair * kBytes;
  unsigned char* v_buf = k_buf + kKStages * kBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) mbar_init(&sh.k_full[s], 1), mbar_init(&sh.k_empty[s], 1);
    for (int s = 0; s < kVStages; ++s)
      mbar_init(&sh.v_landed[s], 1), mbar_init(&sh.v_full[s], 1), mbar_init(&sh.v_empty[s], 1);
    for (int x = 0; x < kPair; ++x) {
      mbar_init(&sh.q_full[x], 1), mbar_init(&sh.q_empty[x], 1);
      mbar_init(&sh.s_full[x], 1);
      mbar_init(&sh.p_full[x][0], 4), mbar_init(&sh.p_full[x][1], 4);
      mbar_init(&sh.o_full[x], 1), mbar_init(&sh.o_empty[x], 4);
    }
    mbar_init(&sh.work_full, 1), mbar_init(&sh.work_empty, 10);
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    sh.odd_values = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {  // the CTA's first item
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the list of items is there
    const int pair = blockIdx.x / c.kv_heads, head = blockIdx.x - pair * c.kv_heads;
    if (c.items == nullptr) {  // no list: a lane per sequence
      const int pair_queries = kPair * c.tile_queries;
      int q_row = 0, queries = 0, k_row = 0, keys = 0;
      if (lane < c.num_seqs) {
        span(c.query_start, lane, c.num_queries, q_row, queries);
        span(c.key_start, lane, c.num_keys, k_row, keys);
      }
      const int mine = (queries + pair_queries - 1) / pair_queries;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      if (pair < upto && pair >= upto - mine) {
        const int first = (pair - (upto - mine)) * pair_queries;
        sh.work = Item{q_row + first, min(queries - first, pair_queries), k_row, keys - queries + first};
      }
      if (lane == 31) sh.pairs = upto, sh.work_head = pair < upto ? head : -1;
    } else if (lane == 0) {  // (all CTAs' first entries lie in the list's memory, used or not)
      sh.work = load_item(c, pair);
      sh.pairs = *c.num_items;
      sh.work_head = pair < sh.pairs ? head : -1;
    }
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == 0) {
      // ------------------------------------------------------ Q and K loads
      if (lane == 0) {
        const uint32_t q_half = static_cast<uint32_t>(c.tile_queries * c.groups * 128);  // bytes of a loaded half tile
        int t = 0, next = 0;
        int loads[kPair] = {0, 0};           // of Q, per tile of the pair
        uint32_t k_armed = 0, k_parity = 0;  // per stage: a load is in flight / its phase parity
        bool ok = true;
        for (int k = 0; !aborted(sh); ++k) {
          if (k > 0) {  // the next item, once every other role has read the last one
            if (!wait1(&sh.work_empty, (k - 1) & 1)) { ok = false; break; }
            publish(c, sh, next);
            mbar_arrive(&sh.work_full);
          }
          const Item w = sh.work;
          const int h = sh.work_head;
          if (h < 0) break;
          const int n[kPair] = {tile_count(c, w, 0), tile_count(c, w, 1)};
          const int tiles = max(n[0], n[1]);
          if (tiles == 0) {
            next = claim(c);
            continue;
          }
          auto load_q = [&](int x) -> bool {
            if (n[x] == 0) return true;
            if (!wait1(&sh.q_empty[x], (loads[x] & 1) ^ 1)) return false;
            mbar_expect_tx(&sh.q_full[x], kHalves * q_half);
            for (int i = 0; i < kHalves; ++i)
              tma_load_4d(q_buf + x * kBytes + i * kHalfBytes, &q_map, &sh.q_full[x], i * 64, 0, h,
                          w.q_row + x * c.tile_queries);
            ++loads[x];
            return true;
          };
          ok = load_q(0);
          for (int kt = 0; ok && kt < tiles; ++kt, ++t) {
            const int s = t % kKStages;
            if (kt == max(tiles - 2, 0)) next = claim(c);  // its latency is hidden, and no CTA holds two for long
            if (!wait1(&sh.k_empty[s], ((t / kKStages) & 1) ^ 1)) { ok = false; break; }
            mbar_expect_tx(&sh.k_full[s], kBytes);
            for (int i = 0; i < kHalves; ++i)
              tma_load_3d(k_buf + s * kBytes + i * kHalfBytes, &k_map, &sh.k_full[s], i * 64, h, w.k_row + kt * kTile);
            k_armed |= 1u << s;
            k_parity = (k_parity & ~(1u << s)) | (static_cast<uint32_t>((t / kKStages) & 1) << s);
            if (kt == 0) ok = load_q(1);  // its tile's slot is the last to be given back
          }
          if (!ok) break;
        }
        if (!ok) report(c, sh, 1);
        // every armed load has landed before the CTA may exit
        for (int s = 0; s < kKStages; ++s)
          if ((k_armed >> s) & 1u) wait1(&sh.k_full[s], (k_parity >> s) & 1u);
        for (int x = 0; x < kPair; ++x)
          if (loads[x] > 0) wait1(&sh.q_full[x], (loads[x] - 1) & 1);
      }
    } else if (warp == 3) {
      // ------------------------------------------------------ V loads, and a look at boundary tiles
      int t = 0, issued = 0;  // tiles so far, and of them the loads that are on their way or done
      bool ok = true;
      constexpr uint32_t kExp2 = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
      constexpr uint32_t kOne2 = std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
      // hands tile u on once it has landed; `from`: its first key that some row does not see
      auto hand_on = [&](int u, int from) -> bool {
        const int s = u % kVStages;
        if (!wait_warp(&sh.v_landed[s], (u / kVStages) & 1)) return false;
        if (from < kTile) {
          // a lane looks at the same 16 bytes of every fourth row; an exponent of all ones carries
          // into its element's sign bit
          uint32_t carries = 0;
          for (int half = 0; half < kHalves; ++half) {
            const uint4* rows = reinterpret_cast<const uint4*>(v_buf + s * kBytes + half * kHalfBytes) + (lane & 7);
#pragma unroll 8
            for (int row = from + (lane >> 3); row < kTile; row += 4) {
              const uint4 v = rows[row * 8];
              carries |= ((v.x & kExp2) + kOne2) | ((v.y & kExp2) + kOne2) | ((v.z & kExp2) + kOne2) | ((v.w & kExp2) + kOne2);
            }
          }
          const bool odd = __any_sync(0xffffffffu, (carries & 0x80008000u) != 0);
          if (odd) {
            constexpr uint32_t kExp = kExp2 & 0xffffu;
            for (int half = 0; half < kHalves; ++half) {
              uint32_t* words = reinterpret_cast<uint32_t*>(v_buf + s * kBytes + half * kHalfBytes) + lane;
              for (int row = from; row < kTile; ++row) {
                uint32_t e = words[row * 32];
                if ((e & kExp) == kExp) e &= 0xffff0000u;
                if (((e >> 16) & kExp) == kExp) e &= 0xffffu;
                words[row * 32] = e;
              }
            }
          }
          if (odd) *reinterpret_cast<volatile int*>(&sh.odd_values) = 1;
          fence_async_smem();  // the replaced values -> the MMA's async-proxy reads
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&sh.v_full[s]);
        return true;
      };
      int held = -1, held_from = 0;  // the tile loaded last, where it is not handed on yet
      for (int k = 0; ok && !aborted(sh); ++k) {
        // the next item may wait for what the products make of the last tile
        if (k > 0 && held >= 0 && !__all_sync(0xffffffffu, mbar_try(&sh.work_full, (k - 1) & 1))) {
          ok = hand_on(held, held_from);
          held = -1;
        }
        Item w;
        int h;
        if (!ok || !take<true>(sh, k, w, h)) { ok = false; break; }
        if (h < 0) break;
        const int tiles = max(tile_count(c, w, 0), tile_count(c, w, 1));
        for (int kt = 0; kt < tiles && ok; ++kt, ++t) {
          const int s = t % kVStages;
          const uint32_t free_parity = ((t / kVStages) & 1) ^ 1;
          // the tile before this one goes on first, unless this one's slot is free already
          if (held >= 0 && !__all_sync(0xffffffffu, mbar_try(&sh.v_empty[s], free_parity))) {
            ok = hand_on(held, held_from);
            held = -1;
          }
          if (!ok || !wait_warp(&sh.v_empty[s], free_parity)) { ok = false; break; }
          if (lane == 0) {
            mbar_expect_tx(&sh.v_landed[s], kBytes);
            for (int i = 0; i < kHalves; ++i)
              tma_load_3d(v_buf + s * kBytes + i * kHalfBytes, &v_map, &sh.v_landed[s], i * 64, h, w.k_row + kt * kTile);
          }
          __syncwarp();
          ++issued;
          if (held >= 0) ok = hand_on(held, held_from);
          held = t, held_from = max(w.pos + 1 - kt * kTile, 0);
        }
      }
      if (held >= 0 && ok) ok = hand_on(held, held_from);
      if (!ok && lane == 0) report(c, sh, 4);
      // every armed load has landed before the CTA may exit
      for (int u = max(issued - kVStages, 0); u < issued; ++u) wait_warp(&sh.v_landed[u % kVStages], (u / kVStages) & 1);
    } else if (warp == 1) {
      // ------------------------------------------------------ MMA issuer
      if (lane == 0) {
        constexpr uint32_t kDescS = instr_desc<T, kTile>();
        constexpr uint32_t kDescPV = instr_desc<T, D>() | (1u << 16);  // B (V) MN-major
        const uint32_t q_addr = smem_u32(q_buf), k_addr = smem_u32(k_buf), v_addr = smem_u32(v_buf);
        const uint32_t tmem = sh.tmem_base;
        int ks = 0, vs = 0;                        // ring slots and their parities: running, since the
        uint32_t kp = 0, vp = 0;                   // divisions would stand between two products
        uint32_t pp[kPair] = {0, 0}, op[kPair] = {1, 1}, qp[kPair] = {0, 0};  // parities of P, of O's release, of Q
        bool ok = true;
        auto issue_s = [&](int x) {
#pragma unroll
          for (int i = 0; i < kHalves; ++i)
            product_s(tmem + x * kTile, desc_lo(q_addr + x * kBytes + i * kHalfBytes),
                      desc_lo(k_addr + ks * kBytes + i * kHalfBytes), kDescS, i > 0);
          umma_commit(&sh.s_full[x]);
        };
        auto issue_pv = [&](int x, int half, uint32_t v_rows, bool onto) {
          tc_fence_after();
          product_pv(tmem + kTmemO + x * kTile, tmem + x * kTile + half * 32, desc_lo_mn(v_rows + half * 64 * 128), kDescPV,
                     onto);
        };
        auto wait_o = [&](int x) -> bool {  // its last item's rows have been read
          op[x] ^= 1;
          return wait1(&sh.o_empty[x], op[x] ^ 1);
        };
        auto next_k = [&]() {
          if (++ks == kKStages) ks = 0, kp ^= 1;
        };
        int n[kPair], items = 0;
        // the next item; false: none.  Its key tiles are 0 where its queries see nothing.
        auto next_item = [&]() -> bool {
          Item w;
          int h;
          if (!take<false>(sh, items++, w, h)) ok = false;
          if (!ok || h < 0) return false;
          n[0] = tile_count(c, w, 0), n[1] = tile_count(c, w, 1);
          return true;
        };
        // the first S of query tile x of that item
        auto start = [&](int x) {
          if (n[x] > 0 && ok) {
            ok = wait1(&sh.q_full[x], qp[x]) && wait1(&sh.k_full[ks], kp);
            qp[x] ^= 1;
            tc_fence_after();
            if (ok) issue_s(x);
          }
          if (x == 1) next_k();
        };
        bool more = next_item(), started = false;
        while (more && ok && !aborted(sh)) {
          const int m[kPair] = {n[0], n[1]};
          const int tiles = max(m[0], m[1]);
          if (tiles == 0) {
            more = next_item();
            continue;
          }
          if (!started) start(0), start(1);
          started = false;
          ok = ok && wait1(&sh.v_full[vs], vp);  // (V of each next tile is looked for behind P V)
          int kt = 0;
          // Tiles that both query tiles have a successor of.  Every look at a barrier stands where the
          // products issued before it still have time to run (the issue of a product waits for the
          // third before it, so 200 cycles); a wait that ran out is acted on at the end of the round.
          for (; ok && kt + 1 < min(m[0], m[1]); ++kt) {
            const uint32_t v_rows = v_addr + vs * kBytes;
            const bool onto = kt > 0;
            if (!onto) ok = wait_o(0);
            ok = wait1(&sh.p_full[0][0], pp[0]) && ok;
            issue_pv(0, 0, v_rows, onto);
            ok = wait1(&sh.k_full[ks], kp) && ok;
            ok = wait1(&sh.p_full[0][1], pp[0]) && ok;
            issue_pv(0, 1, v_rows, true);
            issue_s(0);
            if (!onto) ok = wait_o(1) && ok;
            ok = wait1(&sh.p_full[1][0], pp[1]) && ok;
            issue_pv(1, 0, v_rows, onto);
            ok = wait1(&sh.p_full[1][1], pp[1]) && ok;
            issue_pv(1, 1, v_rows, true);
            if (++vs == kVStages) vs = 0, vp ^= 1;
            ok = wait1(&sh.v_full[vs], vp) && ok;
            issue_s(1);
            next_k();
            pp[0] ^= 1, pp[1] ^= 1;
          }
          // the last tiles of either; behind the very last ones the next item's first S
          for (; ok && kt < tiles; ++kt) {
            const uint32_t v_rows = v_addr + vs * kBytes;
            const bool final = kt + 1 == tiles;
            bool have_k = final;
#pragma unroll
            for (int x = 0; x < kPair; ++x) {
              if (kt < m[x]) {
                if (kt == 0) ok = wait_o(x) && ok;
                ok = wait1(&sh.p_full[x][0], pp[x]) && ok;
                issue_pv(x, 0, v_rows, kt > 0);
                if (!have_k) ok = wait1(&sh.k_full[ks], kp) && ok;
                have_k = true;
                ok = wait1(&sh.p_full[x][1], pp[x]) && ok;
                issue_pv(x, 1, v_rows, true);
                pp[x] ^= 1;
                if (kt + 1 < m[x])
                  issue_s(x);
                else
                  umma_commit(&sh.o_full[x]);
              }
              if (final) {
                if (x == 0) more = next_item(), started = more && max(n[0], n[1]) > 0;
                if (started) start(x);
              }
            }
            if (++vs == kVStages) vs = 0, vp ^= 1;
            if (!final) {
              next_k();
              ok = ok && wait1(&sh.v_full[vs], vp);
            }
          }
        }
        if (!ok) report(c, sh, 2);
        umma_commit(&sh.drain);
        wait1(&sh.drain, 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ------------------------------------------------------ softmax / epilogue
    const int x = (warp - 4) >> 2;           // query tile of the pair
    const int ew = warp & 3;                 // TMEM lanes 32*ew .. +31
    const int row_in_tile = ew * 32 + lane;  // this thread's row
    const uint32_t lane_off = static_cast<uint32_t>(ew * 32) << 16;
    const uint32_t s_tmem = sh.tmem_base + x * kTile + lane_off;
    const uint32_t o_tmem = sh.tmem_base + kTmemO + x * kTile + lane_off;
    const int query_in_tile = row_in_tile / c.groups, group = row_in_tile - query_in_tile * c.groups;
    const int first_query = x * c.tile_queries + ew * 32 / c.groups;  // of the warp's rows
    // This warpgroup gives back what its products were the last to read: K of a tile (and Q with the
    // item's last) once its S is there, V once the next S, or O, is.  The MMA thread would need a
    // commit for each, and a commit behind a commit holds it up until the first has arrived (470
    // cycles of a tile pair's 3,600).
    const bool keeper = ew == 0 && lane == 0;
    int t = 0, o_count = 0, tiles_before = 0;
    bool ok = true;
    for (int k = 0;; ++k) {
      Item w;
      int h;
      if (!take<true>(sh, k, w, h)) { ok = false; break; }
      if (h < 0) break;
      const int n = tile_count(c, w, x), n_b = tile_count(c, w, 1);
      auto last_reader = [&](int kt) { return x == 1 || kt >= n_b; };
      const bool store = query_in_tile < tile_valid(c, w, x);
      const int pos = w.pos + x * c.tile_queries + query_in_tile;  // the last key this row sees
      float m_used = -INFINITY;  // what the exponentials are taken against, in the log2 domain
      float l = 0.0f;
      // whole tiles: up to the last key that the warp's first row sees
      const int first_pos = w.pos + first_query;
      const int whole = min(max(first_pos + 1, 0) / kTile, n);
      // a tile of S
      auto softmax_tile = [&](int kt) {
        if (keeper) {
          if (last_reader(kt)) mbar_arrive(&sh.k_empty[(tiles_before + kt) % kKStages]);
          if (kt > 0 && last_reader(kt - 1)) mbar_arrive(&sh.v_empty[(tiles_before + kt - 1) % kVStages]);
          if (kt + 1 == n) mbar_arrive(&sh.q_empty[x]);
        }
        tc_fence_after();
        uint32_t v[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(s_tmem + q * 32, v[q]);
        tmem_wait_ld();
        if (kt >= whole) {
          const int valid = pos - kt * kTile + 1;
#pragma unroll
          for (int q = 0; q < 4; ++q)  // most of a diagonal tile's quarters are seen by the whole warp
            if (!__all_sync(0xffffffffu, valid >= (q + 1) * 32)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (q * 32 + j >= valid) v[q][j] = __float_as_uint(-INFINITY);
            }
        }
        auto s_of = [&](int j) { return __uint_as_float(v[j >> 5][j & 31]); };
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = fmaxf(s_of(2 * i), s_of(2 * i + 1));
#pragma unroll
        for (int j = 4; j < 64; ++j) mx[j & 3] = max3(mx[j & 3], s_of(2 * j), s_of(2 * j + 1));
        const float tile_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c.scale_log2;
        const bool grow = tile_max > m_used + (kSetLog2<T> + kRescaleLog2) || (m_used == -INFINITY && tile_max > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = grow ? tile_max - kSetLog2<T> : m_used;
          const float corr = grow ? (m_used == -INFINITY ? 0.0f : ex2(m_used - m_new)) : 1.0f;
          if (kt > 0) {  // O holds earlier tiles of this item, all finished: rescale its rows
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              uint32_t o[32];
              tmem_ld32(o_tmem + q * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
              tmem_st32(o_tmem + q * 32, o);
            }
            tmem_wait_st();
          }
          l *= corr;
          m_used = m_new;
        }
        // a row that sees nothing keeps m_used = -inf: its p are exact zeros
        const float base_m = m_used == -INFINITY ? 0.0f : -m_used;
        const float2 nm = make_float2(base_m, base_m), mul = make_float2(c.scale_log2, c.scale_log2);
        float2 sm[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sm[i] = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int part = 0; part < 4; ++part) {  // P of 32 keys: 16 columns over the S that was read
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 s2 = make_float2(s_of(part * 32 + 2 * j), s_of(part * 32 + 2 * j + 1));
            const float2 e2 = __ffma2_rn(s2, mul, nm);
            const float2 p2 = make_float2(ex2(e2.x), ex2(e2.y));
            sm[j & 3] = __fadd2_rn(sm[j & 3], p2);
            packed[j] = pack2<T>(p2.x, p2.y);
          }
          tmem_st16(s_tmem + part * 16, packed);
          if (part & 1) {  // 64 keys: the first of the product's two halves, or the second
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[x][part >> 1]);
          }
        }
        const float2 st = __fadd2_rn(__fadd2_rn(sm[0], sm[1]), __fadd2_rn(sm[2], sm[3]));
        l += st.x + st.y;
      };
      int kt = 0;
#pragma unroll 1
      for (; kt < n; ++kt, ++t) {
        if (!wait_warp(&sh.s_full[x], t & 1)) { ok = false; break; }
        softmax_tile(kt);
      }
      if (!ok) break;
      if (n > 0) {
        if (!wait_warp(&sh.o_full[x], o_count & 1)) { ok = false; break; }
        ++o_count;
        if (keeper && last_reader(n - 1)) mbar_arrive(&sh.v_empty[(tiles_before + n - 1) % kVStages]);
        tc_fence_after();
      }
      tiles_before += max(n, tile_count(c, w, x ^ 1));
      // the P V of the item's boundary tiles came after their look-through
      const bool odd = *reinterpret_cast<volatile int*>(&sh.odd_values) != 0;
      const bool seen = n > 0 && pos >= 0;
      // (2 ulp at most.)  A row that sees no key is zeros; one that does, and of whose logits no weight is
      // left (all -inf), 0 / 0.
      const float inv = pos >= 0 ? __fdividef(1.0f, l) : 0.0f;
      // A row per thread, so a store of 16 bytes each would touch 32 lines (47 cycles of the load/store
      // unit, 6,000 for the item's two tiles, with the other warps' loads behind them).  The packed
      // rows go back to TMEM, over O, and come again as (row, 16 bytes) by lane / 4 and lane % 4:
      // 64 bytes of eight rows a store.
      char* const dst = c.out + (static_cast<int64_t>(w.q_row) + x * c.tile_queries + query_in_tile) * c.out_ts +
                        static_cast<int64_t>(h * c.groups + group) * c.out_hs;
      auto row_of = [&](int i) {  // where the lane's piece of its i-th row goes
        const unsigned long long at =
            __shfl_sync(0xffffffffu, store ? reinterpret_cast<unsigned long long>(dst) : 0ull, i * 8 + (lane >> 2));
        return at == 0 ? nullptr : reinterpret_cast<char*>(at) + (lane & 3) * 16;
      };
      if (n > 0) {
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          tmem_ld32(o_tmem + q * 32, o);
          tmem_wait_ld();
          if (odd && seen && store) add_odd<T>(o, c, w, h, q, pos);
          uint32_t word[16];  // word 4 t + i of the 64 bytes at column 4 i + t
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 y = __fmul2_rn(make_float2(__uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1])), make_float2(inv, inv));
            word[(j & 3) * 4 + (j >> 2)] = pack2<T>(y.x, y.y);
          }
          tmem_st16(o_tmem + q * 16, word);
        }
        tmem_wait_st();
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {  // 16 rows
          uint32_t v[D / 4];
          tmem_ld_rows(o_tmem + (static_cast<uint32_t>(half * 16) << 16), v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            char* const row = row_of(half * 2 + i);
            if (row != nullptr)
#pragma unroll
              for (int q = 0; q < D / 32; ++q)
                *reinterpret_cast<uint4*>(row + q * 64) =
                    make_uint4(v[q * 8 + i], v[q * 8 + 2 + i], v[q * 8 + 4 + i], v[q * 8 + 6 + i]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.o_empty[x]);
      } else {  // the item's rows see nothing
        for (int i = 0; i < 4; ++i) {
          char* const row = row_of(i);
          if (row != nullptr)
#pragma unroll
            for (int q = 0; q < D / 32; ++q) *reinterpret_cast<uint4*>(row + q * 64) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    if (!ok && lane == 0) report(c, sh, 3);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem_base), "r"(kTmemCols) : "memory");
  }
}

// ---------------------------------------------------------------- the list of items
constexpr int kListThreads = 1024;
constexpr int kBuckets = 2048;  // key tiles of an item; longer ones share the last

// Counting sort of all pairs of query tiles by their key tiles, longest first.  One CTA; the
// order inside a bucket is whatever the atomics give, which moves work between CTAs but
// changes no result.
__global__ void __launch_bounds__(kListThreads) list_kernel(const int32_t* __restrict__ query_start,
                                                            const int32_t* __restrict__ key_start, int num_seqs,
                                                            int num_queries, int num_keys, int pair_queries, int capacity,
                                                            Item* __restrict__ items, int* __restrict__ num_items) {
  __shared__ int count[kBuckets], warp_sum[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the products' CTAs set themselves up meanwhile
  for (int b = threadIdx.x; b < kBuckets; b += kListThreads) count[b] = 0;
  __syncthreads();
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = warp; i < num_seqs; i += kListThreads / 32) {
      int q0, qn, k0, kn;
      span(query_start, i, num_queries, q0, qn);
      span(key_start, i, num_keys, k0, kn);
      const int pairs = (qn + pair_queries - 1) / pair_queries;
      for (int p = lane; p < pairs; p += 32) {
        Item w;
        w.q_row = q0 + p * pair_queries;
        w.queries = min(qn - p * pair_queries, pair_queries);
        w.k_row = k0;
        w.pos = kn - qn + p * pair_queries;
        const int last = w.pos + w.queries - 1;
        const int b = kBuckets - 1 - min(last >= 0 ? last / kTile + 1 : 0, kBuckets - 1);  // longest first
        if (pass == 0) {
          atomicAdd(&count[b], 1);
        } else {
          const int at = atomicAdd(&count[b], 1);
          if (at < capacity) items[at] = w;
        }
      }
    }
    __syncthreads();
    if (pass == 0) {  // exclusive scan of the counts
      constexpr int kPer = kBuckets / kListThreads;
      int mine[kPer], sum = 0;
      for (int j = 0; j < kPer; ++j) mine[j] = count[threadIdx.x * kPer + j], sum += mine[j];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      if (lane == 31) warp_sum[warp] = before;
      __syncthreads();
      int base = 0, total = 0;
      for (int u = 0; u < 32; ++u) {
        if (u < warp) base += warp_sum[u];
        total += warp_sum[u];
      }
      before += base - sum;
      for (int j = 0; j < kPer; ++j) count[threadIdx.x * kPer + j] = before, before += mine[j];
      if (threadIdx.x == 0) num_items[0] = min(total, capacity), num_items[1] = 0;
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------- host side
// Pairs of query tiles: at most one part pair per sequence more than whole ones.
int64_t most_items(int64_t num_queries, int64_t num_seqs, int64_t groups) {
  const int64_t pair_queries = kPair * (kTile / groups);
  return num_queries / pair_queries + num_seqs;
}
size_t workspace(int64_t items) { return 256 + static_cast<size_t>(items) * sizeof(Item); }

template <int D>
constexpr size_t smem_bytes() {
  return 1024 + (kPair + kKStages + kVStages) * (D / 64) * static_cast<size_t>(kHalfBytes);
}
static_assert(smem_bytes<128>() + 1024 <= 232448, "shared memory per CTA (static part padded to 1 KiB)");

int check_shape(int64_t num_queries, int64_t num_seqs, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size) {
  CB_SUPPORTED(head_size == 64 || head_size == 128, "prompt attention supports heads of 64 or 128 values (got %lld)",
               (long long)head_size);
  CB_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0,
             "query heads must be a multiple of KV heads");
  CB_SUPPORTED(num_q_heads / num_kv_heads <= kTile, "at most 128 query heads to a KV head");
  CB_REQUIRE(num_queries >= 0 && num_seqs >= 0, "negative size");
  CB_REQUIRE(num_seqs < (int64_t(1) << 20) && num_queries < (int64_t(1) << 30) && num_kv_heads < (int64_t(1) << 16),
             "size out of range");
  CB_REQUIRE(most_items(num_queries, num_seqs, num_q_heads / num_kv_heads) < (int64_t(1) << 30) / num_kv_heads,
             "size out of range");
  return CB_OK;
}

template <typename T, int D>
int launch(const CUtensorMap& q_map, const CUtensorMap& k_map, const CUtensorMap& v_map, const Params& c, int64_t items,
           cudaStream_t s) {
  constexpr size_t kBytes = smem_bytes<D>();
  const int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(prompt_kernel<T, D>), kBytes);
  if (rc != CB_OK) return rc;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(items * c.kv_heads, kSmCount)));
  if (c.items == nullptr) {
    prompt_kernel<T, D><<<grid, kThreads, kBytes, s>>>(q_map, k_map, v_map, c);
    return launch_status("cb_prompt_attention");
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(kThreads), config.dynamicSmemBytes = kBytes, config.stream = s;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute, config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, prompt_kernel<T, D>, q_map, k_map, v_map, c);
  if (e != cudaSuccess) {
    set_error("cb_prompt_attention launch failed: %s", cudaGetErrorString(e));
    return CB_ERR_CUDA;
  }
  return launch_status("cb_prompt_attention");
}

}  // namespace prompt
}  // namespace cb

using namespace cb;

extern "C" int cb_prompt_attention_workspace_size(int64_t num_queries, int64_t num_seqs, int64_t num_q_heads,
                                                  int64_t num_kv_heads, int64_t head_size, int64_t* bytes) {
  clear_error();
  CB_REQUIRE(bytes != nullptr, "null output");
  const int rc = prompt::check_shape(num_queries, num_seqs, num_q_heads, num_kv_heads, head_size);
  if (rc != CB_OK) return rc;
  *bytes = num_queries == 0 ? 0
                            : static_cast<int64_t>(prompt::workspace(
                                  prompt::most_items(num_queries, num_seqs, num_q_heads / num_kv_heads)));
  return CB_OK;
}

extern "C" int cb_prompt_attention(const void* query, int64_t query_token_stride, int64_t query_head_stride,
                                   const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                                   int64_t value_token_stride, int64_t value_head_stride, int64_t num_queries,
                                   int64_t num_keys, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_size,
                                   int dtype, const int32_t* query_start, const int32_t* key_start, int64_t num_seqs,
                                   float scale, void* out, int64_t out_token_stride, int64_t out_head_stride,
                                   void* workspace, int64_t workspace_bytes, int32_t* device_error, void* stream) {
  CB_BIND(stream, out);
  CB_SUPPORTED(dtype == CB_DTYPE_BF16 || dtype == CB_DTYPE_FP16, "prompt attention needs bf16 or fp16");
  int rc = prompt::check_shape(num_queries, num_seqs, num_q_heads, num_kv_heads, head_size);
  if (rc != CB_OK) return rc;
  CB_REQUIRE(num_keys >= 0 && num_keys < (int64_t(1) << 30), "size out of range");
  CB_REQUIRE(scale > 0.0f && std::isfinite(scale * prompt::kLog2e), "the scale must be positive and finite (got %g)",
             static_cast<double>(scale));
  if (num_queries == 0 || num_seqs == 0) return CB_OK;
  CB_REQUIRE(query && query_start && key_start && out && workspace, "null pointer argument");
  CB_REQUIRE(num_keys == 0 || (key && value), "null key or value pointer");
  const uint64_t acc = reinterpret_cast<uint64_t>(query) | reinterpret_cast<uint64_t>(key) |
                       reinterpret_cast<uint64_t>(value) | reinterpret_cast<uint64_t>(out) | (uint64_t)query_token_stride |
                       (uint64_t)query_head_stride | (uint64_t)key_token_stride | (uint64_t)key_head_stride |
                       (uint64_t)value_token_stride | (uint64_t)value_head_stride | (uint64_t)out_token_stride |
                       (uint64_t)out_head_stride | reinterpret_cast<uint64_t>(workspace);
  CB_SUPPORTED((acc & 15u) == 0, "prompt attention needs 16-byte aligned rows and strides");
  const int64_t groups = num_q_heads / num_kv_heads;
  const int64_t items = prompt::most_items(num_queries, num_seqs, groups);
  CB_REQUIRE(workspace_bytes >= static_cast<int64_t>(prompt::workspace(items)), "workspace too small (%lld < %zu)",
             (long long)workspace_bytes, prompt::workspace(items));
  const int tile_queries = static_cast<int>(tc::kTile / groups);
  tc::EncodeTiled encode = nullptr;
  rc = tc::get_encoder(&encode);
  if (rc != CB_OK) return rc;
  CUtensorMap q_map, k_map, v_map;
  {
    // query as (dims, group, KV head, token)
    const uint64_t dims[4] = {static_cast<uint64_t>(head_size), static_cast<uint64_t>(groups),
                              static_cast<uint64_t>(num_kv_heads), static_cast<uint64_t>(num_queries)};
    const uint64_t strides[3] = {static_cast<uint64_t>(query_head_stride), static_cast<uint64_t>(groups * query_head_stride),
                                 static_cast<uint64_t>(query_token_stride)};
    rc = tc::encode_4d(encode, &q_map, dtype, query, dims, strides, static_cast<uint32_t>(groups), 1,
                       static_cast<uint32_t>(tile_queries));
  }
  if (num_keys == 0) k_map = v_map = q_map;  // every row is zeros, and neither map is used
  if (rc == CB_OK && num_keys > 0)
    rc = tc::encode_3d(encode, &k_map, dtype, key, head_size, num_kv_heads, num_keys, key_head_stride, key_token_stride, 1,
                       tc::kTile);
  if (rc == CB_OK && num_keys > 0)
    rc = tc::encode_3d(encode, &v_map, dtype, value, head_size, num_kv_heads, num_keys, value_head_stride,
                       value_token_stride, 1, tc::kTile);
  if (rc != CB_OK) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  prompt::Params c{};
  c.kv_heads = static_cast<int>(num_kv_heads), c.groups = static_cast<int>(groups), c.tile_queries = tile_queries;
  c.scale_log2 = scale * prompt::kLog2e;
  c.value = static_cast<const char*>(value), c.value_ts = value_token_stride, c.value_hs = value_head_stride;
  c.out = static_cast<char*>(out), c.out_ts = out_token_stride, c.out_hs = out_head_stride;
  c.error = device_error;
  c.query_start = query_start, c.key_start = key_start;
  c.num_seqs = static_cast<int>(num_seqs), c.num_queries = static_cast<int>(num_queries), c.num_keys = static_cast<int>(num_keys);
  // An item per CTA and a sequence per lane: each finds its own, and there is one launch less (4
  // prompts of 300 tokens: 9.9 us, 12.5 with it).  Not where CTAs take several: the list kernel also clears their counter.
  if (num_seqs > 32 || items * num_kv_heads > kSmCount) {
    int* num_items = static_cast<int*>(workspace);
    prompt::Item* list = reinterpret_cast<prompt::Item*>(static_cast<char*>(workspace) + 256);
    c.items = list, c.num_items = num_items;
    prompt::list_kernel<<<1, prompt::kListThreads, 0, s>>>(query_start, key_start, static_cast<int>(num_seqs), c.num_queries,
                                                           c.num_keys, prompt::kPair * tile_queries,
                                                           static_cast<int>(items), list, num_items);
    rc = launch_status("cb_prompt_attention (list)");
    if (rc != CB_OK) return rc;
  }
  if (dtype == CB_DTYPE_BF16)
    return head_size == 128 ? prompt::launch<__nv_bfloat16, 128>(q_map, k_map, v_map, c, items, s)
                            : prompt::launch<__nv_bfloat16, 64>(q_map, k_map, v_map, c, items, s);
  return head_size == 128 ? prompt::launch<__half, 128>(q_map, k_map, v_map, c, items, s)
                          : prompt::launch<__half, 64>(q_map, k_map, v_map, c, items, s);
}
