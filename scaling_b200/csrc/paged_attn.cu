// Attention of new tokens over a paged key/value cache for sm_100a: one decoding token or a long chunk per sequence,
// MQA / GQA, causal or not, local windows.  (src/scaling/core/nn/attention/attention.py:846-884 concatenates the cache of
// one sequence at every step and runs variable-length attention on it.)
//
// For query row i (a token and head) at position pos_i with visible keys J_i = [lo_i, hi_i):
//   out_i = sum_{j in J_i} p_ij v_j / sum_j p_ij,   p_ij = 2^(sl2 q_i k_j - ref_i),   sl2 = scale log2(e)
// with a running reference ref_i: it follows the row maximum only when that grows by more than 2^8, so the accumulated
// output is rescaled a few times per row instead of at every step; any reference gives the same quotient and
// p_ij <= 2^8 stays far from overflow in both 16-bit types and in the fp32 sums.
//
// Two kernels share the frame.  An item is a block of query rows (tokens x heads that share a KV head, token-major) of one
// sequence and KV head.  All items together are a line of 128-key tiles that is cut into equal pieces, one per CTA (one CTA
// per SM): ragged lengths are balanced without the host knowing them.  A piece that starts or ends inside an item leaves an
// unnormalised partial result; a last kernel joins them in the order of the CTAs, so results do not depend on timing.
// K and V tiles come by TMA through a ring that does not know items: the loaders run ahead into the next ones.
//
// Wide (sequences with more than 64 rows): matrix products.  Items of 256 rows, S = Q K^T with query rows in the 128 TMEM
//   lanes.  Two groups of four softmax warps (thread = query row = lane), each with an MMA warp of its own, so that the
//   tensor core computes for one while the other takes exponentials.  Items of more than 128 rows give each group 128
//   rows of its own ("two_q"); smaller items give both the same rows and half the keys of each tile, and join the two
//   states at the end.  A group works on half tiles of 64 keys with two S in TMEM, so it never waits for the product that follows its
//   own probabilities; these overwrite the first half of their S as packed 16-bit values and are the TMEM operand of
//   O += P V.  O stays in TMEM over the whole item.
// Narrow (at most 64 rows: decoding): a stream over K and V, so everything else has to be small against the tile's bytes.
//   Rows in lanes would leave most lanes and three of four warps idle; here the keys are in the lanes: S^T = K Q^T
//   [128 keys x rows], a thread takes the exponentials of one key for all rows, and O^T += V^T P [D x rows].  S^T of four
//   tiles is in flight.  The rows' references are shared by the four warps of a group, which agree once per tile whether
//   any score has outgrown them (then the tile's P is written again).
//
// Warp roles: 0-3 and 4-7 softmax groups, 10 scheduler, which also copies the queries.  Narrow: 8 and 11 TMA loaders of K and
// of V (a page of 16 tokens is a copy of its own, and one warp alone issues them no faster than the memory delivers), 9 MMA
// issuer.  Wide: 8 loader of both, 9 and 11 MMA issuers of the two groups.
//
// What bounds it, measured on one B200 (6.57 TB/s copy, 1634 TFLOP/s), device time in a captured graph:
//   decoding, 64 requests of up to 8000 tokens, 32 heads over 8 of 128, pages of 16: 147 to 150 us (5.9 to 6.0 TB/s, 0.90 to
//     0.92 of the copy): the stream of K and V.
//   decoding, two long contexts, 40 heads over one of 128: 43 to 45 us (2.9 TB/s): about 3 us per item end, the softmax of 40
//     rows per key and the joining of some 70 parts per row, against 20 us for the bytes.
//   chunks of 2048 tokens on long contexts, heads of 128: 420 to 440 us, 970 to 1015 TFLOP/s (0.59 to 0.62): per half tile the
//     chain S product -> wait -> 64 exponentials per row -> wait -> P V product; two groups and two S each hide most of it.
//     Calls back to back without pause take 474 to 482 us, because the power cap lowers the clock.
//   one request: 10.8 us (an eager call 30: the enqueue): launch, work line, queries, tile, epilogue in a chain.
//   24 ragged sequences of 1 to 300 new tokens: 55 to 60 us, two kernels one after the other on most SMs and 3 to 4 us per item.
//
// Rounding: scores, sums and outputs are fp32; P is rounded to the 16-bit element type for the second product, the output once.
// The rounding of P is the larger part of what a result is off: relative to the 64-bit value 0.0023 in bf16 and 0.00025 in
// fp16, where the output's rounding alone gives 0.0017 and 0.00021.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"

namespace {

constexpr int PA_TILE = 128;
constexpr int PA_HALF = 64;  // keys per step of the wide kernel
constexpr int PA_WIDE_ROWS = 256, PA_NARROW_ROWS = 64;  // rows per item (narrow: at most)
constexpr int PA_WARPS = 12;
constexpr int PA_THREADS = PA_WARPS * 32;
// registers per thread after the roles part: 128 x 80 + 256 x 208 = 63488 of the 384 x 168 that the launch holds
constexpr int PA_REGS_FEW = 80, PA_REGS_MANY = 208;
constexpr int PA_PANEL = 16384;   // 128 rows x 128 bytes
constexpr int PA_ITEMS = 4;       // descriptors in flight
// The tensor core truncates when it adds to TMEM: with equal weights an output of one was 0.997 after 2^20 keys and 0.987 after
// 2^22.  So a group's sums (O and the row sums) go to a second place after that many tiles of 128 keys (2^14 keys) and
// start from zero; what is added there is rounded to nearest.
constexpr int PA_FOLD = 128;
constexpr int PA_COMBINE_THREADS = 256;
// A wait can last as long as one item: 2^19 tiles at the longest.  Measured per tile: 2 to 3 us, 5.5 us where all CTAs read
// the same page; so 1 to 3 s, and some room for other work on the GPU.
constexpr unsigned long long PA_WAIT_NS = 10000000000ull;
// ROWS (rows per item) tells the kernels apart in the functions that they share.
template <int ROWS> struct PaKind {
  static constexpr bool NARROW = ROWS <= PA_NARROW_ROWS;
  static constexpr int SLOT_ROWS = NARROW ? ROWS : PA_TILE;  // rows per query slot
};

struct PaParams {
  const void* q;
  void* out;
  const int* table;
  const int* cu;
  const int* lens;
  long table_ld, q_tok, q_head, o_tok, o_head;
  int T, batch, Hkv, group, D, cols, num_pages, page_shift;
  uint32_t group_inv;  // floor(2^32 / group) + 1 (group > 1): (n * group_inv) >> 32 = n / group for n < 2^32 / group
  // layout of a K or V tile in shared memory: 8-row groups of 128-byte rows, `group_step` bytes apart, the second 64
  // columns `panel_step` bytes behind the first.  boxes: copies per page (1: both panels at once); page8: 8-row groups of
  // the tensor maps from one page to the next, outside: a group beyond the cache
  uint32_t group_step, panel_step;
  int boxes, k_page8, v_page8, k_outside, v_outside;
  int causal, window;  // window < 0: unlimited
  int narrow_max;      // sequences with at most this many rows belong to the narrow kernel
  int cost;            // what the start and the end of an item cost, in tiles: added to its length on the work line
  int whole;           // items count as one each and are not divided
  float sl2;
  float* part_o;       // [2 slots per CTA][part_rows][DP]
  float2* part_ml;     // [2 slots per CTA][part_rows]: reference (log2 domain) and sum
  int* part_desc;      // [CTAs][8]: item that starts in this CTA and ends in a later one (first word: there is one; -1: refused)
  int part_rows, zero_tail;
  int* status;
};

// One descriptor of the scheduler's ring.
struct PaItem {
  int row0, pos0;    // packed row and position of the item's first token
  int L, seq, hk;    // total tokens, sequence, KV head
  int rows, rem;     // query rows; the first one is head `rem` of the group
  int tile0, count;  // first key tile and number of key tiles (0: the end)
  int lo, hi;        // keys that some row of the item sees
  int slot;          // partial slot, or -1: the item is complete
};

template <int PANELS> struct PaCfg {
  static constexpr int DP = PANELS * 64;
  static constexpr int TILE_BYTES = PANELS * PA_PANEL;
  static constexpr int STAGES = PANELS == 2 ? 5 : 10;
  // wide: two slots of 128 query rows; narrow: two slots of 64 query rows and P of each group, [128 keys][64 rows]
  static constexpr int FRONT = 65536;
  static constexpr int DATA = FRONT + STAGES * TILE_BYTES;  // 224 KiB
  static constexpr int SMEM = DATA + 2048 + 1024;           // exchange between the softmax warps, control words
};

template <int STAGES> struct PaCtrl {
  uint64_t full[STAGES], empty[STAGES];  // ring
  uint64_t q_full[2], q_empty[2];
  uint64_t s_full[4], p_full[4], p_empty[4], merge[8], vote[2], fin, epi_done;
  uint64_t item_full[PA_ITEMS], item_empty[PA_ITEMS];
  PaItem items[PA_ITEMS];
  alignas(16) int need[2][2][4];  // narrow: [group][round parity][warp]
  uint32_t tmem_slot;
  int abort;
};
static_assert(sizeof(PaCtrl<10>) <= 1024, "control words");

__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16> __device__ __forceinline__ uint32_t pa_pack(float a, float b) {
  if constexpr (F16) {
    __half2 t = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}
__device__ __forceinline__ void pa_tma_5d(uint32_t dst, const void* tmap, uint64_t* bar, int x, int group8, int head) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(tmap), "r"(sb::smem_u32(bar)), "r"(x), "r"(0), "r"(group8), "r"(head)
      : "memory");
}
__device__ __forceinline__ float pa_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 pa_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 pa_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// Bounded wait: up to PA_WAIT_NS, then the flag is raised and every other wait of the CTA ends as well.
__device__ __forceinline__ bool pa_wait_lane(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (sb::mbar_try_wait(bar, parity)) return true;
  const unsigned long long start = sb::globaltimer_ns();
  for (uint32_t i = 1;; ++i) {
    if (sb::mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 0) {
      if (*abort_flag) return false;
      if (sb::globaltimer_ns() - start > PA_WAIT_NS) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
// Bounded wait of a whole warp: every lane gets the same answer, also when the wait gives up, so that no lane is missing
// from the warp-wide instructions that follow.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, pa_wait_lane(bar, parity, abort_flag));
}
// D[tmem] (+)= A[tmem] * B[smem]: A holds two 16-bit values of a row per 32-bit column
__device__ __forceinline__ void pa_umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <int N> __device__ __forceinline__ void pa_tmem_ld8(uint32_t taddr, uint32_t (&r)[N], int at) {
  static_assert(N >= 8, "");
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[at]), "=r"(r[at + 1]), "=r"(r[at + 2]), "=r"(r[at + 3]), "=r"(r[at + 4]), "=r"(r[at + 5]),
                 "=r"(r[at + 6]), "=r"(r[at + 7])
               : "r"(taddr)
               : "memory");
}
template <int N> __device__ __forceinline__ void pa_regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void pa_regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void pa_tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool take) {  // zeros when !take
  const int bytes = take ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void pa_tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ------------------------------------------------------------------------------------------------ work line
struct PaSeq { int row0, n, L; };

__device__ __forceinline__ PaSeq pa_seq(const PaParams& p, int b) {
  PaSeq s;
  const int start = p.cu[b], end = p.cu[b + 1];
  s.row0 = min(max(start, 0), p.T);
  s.n = min(max(end, s.row0), p.T) - s.row0;
  const long cap = (long)p.cols << p.page_shift;
  int L = p.lens[b];
  if (L < 0 || L > cap || start != s.row0 || end != s.row0 + s.n) {
    // a length that the table does not cover, rows that do not follow one another inside the T: reported, cut to what there is
    *p.status = SB_ERR_BAD_ARG;
    L = (int)min((long)max(L, 0), cap);
  }
  s.L = L;
  return s;
}
// n / group for n < group + 256
__device__ __forceinline__ int pa_div(const PaParams& p, int n) { return p.group == 1 ? n : (int)__umulhi(n, p.group_inv); }
// keys that some row of item m sees
template <int ROWS> __device__ __forceinline__ void pa_item_keys(const PaParams& p, int n, int L, int m, int& lo, int& hi) {
  const int rows = n * p.group;
  const int first = m * ROWS / p.group, last = (min(rows, (m + 1) * ROWS) - 1) / p.group;
  const int pos0 = L - n + first, pos1 = L - n + last;
  lo = p.window >= 0 ? max(0, pos0 - p.window) : 0;
  hi = p.causal ? pos1 + 1 : (p.window >= 0 ? (int)min((long)L, (long)pos1 + p.window + 1) : L);
  hi = max(min(hi, L), 0);
}
// key tiles between lo and hi, at least one: a row without keys still has to be written
__device__ __forceinline__ int pa_tiles(int lo, int hi) { return max((hi + PA_TILE - 1) / PA_TILE - lo / PA_TILE, 1); }
// length of item m on the line
template <int ROWS> __device__ __forceinline__ int pa_item_cost(const PaParams& p, int n, int L, int m) {
  if (p.whole) return 1;
  int lo, hi;
  pa_item_keys<ROWS>(p, n, L, m, lo, hi);
  return pa_tiles(lo, hi) + p.cost;
}
// items of a sequence of n new tokens in this kernel, per KV head
template <int ROWS> __device__ __forceinline__ int pa_items(const PaParams& p, int n) {
  const int rows = n * p.group;
  return (rows <= p.narrow_max) == PaKind<ROWS>::NARROW ? (rows + ROWS - 1) / ROWS : 0;
}
__device__ __forceinline__ int pa_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
// Sum over the lanes.  Lengths are kept in 32 bits: one that does not fit becomes the largest value, which pa_find refuses
// (a part of the whole that large makes the whole too large, however the sequences are grouped).
__device__ __forceinline__ int pa_sum(long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return (int)min(v, 0x7fffffffLL);
}
// Length of all items of one KV head of sequence 32 * chunk + lane (0 beyond the last sequence); the whole warp calls.
template <int ROWS> __device__ __forceinline__ int pa_chunk_cost(const PaParams& p, int chunk, int lane, PaSeq& s) {
  const int b = chunk * 32 + lane;
  s = PaSeq{0, 0, 0};
  if (b < p.batch) s = pa_seq(p, b);
  const int items = pa_items<ROWS>(p, s.n);
  int cost = items == 1 ? pa_item_cost<ROWS>(p, s.n, s.L, 0) : 0;
  unsigned many = __ballot_sync(0xffffffffu, items > 1);
  while (many) {  // the warp shares the items of one sequence
    const int src = __ffs(many) - 1;
    many &= many - 1;
    const int n = __shfl_sync(0xffffffffu, s.n, src), L = __shfl_sync(0xffffffffu, s.L, src);
    const int cnt = pa_items<ROWS>(p, n);
    long long mine = 0;
    for (int m = lane; m < cnt; m += 32) mine += pa_item_cost<ROWS>(p, n, L, m);
    const int sum = pa_sum(mine);
    if (lane == src) cost = sum;
  }
  return cost;
}

// The line is cut into `ctas` pieces of `per`, the first `rest` of them one longer.
struct PaCut {
  int ctas, per, rest;
  __device__ __forceinline__ int start(int c) const { return c * per + min(c, rest); }
  __device__ __forceinline__ int owner(int place) const {
    const int longer = rest * (per + 1);
    return place < longer ? place / (per + 1) : rest + (place - longer) / per;
  }
};
struct PaCursor {  // where a CTA's piece of the line starts, and how long it is; refused: the line is too long for any
  PaSeq s;
  int seq, hk, m, tile, left, place;
  bool refused;
  PaCut cut;
};

// The whole warp; sums[c] = length per KV head of sequences 32 c .. 32 c + 31.
template <int ROWS>
__device__ __forceinline__ void pa_find(const PaParams& p, const int* sums, int chunks, int lane, PaCursor& c) {
  c = PaCursor{};
  PaSeq s = {0, 0, 0};
  int cost = 0;  // of sequence 32 chunk + lane
  long long all = 0;
  if (chunks > 1) {
    for (int i = lane; i < chunks; i += 32) all += sums[i];
  } else {
    cost = pa_chunk_cost<ROWS>(p, 0, lane, s);
    all = cost;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  all *= p.Hkv;
  if (all >= 0x7fffffff) {  // half a minute of work and more: reported, the last kernel writes zeros
    if (lane == 0) *p.status = SB_ERR_TOO_LARGE;
    c.refused = true;
    return;
  }
  PaCut& cut = c.cut;
  const int total = (int)all;
  // two tiles per CTA at least, one for each softmax group
  cut.ctas = min((int)gridDim.x, p.whole ? total : (total + 1) / (2 + p.cost));
  if (total > 0) cut.ctas = max(cut.ctas, 1);
  if ((int)blockIdx.x >= cut.ctas) return;
  cut.per = total / cut.ctas;
  cut.rest = total - cut.per * cut.ctas;
  c.place = cut.start(blockIdx.x);
  c.left = cut.per + ((int)blockIdx.x < cut.rest);
  int off = c.place, chunk = 0;
  if (chunks > 1) {
    for (int base = 0; base < chunks; base += 32) {
      const int v = base + lane < chunks ? sums[base + lane] * p.Hkv : 0, inc = pa_scan(v, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, inc > off);
      if (hit) {
        const int k = __ffs(hit) - 1;
        chunk = base + k;
        off -= __shfl_sync(0xffffffffu, inc - v, k);
        break;
      }
      off -= __shfl_sync(0xffffffffu, inc, 31);
    }
    cost = pa_chunk_cost<ROWS>(p, chunk, lane, s);
  }
  const int v = cost * p.Hkv, inc = pa_scan(v, lane);
  const int k = __ffs(__ballot_sync(0xffffffffu, inc > off)) - 1;
  off -= __shfl_sync(0xffffffffu, inc - v, k);
  const int per_head = __shfl_sync(0xffffffffu, cost, k);
  c.s = PaSeq{__shfl_sync(0xffffffffu, s.row0, k), __shfl_sync(0xffffffffu, s.n, k), __shfl_sync(0xffffffffu, s.L, k)};
  c.seq = chunk * 32 + k;
  c.hk = off / per_head;
  off -= c.hk * per_head;
  const int items = pa_items<ROWS>(p, c.s.n);
  c.tile = off;
  if (items > 1) {
    for (int base = 0; base < items; base += 32) {
      const int t = base + lane < items ? pa_item_cost<ROWS>(p, c.s.n, c.s.L, base + lane) : 0, ti = pa_scan(t, lane);
      const unsigned hit = __ballot_sync(0xffffffffu, ti > off);
      if (hit) {
        const int j = __ffs(hit) - 1;
        c.m = base + j;
        c.tile = off - __shfl_sync(0xffffffffu, ti - t, j);
        break;
      }
      off -= __shfl_sync(0xffffffffu, ti, 31);
    }
  }
}

// Places of K and V tiles of an item in the ring: `lead` K tiles run ahead of V, then V and K alternate - the order in which
// the MMA warp takes them (narrow: 4; wide: 1 with two_q, else 2, the first S of both groups).
__device__ __forceinline__ uint32_t pa_k_place(int t, int lead) { return t < lead ? t : 2 * t - lead + 1; }
__device__ __forceinline__ uint32_t pa_v_place(int t, int lead, int count) { return t + min(t + lead, count); }
template <int ROWS> __device__ __forceinline__ int pa_lead(int rows) { return PaKind<ROWS>::NARROW ? 4 : rows > PA_TILE ? 1 : 2; }

// ============================================================================ roles that both kernels share
// Warp 10: cuts the piece into items, publishes their descriptors and copies their queries.
template <int ROWS, int PANELS>
__device__ __forceinline__ void pa_schedule(const PaParams& p, PaCtrl<PaCfg<PANELS>::STAGES>& c, uint8_t* sQ, int chunks,
                                            int lane) {
  constexpr int DP = PANELS * 64;
  constexpr int SLOT_ROWS = PaKind<ROWS>::SLOT_ROWS, SLOT_BYTES = PANELS * SLOT_ROWS * 128;
  volatile int* abort_flag = &c.abort;
  PaCursor cur;
  pa_find<ROWS>(p, reinterpret_cast<const int*>(sQ), chunks, lane, cur);
  __syncwarp();
  int* desc = p.part_desc + 8 * blockIdx.x;
  bool starts = false, ok = true;
  int q_cnt = 0;
  for (int i = 0; ok; ++i) {
    const int slot = i % PA_ITEMS;
    if (!pa_wait(&c.item_empty[slot], ((i / PA_ITEMS) & 1) ^ 1, abort_flag)) break;
    PaItem it = {};
    int lo, hi, tiles = 0;
    while (cur.left > 0) {  // the next item with a tile in this piece
      pa_item_keys<ROWS>(p, cur.s.n, cur.s.L, cur.m, lo, hi);
      tiles = pa_tiles(lo, hi);
      if (cur.tile < tiles) {
        const int take = p.whole ? tiles : min(tiles - cur.tile, cur.left);
        const bool first = cur.tile == 0, last = cur.tile + take == tiles;
        const int tok0 = cur.m * ROWS / p.group;
        it = PaItem{cur.s.row0 + tok0, cur.s.L - cur.s.n + tok0, cur.s.L, cur.seq, cur.hk,
                    min(cur.s.n * p.group - cur.m * ROWS, ROWS), cur.m * ROWS - tok0 * p.group,
                    lo / PA_TILE + cur.tile, take, lo, hi,
                    first && last ? -1 : 2 * (int)blockIdx.x + (first ? 1 : 0)};
        if (first && !last) {  // the CTA that starts an item names the one that ends it
          starts = true;
          if (lane == 0) {
            desc[1] = it.row0; desc[2] = it.rem; desc[3] = it.hk; desc[4] = it.rows;
            desc[5] = cur.cut.owner(cur.place + tiles - 1);
          }
        }
      }
      const int used = p.whole ? 1 : min(tiles + p.cost - cur.tile, cur.left);
      cur.left -= used;
      cur.place += used;
      cur.tile = 0;
      if (cur.left > 0 && ++cur.m == pa_items<ROWS>(p, cur.s.n)) {
        cur.m = 0;
        if (++cur.hk == p.Hkv) {
          cur.hk = 0;
          do { cur.s = pa_seq(p, ++cur.seq); } while (pa_items<ROWS>(p, cur.s.n) == 0 && cur.seq + 1 < p.batch);
        }
      }
      if (it.count) break;
    }
    if (lane == 0) {
      c.items[slot] = it;
      sb::mbar_arrive(&c.item_full[slot]);
    }
    if (it.count == 0) break;
    // queries: one slot, or two of them, as 16-byte chunks in the swizzled K-major layout, rows up to the next full block
    const int slots = it.rows > SLOT_ROWS ? 2 : 1;
    for (int x = 0; x < slots; ++x) {
      const int qs = (q_cnt + x) & 1;
      ok = pa_wait(&c.q_empty[qs], (((q_cnt + x) >> 1) & 1) ^ 1, abort_flag);
      if (!ok) break;
      constexpr int CH = DP / 8, STEP = 32 / CH;  // chunks per row, rows per instruction
      const int ch = lane % CH, live = min(it.rows - x * SLOT_ROWS, SLOT_ROWS), end = PaKind<ROWS>::NARROW ? (live + 15) & ~15 : (live + 31) & ~31;
      const uint32_t dst = sb::smem_u32(sQ + qs * SLOT_BYTES) + (ch >> 3) * (SLOT_ROWS * 128);
      // row -> (token, head) by steps, without a division per row
      const int row = it.rem + x * SLOT_ROWS + lane / CH, t0 = pa_div(p, row);
      int h = row - t0 * p.group;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (long)(it.row0 + t0) * p.q_tok +
                            (long)(it.hk * p.group + h) * p.q_head + ch * 8;
      const int dt = pa_div(p, STEP), dh = STEP - dt * p.group;
      const long go = dt * p.q_tok + dh * p.q_head, wrap = p.q_tok - p.group * p.q_head;
#pragma unroll 2
      for (int r = lane / CH; r < end; r += STEP) {
        const bool take = r < live && ch * 8 < p.D;
        pa_cp16(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4), take ? src : reinterpret_cast<const uint16_t*>(p.q), take);
        src += go;
        h += dh;
        if (h >= p.group) {
          h -= p.group;
          src += wrap;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      sb::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.q_full[qs]);
    }
    q_cnt += slots;
  }
  if (lane == 0) desc[0] = cur.refused ? -1 : starts && ok;
}

// K tiles, V tiles, or both in the order of the ring.
template <int ROWS, int PANELS, bool K, bool V>
__device__ __forceinline__ void pa_load(const PaParams& p, PaCtrl<PaCfg<PANELS>::STAGES>& c, uint8_t* sRing,
                                        const CUtensorMap* tmK, const CUtensorMap* tmV, int lane) {
  constexpr int STAGES = PaCfg<PANELS>::STAGES, TILE_BYTES = PaCfg<PANELS>::TILE_BYTES;
  volatile int* abort_flag = &c.abort;
  if (lane == 0) {
    if (K) sb::tma_prefetch_desc(tmK);
    if (V) sb::tma_prefetch_desc(tmV);
  }
  const int page = 1 << p.page_shift;
  const int box = min(page, PA_TILE), per_tile = PA_TILE / box;  // rows per copy, pages per tile
  const int bi = lane % per_tile, pn = lane / per_tile;          // this lane's page of the tile, and its panel
  const uint32_t dst = sb::smem_u32(sRing) + bi * (box >> 3) * p.group_step + pn * p.panel_step;
  uint32_t ring = 0;
  bool ok = true;
  for (int i = 0; ok; ++i) {
    const int slot = i % PA_ITEMS;
    if (!pa_wait(&c.item_full[slot], (i / PA_ITEMS) & 1, abort_flag)) break;
    const PaItem it = c.items[slot];
    __syncwarp();
    if (lane == 0) sb::mbar_arrive(&c.item_empty[slot]);
    if (it.count == 0) break;
    const int lead = pa_lead<ROWS>(it.rows);
    const int* trow = p.table + (long)it.seq * p.table_ld;
    int win[2] = {-64, -64}, where[2] = {0, 0};  // 32 pages at a time, for K and V: their first 8-row group in the tensor map
    auto load = [&](int t, int kv) -> bool {
      const int key0 = (it.tile0 + t) * PA_TILE, page0 = key0 >> p.page_shift;
      if (page0 + per_tile > win[kv] + 32) {
        win[kv] = page0;
        const int idx = page0 + lane;
        int at = kv ? p.v_outside : p.k_outside;  // a copy from outside the cache reads zeros
        if (idx < p.cols && ((idx + 1) << p.page_shift) > it.lo && (idx << p.page_shift) < it.hi) {
          const int got = trow[idx];
          if (got >= 0 && got < p.num_pages) at = got * (kv ? p.v_page8 : p.k_page8);
          else *p.status = SB_ERR_BAD_ARG;  // a visible page outside the cache: reported, its keys read as zeros
        }
        where[kv] = at;
      }
      const int first8 = __shfl_sync(0xffffffffu, where[kv], page0 - win[kv] + bi);
      const uint32_t e = ring + (kv ? pa_v_place(t, lead, it.count) : pa_k_place(t, lead)), st = e % STAGES;
      if (!pa_wait(&c.empty[st], ((e / STAGES) & 1) ^ 1, abort_flag)) return false;
      if (lane == 0) sb::mbar_expect_tx(&c.full[st], TILE_BYTES);
      __syncwarp();
      if (pn < p.boxes)
        pa_tma_5d(dst + st * TILE_BYTES, kv ? tmV : tmK, &c.full[st], pn * 64, first8 + ((key0 & (page - 1)) >> 3), it.hk);
      return true;
    };
    for (int t = -lead; t < it.count && ok; ++t) {
      if (V && t >= 0) ok = load(t, 1);
      if (K && ok && t + lead < it.count) ok = load(t + lead, 0);
    }
    ring += 2 * it.count;
  }
}

// Values behind the last visible key may be anything, NaN included, and 0 * NaN is NaN: row r of a V tile in shared memory
// becomes zeros.
template <int PANELS> __device__ __forceinline__ void pa_zero_v_row(const PaParams& p, uint8_t* tile, int r) {
  uint8_t* dst = tile + (r >> 3) * p.group_step + (r & 7) * 128;
#pragma unroll
  for (int c = 0; c < PANELS * 8; ++c)
    *reinterpret_cast<uint4*>(dst + (c >> 3) * p.panel_step + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
}

// Barriers, TMEM and the lengths of 32 sequences at a time (left where the scheduler puts the queries
// afterwards; with one such group the scheduler works it out alone).
// Returns false if shared memory does not start on a 1024-byte boundary, as the swizzled tiles need.
template <int ROWS, int STAGES>
__device__ __forceinline__ bool pa_begin(const PaParams& p, PaCtrl<STAGES>& c, uint8_t* smem, int warp, int lane) {
  constexpr int ISSUERS = PaKind<ROWS>::NARROW ? 1 : 2;  // warps that issue MMAs: each releases what the MMAs read
  if (sb::smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) {
      *p.status = SB_ERR_BAD_ARG;
      p.part_desc[8 * blockIdx.x] = 0;
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // as in pa_end
    return false;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      sb::mbar_init(&c.full[i], 1);
      sb::mbar_init(&c.empty[i], ISSUERS);
    }
    for (int i = 0; i < 2; ++i) {
      sb::mbar_init(&c.q_full[i], 1);
      sb::mbar_init(&c.q_empty[i], ISSUERS);
      sb::mbar_init(&c.vote[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      sb::mbar_init(&c.p_empty[i], 1);
      sb::mbar_init(&c.s_full[i], 1);
      sb::mbar_init(&c.p_full[i], 4);
    }
    for (int i = 0; i < 8; ++i) sb::mbar_init(&c.merge[i], 1);
    sb::mbar_init(&c.fin, 8);
    sb::mbar_init(&c.epi_done, 8);
    for (int i = 0; i < PA_ITEMS; ++i) {
      sb::mbar_init(&c.item_full[i], 1);
      sb::mbar_init(&c.item_empty[i], 11);  // loaders and MMA warps (three in all), eight softmax warps
    }
    c.abort = 0;
    sb::mbar_fence_init();
  }
  if (warp == 9) {
    sb::tmem_alloc(&c.tmem_slot, 512);
    sb::tmem_relinquish();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int* sums = reinterpret_cast<int*>(smem);
  const int chunks = (p.batch + 31) / 32;
  for (int k = chunks > 1 ? warp : chunks; k < chunks; k += PA_WARPS) {
    PaSeq s;
    const int t = pa_sum(pa_chunk_cost<ROWS>(p, k, lane, s));
    if (lane == 0) sums[k] = t;
  }
  sb::tc_fence_before();
  __syncthreads();
  sb::tc_fence_after();
  return true;
}
template <int STAGES> __device__ __forceinline__ void pa_end(const PaParams& p, PaCtrl<STAGES>& c, int warp) {
  __syncwarp();
  volatile int* abort_flag = &c.abort;
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies and MMAs in flight end
  }
  sb::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    sb::tc_fence_after();
    sb::tmem_dealloc(c.tmem_slot, 512);
  }
  // the narrow kernel may have started before the wide one ended: it does not end before it
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0 && *abort_flag) *p.status = SB_ERR_WAIT_TIMEOUT;
}

// ============================================================================ wide kernel
template <int PANELS, bool F16>
__global__ void __launch_bounds__(PA_THREADS, 1)
    pa_wide_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PaParams p) {
  using Cfg = PaCfg<PANELS>;
  constexpr int DP = Cfg::DP, TILE_BYTES = Cfg::TILE_BYTES, STAGES = Cfg::STAGES;
  constexpr uint32_t S_COL = 0, O_COL = 256;  // two S of 64 columns per group, two O of DP
  constexpr int FOLD = 2 * PA_FOLD;           // in half tiles
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;  // two slots of 128 rows
  uint8_t* sRing = smem + Cfg::FRONT;
  float2* xml = reinterpret_cast<float2*>(smem + Cfg::DATA);  // [group][row]
  PaCtrl<STAGES>& c = *reinterpret_cast<PaCtrl<STAGES>*>(smem + Cfg::DATA + 2048);
  volatile int* abort_flag = &c.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!pa_begin<PA_WIDE_ROWS>(p, c, smem, warp, lane)) return;
  const uint32_t tmem_base = c.tmem_slot;

  if (warp >= 8) {
    pa_regs_dec<PA_REGS_FEW>();  // one instruction for the whole warpgroup
    if (warp == 10) {
      pa_schedule<PA_WIDE_ROWS, PANELS>(p, c, sQ, (p.batch + 31) / 32, lane);
    } else if (warp == 8) {
      pa_load<PA_WIDE_ROWS, PANELS, true, true>(p, c, sRing, &tmK, &tmV, lane);
    } else if (lane == 0) {
      // MMAs of one group.  Half tiles of 64 keys: S(u) goes to buffer u & 1, P(u) overwrites its first 32 columns, and
      // S(u + 2) follows P(u) V in the same buffer while the softmax warps work on S(u + 1).
      const int x = warp == 11;
      const uint32_t idesc_s = sb::umma_idesc_f16(PA_TILE, PA_HALF, F16 ? 0 : 1, 0, 0);  // K-major both
      const uint32_t idesc_o = sb::umma_idesc_f16(PA_TILE, DP, F16 ? 0 : 1, 0, 1);       // V is MN-major
      const uint64_t q_desc = sb::umma_smem_desc(sb::smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = sb::umma_smem_desc(sb::smem_u32(sRing), 16, p.group_step);
      const uint64_t v_desc = sb::umma_smem_desc(sb::smem_u32(sRing), p.panel_step, p.group_step);
      const uint32_t k_panel = p.panel_step >> 4, half_step = (8 * p.group_step) >> 4, v_step = (2 * p.group_step) >> 4;
      const uint32_t s_col = tmem_base + S_COL + x * PA_TILE, o_col = tmem_base + O_COL + x * DP;
      uint32_t ring = 0, p_cnt0 = 0, p_cnt1 = 0;
      int q_cnt = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const int slot = i % PA_ITEMS;
        if (!pa_wait_lane(&c.item_full[slot], (i / PA_ITEMS) & 1, abort_flag)) break;
        const int count = c.items[slot].count, two_q = c.items[slot].rows > PA_TILE;
        sb::mbar_arrive(&c.item_empty[slot]);
        if (count == 0) break;
        // step u: with two_q tile u / 2 and its halves in turn, else tile u and half x.  Both groups take every tile in
        // the ring's order: the parity of a barrier that a warp has not followed phase by phase says nothing.
        const int lead = two_q ? 1 : 2, n = two_q ? 2 * count : count;
        const int qu = q_cnt + (two_q ? x : 0), qs = qu & 1;
        ok = pa_wait_lane(&c.q_full[qs], (qu >> 1) & 1, abort_flag);
        // ring places of the next K and V tile, as stage and parity
        uint32_t ks = ring % STAGES, kp = (ring / STAGES) & 1, ve = ring + pa_v_place(0, lead, count), vs = ve % STAGES,
                 vp = (ve / STAGES) & 1;
        auto advance = [](uint32_t& st, uint32_t& parity, uint32_t by) {
          st += by;
          if (st >= STAGES) {
            st -= STAGES;
            parity ^= 1;
          }
        };
        int kt = 0, vt = 0;
#pragma unroll 1
        for (int u = -2; u < n && ok; ++u) {
          const int b = u & 1, half = two_q ? b : x;
          const bool next = u + 2 < n;
          // All that this step needs is asked for together, because each answer takes some 180 cycles.  The first step on a
          // tile waits for its copy, the last one releases it.
          const bool opens = !two_q || b == 0, closes = !two_q || b, need_k = next && opens, need_v = u >= 0 && opens;
          const uint32_t pc = (b ? p_cnt1 : p_cnt0) & 1;
          const uint32_t got_k = need_k ? sb::mbar_try_wait(&c.full[ks], kp) : 1;
          const uint32_t got_v = need_v ? sb::mbar_try_wait(&c.full[vs], vp) : 1;
          const uint32_t got_p = u >= 0 ? sb::mbar_try_wait(&c.p_full[x * 2 + b], pc) : 1;
          if (!(got_k & got_v & got_p)) {
            if (need_v) ok = pa_wait_lane(&c.full[vs], vp, abort_flag);
            if (ok && need_k) ok = pa_wait_lane(&c.full[ks], kp, abort_flag);
            if (ok && u >= 0) ok = pa_wait_lane(&c.p_full[x * 2 + b], pc, abort_flag);
          }
          if (ok && u == 0 && i > 0) ok = pa_wait_lane(&c.epi_done, (i - 1) & 1, abort_flag);  // O of the item before is read
          if (!ok) break;
          sb::tc_fence_after();
          if (u >= 0) {
            const uint64_t vd = v_desc + vs * (TILE_BYTES >> 4) + half * half_step;
#pragma unroll
            for (int kk = 0; kk < PA_HALF / 16; ++kk)
              pa_umma_ts(o_col, s_col + b * PA_HALF + kk * 8, vd + kk * v_step, idesc_o, u % FOLD != 0 || kk != 0);
          }
          if (next) {
            const uint64_t qd = q_desc + qs * (TILE_BYTES >> 4), kd = k_desc + ks * (TILE_BYTES >> 4) + half * half_step;
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
              sb::umma_f16_ss(s_col + b * PA_HALF, qd + (kk >> 2) * (PA_PANEL >> 4) + (kk & 3) * 2,
                              kd + (kk >> 2) * k_panel + (kk & 3) * 2, idesc_s, kk != 0);
            sb::umma_commit(&c.s_full[x * 2 + b]);  // also says that P(u) V is complete
            if (u + 3 == n) {  // the slot's two releases come from both groups, or from the one that reads it
              sb::umma_commit(&c.q_empty[qs]);
              if (two_q) sb::umma_commit(&c.q_empty[qs]);
            }
            if (closes) {
              sb::umma_commit(&c.empty[ks]);
              advance(ks, kp, ++kt < lead ? 1 : 2);
            }
          } else {
            // the last two products of the item, no S after them: a barrier each, one phase per item
            sb::umma_commit(&c.p_empty[x * 2 + (u + 1 == n)]);
          }
          if (u >= 0) {
            if (b) ++p_cnt1; else ++p_cnt0;
            if (closes) {
              sb::umma_commit(&c.empty[vs]);
              advance(vs, vp, vt++ + lead < count ? 2 : 1);
            }
          }
        }
        ring += 2 * count;
        q_cnt += 1 + two_q;
      }
    }
  } else {
    pa_regs_inc<PA_REGS_MANY>();
    const int x = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t o_addr = t_lane + O_COL + x * DP;
    const float sl2 = p.sl2;
    uint32_t ring = 0, s_cnt0 = 0, s_cnt1 = 0, merges = 0;  // s_cnt: steps taken on each buffer
    // second place of this thread's row: the second partial slot, which no item but the CTA's last one writes, at its end
    float* const far = p.part_o + ((2L * blockIdx.x + 1) * p.part_rows + x * PA_TILE + r) * DP;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const int islot = i % PA_ITEMS;
      if (!pa_wait(&c.item_full[islot], (i / PA_ITEMS) & 1, abort_flag)) break;
      const PaItem it = c.items[islot];
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.item_empty[islot]);
      if (it.count == 0) break;
      const int rows = it.rows;
      const bool two_q = rows > PA_TILE;
      const int lead = two_q ? 1 : 2;
      const int row = two_q ? x * PA_TILE + r : r;          // row of the item
      const int warp_rows = rows - (row - lane);             // <= 0: no row of this warp exists
      const int tok = pa_div(p, it.rem + row), head = it.hk * p.group + (it.rem + row - tok * p.group);
      // visible keys of the row; lanes without a row see everything (their queries are zeros), so that they do not
      // send the warp through the masked path
      int lo = 0, hi = 0x7fffffff;
      if (row < rows) {
        const int pos = it.pos0 + tok;
        if (p.window >= 0) lo = max(0, pos - p.window);
        hi = p.causal ? min(pos + 1, it.L) : (p.window >= 0 ? (int)min((long)it.L, (long)pos + p.window + 1) : it.L);
      }
      float ref = -INFINITY, l = 0.f;
      float far_ref = -INFINITY, far_l = 0.f;  // what the sums of the second place refer to, and its row sum
      const int n = two_q ? 2 * it.count : it.count;  // half tiles of this group
      for (int u = 0; u < n; ++u) {
        const int t = two_q ? u >> 1 : u, b = u & 1, half = two_q ? b : x;
        const int key0 = (it.tile0 + t) * PA_TILE + half * PA_HALF;
        if (!pa_wait(&c.s_full[x * 2 + b], (b ? s_cnt1 : s_cnt0) & 1, abort_flag)) { ok = false; break; }
        if (b) ++s_cnt1; else ++s_cnt0;
        sb::tc_fence_after();
        const uint32_t s_addr = t_lane + S_COL + x * PA_TILE + b * PA_HALF;
        if (warp_rows > 0) {
          uint32_t s[PA_HALF];
#pragma unroll
          for (int ch = 0; ch < 2; ++ch) sb::tmem_ld32(s_addr + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(s + ch * 32));
          sb::tmem_ld_wait();
          if (!__all_sync(0xffffffffu, key0 >= lo && key0 + PA_HALF <= hi)) {
#pragma unroll
            for (int j = 0; j < PA_HALF; ++j)
              if (key0 + j < lo || key0 + j >= hi) s[j] = 0xff800000u;  // -inf, whatever the score was
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < PA_HALF; j += 2)
            m4[(j >> 1) & 3] = pa_max3(m4[(j >> 1) & 3], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
          const float mx = pa_max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]);
          const bool move = (mx - ref) * sl2 > 8.f || (ref == -INFINITY && mx > -INFINITY);
          const bool fold = u > 0 && u % FOLD == 0;
          if (fold || __any_sync(0xffffffffu, move)) {
            const float next = move ? mx : ref;
            const float alpha = move ? (ref == -INFINITY ? 0.f : pa_exp2((ref - next) * sl2)) : 1.f;
            ref = next;
            l *= alpha;
            if (u > 0) {
              // O holds the half tiles before, once their last product is complete: S(u + 1) follows it (and S(u) the one
              // before it); at the item's end it has a barrier of its own
              if (u + 1 < n ? !pa_wait(&c.s_full[x * 2 + (b ^ 1)], (b ? s_cnt0 : s_cnt1) & 1, abort_flag)
                            : !pa_wait(&c.p_empty[x * 2], i & 1, abort_flag)) { ok = false; break; }
              sb::tc_fence_after();
              const float beta = far_ref == -INFINITY ? 0.f : pa_exp2((far_ref - ref) * sl2);
#pragma unroll 1
              for (int ch = 0; ch < DP / 32; ++ch) {
                uint32_t o[32];
                sb::tmem_ld32(o_addr + ch * 32, o);
                sb::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                if (!fold) {
                  pa_tmem_st32(o_addr + ch * 32, o);
                } else {
#pragma unroll
                  for (int j = 0; j < 32; j += 4) {
                    float4* at = reinterpret_cast<float4*>(far + ch * 32 + j);
                    const float4 v = u > FOLD ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
                    *at = make_float4(fmaf(v.x, beta, __uint_as_float(o[j])), fmaf(v.y, beta, __uint_as_float(o[j + 1])),
                                      fmaf(v.z, beta, __uint_as_float(o[j + 2])), fmaf(v.w, beta, __uint_as_float(o[j + 3])));
                  }
                }
              }
              if (fold) {
                far_l = fmaf(far_l, beta, l);
                far_ref = ref;
                l = 0.f;
              }
            }
          }
          const float neg = ref == -INFINITY ? 0.f : -ref * sl2;
          const float2 scale2 = make_float2(sl2, sl2), neg2 = make_float2(neg, neg);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          uint32_t pk[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float2 z = pa_fma2(make_float2(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), scale2, neg2);
            const float2 e = make_float2(pa_exp2(z.x), pa_exp2(z.y));
            sum[j & 1] = pa_add2(sum[j & 1], e);
            pk[j] = pa_pack<F16>(e.x, e.y);
          }
          pa_tmem_st32(s_addr, pk);
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          sb::tmem_st_wait();
        }
        if (key0 + PA_HALF > it.hi) {  // rows of V behind the last visible key (by both groups with two_q, which does no harm)
          const uint32_t e = ring + pa_v_place(t, lead, it.count), st = e % STAGES;
          if (!pa_wait(&c.full[st], (e / STAGES) & 1, abort_flag)) { ok = false; break; }
          if (r < PA_HALF && key0 + r >= it.hi) pa_zero_v_row<PANELS>(p, sRing + st * TILE_BYTES, half * PA_HALF + r);
          sb::fence_proxy_async_smem();
        }
        sb::tc_fence_before();
        __syncwarp();
        if (lane == 0) sb::mbar_arrive(&c.p_full[x * 2 + b]);
      }
      ring += 2 * it.count;
      if (!ok) break;
      if (!pa_wait(&c.p_empty[x * 2 + 1], i & 1, abort_flag)) break;  // the last product
      sb::tc_fence_after();
      if (n > FOLD && warp_rows > 0) {  // back from the second place
        const float beta = far_ref == -INFINITY ? 0.f : pa_exp2((far_ref - ref) * sl2);
        l = fmaf(far_l, beta, l);
#pragma unroll 1
        for (int ch = 0; ch < DP / 32; ++ch) {
          uint32_t o[32];
          sb::tmem_ld32(o_addr + ch * 32, o);
          sb::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(far + ch * 32 + j);
            o[j] = __float_as_uint(fmaf(v.x, beta, __uint_as_float(o[j])));
            o[j + 1] = __float_as_uint(fmaf(v.y, beta, __uint_as_float(o[j + 1])));
            o[j + 2] = __float_as_uint(fmaf(v.z, beta, __uint_as_float(o[j + 2])));
            o[j + 3] = __float_as_uint(fmaf(v.w, beta, __uint_as_float(o[j + 3])));
          }
          pa_tmem_st32(o_addr + ch * 32, o);
        }
        sb::tmem_st_wait();
      }
      // the two states of a row: fa, fb scale the groups' outputs to a common reference
      float fa = x == 0 ? 1.f : 0.f, fb = 1.f - fa;
      int c0 = 0, c1 = DP / 32;
      if (!two_q) {
        if (i > 0 && !pa_wait(&c.epi_done, (i - 1) & 1, abort_flag)) break;  // xml of the item before is read
        xml[x * PA_TILE + r] = make_float2(ref, l);
        sb::tc_fence_before();
        __syncwarp();
        if (lane == 0) sb::mbar_arrive(&c.merge[x * 4 + quad]);
        if (!pa_wait(&c.merge[(x ^ 1) * 4 + quad], merges & 1, abort_flag)) break;
        ++merges;
        sb::tc_fence_after();
        const float2 a = xml[r], b = xml[PA_TILE + r];
        const float top = fmaxf(a.x, b.x);
        fa = a.x == -INFINITY ? 0.f : pa_exp2((a.x - top) * sl2);
        fb = b.x == -INFINITY ? 0.f : pa_exp2((b.x - top) * sl2);
        ref = top;
        l = a.y * fa + b.y * fb;
        c0 = x * (DP / 64);
        c1 = c0 + DP / 64;
      }
      if (warp_rows > 0) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // no visible key: zeros; NaN stays
        const float ga = it.slot < 0 ? fa * inv : fa, gb = it.slot < 0 ? fb * inv : fb;
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (long)(it.row0 + tok) * p.o_tok + (long)head * p.o_head;
        const long prow = (long)it.slot * p.part_rows + row;
        for (int ch = c0; ch < c1; ++ch) {
          uint32_t a[32], b[32];
          float o[32];
          if (!two_q) {
            sb::tmem_ld32(t_lane + O_COL + ch * 32, a);
            sb::tmem_ld32(t_lane + O_COL + DP + ch * 32, b);
            sb::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = fmaf(__uint_as_float(a[j]), ga, __uint_as_float(b[j]) * gb);
          } else {
            sb::tmem_ld32(o_addr + ch * 32, a);
            sb::tmem_ld_wait();
            const float f = x ? gb : ga;
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __uint_as_float(a[j]) * f;
          }
          if (row >= rows) {
          } else if (it.slot < 0) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              if (ch * 32 + j < p.D) {
                uint4 u;
                u.x = pa_pack<F16>(o[j], o[j + 1]);
                u.y = pa_pack<F16>(o[j + 2], o[j + 3]);
                u.z = pa_pack<F16>(o[j + 4], o[j + 5]);
                u.w = pa_pack<F16>(o[j + 6], o[j + 7]);
                *reinterpret_cast<uint4*>(dst + ch * 32 + j) = u;
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(p.part_o + prow * DP + ch * 32 + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
          __syncwarp();
        }
        if (it.slot >= 0 && row < rows && (two_q || x == 0))
          p.part_ml[prow] = make_float2(ref == -INFINITY ? -INFINITY : ref * sl2, l);
      }
      sb::tc_fence_before();
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.epi_done);
    }
  }
  pa_end(p, c, warp);
}

// ============================================================================ narrow kernel
// v[j] of all lanes joined by f: lanes r and r + 16 end with the result of j = r.
template <typename F> __device__ __forceinline__ float pa_transpose_reduce(float (&v)[16], int lane, F f) {
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = f(v[j], __shfl_xor_sync(0xffffffffu, v[j], 16));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int j = 0; j < o; ++j) {
      const bool up = lane & o;
      const float send = up ? v[j] : v[j + o], keep = up ? v[j + o] : v[j];
      v[j] = f(keep, __shfl_xor_sync(0xffffffffu, send, o));
    }
  return v[0];
}

// All loops over the rows go by blocks of 16 and are not unrolled further: code that does not fit the instruction caches
// costs more than the work here (unrolled over 64 rows the long decode above took 59 us, now 42).  So what a
// thread keeps of the rows between tiles has to be little: row r is kept by lane r % 32 of every warp.
template <int PANELS, bool F16>
__global__ void __launch_bounds__(PA_THREADS, 1)
    pa_narrow_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PaParams p) {
  using Cfg = PaCfg<PANELS>;
  constexpr int DP = Cfg::DP, TILE_BYTES = Cfg::TILE_BYTES, STAGES = Cfg::STAGES;
  constexpr int R = PA_NARROW_ROWS, Q_SLOT = PANELS * R * 128, P_BYTES = PA_TILE * 128;
  constexpr uint32_t S_COL = 0, O_COL = 256, FAR_COL = 384;  // four S^T, two O^T and their second places, of 64 columns
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                    // two slots of 64 rows
  uint8_t* sP = smem + 2 * 16384;        // [group][key][64 rows], 128-byte swizzle
  uint8_t* sRing = smem + Cfg::FRONT;
  float* sRef = reinterpret_cast<float*>(smem + Cfg::DATA);  // [group][old / new][row]: -reference, +inf where unset
  PaCtrl<STAGES>& c = *reinterpret_cast<PaCtrl<STAGES>*>(smem + Cfg::DATA + 2048);
  volatile int* abort_flag = &c.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!pa_begin<R>(p, c, smem, warp, lane)) return;
  const uint32_t tmem_base = c.tmem_slot;

  if (warp == 10) {
    pa_schedule<R, PANELS>(p, c, sQ, (p.batch + 31) / 32, lane);
  } else if (warp == 8) {
    pa_load<R, PANELS, true, false>(p, c, sRing, &tmK, &tmV, lane);
  } else if (warp == 11) {
    pa_load<R, PANELS, false, true>(p, c, sRing, &tmK, &tmV, lane);
    if (p.zero_tail) {  // rows before the first and behind the last sequence
      const int before = p.batch > 0 ? min(max(p.cu[0], 0), p.T) : 0, heads = p.Hkv * p.group;
      const int gap = p.batch > 0 ? max(min(p.cu[p.batch], p.T), before) - before : 0, per_row = p.D / 8;
      for (int at = blockIdx.x; at < (p.T - gap) * heads; at += gridDim.x) {
        const int row = at < before * heads ? at : at + gap * heads, t = row / heads;
        if (lane < per_row)
          *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + (long)t * p.o_tok + (long)(row - t * heads) * p.o_head + lane * 8) =
              make_uint4(0, 0, 0, 0);
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      const uint64_t q_desc = sb::umma_smem_desc(sb::smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = sb::umma_smem_desc(sb::smem_u32(sRing), 16, p.group_step);
      // V^T: 128 rows of the product are the columns of the tile; with a head size up to 64 the second half of them reads
      // the next rows of the tile and goes to lanes that nobody looks at
      const uint64_t v_desc = sb::umma_smem_desc(sb::smem_u32(sRing), PANELS == 2 ? p.panel_step : 1024, p.group_step);
      const uint64_t p_desc = sb::umma_smem_desc(sb::smem_u32(sP), 1024, 1024);
      const uint32_t k_panel = p.panel_step >> 4, v_step = (2 * p.group_step) >> 4;
      uint32_t ring = 0, p_cnt0 = 0, p_cnt1 = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const int slot = i % PA_ITEMS;
        if (!pa_wait_lane(&c.item_full[slot], (i / PA_ITEMS) & 1, abort_flag)) break;
        const int n = c.items[slot].count, cols = (c.items[slot].rows + 15) & ~15;
        sb::mbar_arrive(&c.item_empty[slot]);
        if (n == 0) break;
        const uint32_t idesc_s = sb::umma_idesc_f16(PA_TILE, cols, F16 ? 0 : 1, 0, 0);
        const uint32_t idesc_o = sb::umma_idesc_f16(PA_TILE, cols, F16 ? 0 : 1, 1, 1);
        const int qs = i & 1;
        ok = pa_wait_lane(&c.q_full[qs], (i >> 1) & 1, abort_flag);
        auto issue_s = [&](int t) -> bool {
          const uint32_t e = ring + pa_k_place(t, 4), st = e % STAGES;
          if (!pa_wait_lane(&c.full[st], (e / STAGES) & 1, abort_flag)) return false;
          sb::tc_fence_after();
          const uint64_t qd = q_desc + qs * (Q_SLOT >> 4), kd = k_desc + st * (TILE_BYTES >> 4);
          const int buf = (t & 1) * 2 + ((t >> 1) & 1);
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            sb::umma_f16_ss(tmem_base + S_COL + buf * R, kd + (kk >> 2) * k_panel + (kk & 3) * 2,
                            qd + (kk >> 2) * (R * 128 >> 4) + (kk & 3) * 2, idesc_s, kk != 0);
          sb::umma_commit(&c.s_full[buf]);
          sb::umma_commit(&c.empty[st]);
          if (t == n - 1) sb::umma_commit(&c.q_empty[qs]);
          return true;
        };
#pragma unroll 1
        for (int t = -4; t < n && ok; ++t) {
          if (t >= 0) {
            const int x = t & 1;
            const uint32_t e = ring + pa_v_place(t, 4, n), st = e % STAGES;
            ok = pa_wait_lane(&c.full[st], (e / STAGES) & 1, abort_flag);
            if (ok && t == 0 && i > 0) ok = pa_wait_lane(&c.epi_done, (i - 1) & 1, abort_flag);  // O of the item before is read
            ok = ok && pa_wait_lane(&c.p_full[x], (x ? p_cnt1 : p_cnt0) & 1, abort_flag);
            if (!ok) break;
            if (x) ++p_cnt1; else ++p_cnt0;
            sb::tc_fence_after();
            const uint64_t vd = v_desc + st * (TILE_BYTES >> 4), pd = p_desc + x * (P_BYTES >> 4);
#pragma unroll
            for (int kk = 0; kk < PA_TILE / 16; ++kk)
              sb::umma_f16_ss(tmem_base + O_COL + x * R, vd + kk * v_step, pd + kk * (2048 >> 4), idesc_o,
                              (t >> 1) % PA_FOLD != 0 || kk != 0);
            sb::umma_commit(&c.empty[st]);
            sb::umma_commit(&c.p_empty[x]);
          }
          if (t + 4 < n) ok = issue_s(t + 4);
        }
        ring += 2 * n;
      }
    }
  } else {
    const int x = warp >> 2, quad = warp & 3, key = quad * 32 + lane;  // thread = key of the tile, later a column of V
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const float sl2 = p.sl2;
    float* wmax = reinterpret_cast<float*>(sP + x * P_BYTES);  // [warp of the group][64], where P is not in use
    uint8_t* prow = sP + x * P_BYTES + key * 128;
    uint32_t ring = 0, s_cnt0 = 0, s_cnt1 = 0, issued = 0, retired = 0, votes = 0;
    bool ok = true;
    // all four warps of the group have come here
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.vote[x]);
      return pa_wait(&c.vote[x], votes++ & 1, abort_flag);
    };
    for (int i = 0; ok; ++i) {
      const int islot = i % PA_ITEMS;
      if (!pa_wait(&c.item_full[islot], (i / PA_ITEMS) & 1, abort_flag)) break;
      const PaItem it = c.items[islot];
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.item_empty[islot]);
      if (it.count == 0) break;
      if (i > 0 && !pa_wait(&c.epi_done, (i - 1) & 1, abort_flag)) break;  // sRef of the item before is read
      const int nb = (it.rows + 15) >> 4, n = it.count;
      // keys that every row sees: tiles inside need no mask
      const int pos1 = it.pos0 + pa_div(p, it.rem + it.rows - 1);
      const int lo_all = p.window >= 0 ? max(0, pos1 - p.window) : 0;
      const int hi_all = p.causal ? min(it.pos0 + 1, it.L)
                                  : (p.window >= 0 ? (int)min((long)it.L, (long)it.pos0 + p.window + 1) : it.L);
      int cur = 0;
      float* ref = sRef + x * 2 * R;
      // row sums: of the first 16 rows per key in every thread, of the others over the warp's keys in lane row % 32; far0 and
      // far1 take all of them from time to time
      float l[16], l0 = 0.f, l1 = 0.f, far0 = 0.f, far1 = 0.f;
#pragma unroll
      for (int u = 0; u < 16; ++u) l[u] = 0.f;
      for (int t = x; t < n; t += 2) {
        const int key0 = (it.tile0 + t) * PA_TILE, buf = (t >> 1) & 1;
        if (retired < issued) {  // P V of this group's tile before: P may be overwritten, O rescaled
          if (!pa_wait(&c.p_empty[x], retired & 1, abort_flag)) { ok = false; break; }
          ++retired;
        }
        if (!pa_wait(&c.s_full[x * 2 + buf], (buf ? s_cnt1 : s_cnt0) & 1, abort_flag)) { ok = false; break; }
        if (buf) ++s_cnt1; else ++s_cnt0;
        sb::tc_fence_after();
        const uint32_t s_addr = t_lane + S_COL + (x * 2 + buf) * R;
        const bool inside = key0 >= lo_all && key0 + PA_TILE <= hi_all;
        // scores of a block of 16 rows, -inf where a row does not see the thread's key
        auto scores = [&](int b, float (&s)[16]) {
          sb::tmem_ld16(s_addr + b * 16, reinterpret_cast<uint32_t(&)[16]>(s));
          sb::tmem_ld_wait();
          if (!inside) {
            const int j = key0 + key, tok = pa_div(p, it.rem + b * 16);
            int pos = it.pos0 + tok, h = it.rem + b * 16 - tok * p.group;
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              const int lo = p.window >= 0 ? pos - p.window : 0;
              const int hi = p.causal ? min(pos + 1, it.L)
                                      : (p.window >= 0 ? (int)min((long)it.L, (long)pos + p.window + 1) : it.L);
              if (b * 16 + u < it.rows && (j < lo || j >= hi)) s[u] = -INFINITY;
              if (++h == p.group) {
                h = 0;
                ++pos;
              }
            }
          }
        };
        // P of the tile against the current references and its row sums; returns the largest exponent
        float t0 = 0.f, t1 = 0.f, first[16];
        auto probabilities = [&]() -> float {
          float top = -INFINITY;
#pragma unroll 1
          for (int b = 0; b < nb; ++b) {
            float s[16];
            scores(b, s);
            uint32_t pk[8];
#pragma unroll
            for (int u = 0; u < 16; u += 4) {
              const float4 f = *reinterpret_cast<const float4*>(ref + cur * R + b * 16 + u);
              const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                float z = fmaf(s[u + k], sl2, fs[k]);
                if (!inside && s[u + k] == -INFINITY) z = -INFINITY;  // also where the reference is unset
                top = fmaxf(top, z);
                s[u + k] = pa_exp2(z);
              }
              pk[u / 2] = pa_pack<F16>(s[u], s[u + 1]);
              pk[u / 2 + 1] = pa_pack<F16>(s[u + 2], s[u + 3]);
            }
            *reinterpret_cast<uint4*>(prow + (((b * 2) ^ (key & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            *reinterpret_cast<uint4*>(prow + (((b * 2 + 1) ^ (key & 7)) << 4)) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
            if (b == 0) {
#pragma unroll
              for (int u = 0; u < 16; ++u) first[u] = s[u];
            } else {
              const float sum = pa_transpose_reduce(s, lane, [](float a, float b) { return a + b; });
              if (lane >> 4 == (b & 1)) {
                if (b < 2) t0 = sum; else t1 = sum;
              }
            }
          }
          return top;
        };
        const bool fold = t >= 2 && (t >> 1) % PA_FOLD == 0;
        bool need = t < 2 || fold;  // no reference yet, or another place for the sums
        if (!need) {
          const int mine = __any_sync(0xffffffffu, probabilities() > 8.f);
          int* flags = c.need[x][votes & 1];
          if (lane == 0) flags[quad] = mine;
          if (!meet()) { ok = false; break; }
          const int4 all = *reinterpret_cast<const int4*>(flags);
          need = (all.x | all.y | all.z | all.w) != 0;
        }
        if (need) {
#pragma unroll 1
          for (int b = 0; b < nb; ++b) {  // maxima over the warp's keys
            float s[16];
            scores(b, s);
            const float m = pa_transpose_reduce(s, lane, [](float a, float b) { return fmaxf(a, b); });
            if (lane < 16) wmax[quad * R + b * 16 + lane] = m;
          }
          if (!meet()) { ok = false; break; }
          float alpha[2];  // of rows lane and lane + 32; every warp works them out
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = h * 32 + lane;
            float m = wmax[row];
#pragma unroll
            for (int w = 1; w < 4; ++w) m = fmaxf(m, wmax[w * R + row]);
            const float old = t < 2 ? INFINITY : ref[cur * R + row];
            const float next = m == -INFINITY ? old : fminf(old, -m * sl2);
            alpha[h] = old == INFINITY ? 0.f : pa_exp2(next - old);
            if (row < nb * 16) ref[(cur ^ 1) * R + row] = next;
          }
          cur ^= 1;
          l0 *= alpha[0];
          l1 *= alpha[1];
          far0 *= alpha[0];
          far1 *= alpha[1];
#pragma unroll
          for (int u = 0; u < 16; ++u) l[u] *= __shfl_sync(0xffffffffu, alpha[0], u);
          if (t >= 2) {
            const int folds = (t >> 1) / PA_FOLD;  // with this one
#pragma unroll 1
            for (int b = 0; b < nb; ++b) {
              float o[16], f[16], a[16];
              sb::tmem_ld16(t_lane + O_COL + x * R + b * 16, reinterpret_cast<uint32_t(&)[16]>(o));
              sb::tmem_ld16(t_lane + FAR_COL + x * R + b * 16, reinterpret_cast<uint32_t(&)[16]>(f));
              sb::tmem_ld_wait();
#pragma unroll
              for (int u = 0; u < 16; ++u) {
                a[u] = __shfl_sync(0xffffffffu, b < 2 ? alpha[0] : alpha[1], (b & 1) * 16 + u);
                o[u] *= a[u];
              }
              if (!fold) pa_tmem_st16(t_lane + O_COL + x * R + b * 16, reinterpret_cast<uint32_t*>(o));
              if (folds > 0) {
#pragma unroll
                for (int u = 0; u < 16; ++u) f[u] = (folds > fold ? f[u] * a[u] : 0.f) + (fold ? o[u] : 0.f);
                pa_tmem_st16(t_lane + FAR_COL + x * R + b * 16, reinterpret_cast<uint32_t*>(f));
              }
            }
            sb::tmem_st_wait();
            if (fold) {
              const float sum16 = pa_transpose_reduce(l, lane, [](float a, float b) { return a + b; });
              far0 += lane < 16 ? sum16 : l0;
              far1 += l1;
              l0 = l1 = 0.f;
#pragma unroll
              for (int u = 0; u < 16; ++u) l[u] = 0.f;
            }
          }
          if (!meet()) { ok = false; break; }  // every warp has read the maxima: P goes to the same place
          probabilities();
        }
        l0 += t0;
        l1 += t1;
#pragma unroll
        for (int u = 0; u < 16; ++u) l[u] += first[u];
        if (key0 + PA_TILE > it.hi) {
          const uint32_t e = ring + pa_v_place(t, 4, n), st = e % STAGES;
          if (!pa_wait(&c.full[st], (e / STAGES) & 1, abort_flag)) { ok = false; break; }
          if (key0 + key >= it.hi) pa_zero_v_row<PANELS>(p, sRing + st * TILE_BYTES, key);
        }
        sb::fence_proxy_async_smem();
        sb::tc_fence_before();
        __syncwarp();
        if (lane == 0) sb::mbar_arrive(&c.p_full[x]);
        ++issued;
      }
      ring += 2 * n;
      if (!ok) break;
      if (retired < issued) {
        if (!pa_wait(&c.p_empty[x], retired & 1, abort_flag)) break;
        ++retired;
      }
      const float sum16 = pa_transpose_reduce(l, lane, [](float a, float b) { return a + b; });
      if (lane < 16) l0 = sum16;
      if (n - x > 2 * PA_FOLD) {  // back from the second place
        l0 += far0;
        l1 += far1;
        sb::tc_fence_after();
#pragma unroll 1
        for (int b = 0; b < nb; ++b) {
          float o[16], f[16];
          sb::tmem_ld16(t_lane + O_COL + x * R + b * 16, reinterpret_cast<uint32_t(&)[16]>(o));
          sb::tmem_ld16(t_lane + FAR_COL + x * R + b * 16, reinterpret_cast<uint32_t(&)[16]>(f));
          sb::tmem_ld_wait();
#pragma unroll
          for (int u = 0; u < 16; ++u) o[u] += f[u];
          pa_tmem_st16(t_lane + O_COL + x * R + b * 16, reinterpret_cast<uint32_t*>(o));
        }
        sb::tmem_st_wait();
        sb::tc_fence_before();
      }
      wmax[quad * R + lane] = l0;  // P of this group is not in use: its place takes the warps' sums
      wmax[quad * R + 32 + lane] = l1;
      if (quad == 0 && lane == 0) c.need[x][0][0] = cur;  // no vote is under way
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.fin);
      if (!pa_wait(&c.fin, i & 1, abort_flag)) break;
      sb::tc_fence_after();
      // Both groups' states are joined: group x writes rows x * 8 nb .. (x + 1) * 8 nb, thread = column of the head.
      // Lane r works out the factors of row first + r, so that their chain of loads and exponentials is waited for once.
      const int first = x * nb * 8, mine = min(first + lane, R - 1);
      float g0, g1;
      {
        const float* sum0 = reinterpret_cast<const float*>(sP);
        const float* sum1 = reinterpret_cast<const float*>(sP + P_BYTES);
        const float r0 = sRef[c.need[0][0][0] * R + mine];
        const float r1 = n > 1 ? sRef[(2 + c.need[1][0][0]) * R + mine] : INFINITY;
        const float a0 = (sum0[mine] + sum0[R + mine]) + (sum0[2 * R + mine] + sum0[3 * R + mine]);
        const float a1 = (sum1[mine] + sum1[R + mine]) + (sum1[2 * R + mine] + sum1[3 * R + mine]);
        const float top = fminf(r0, r1);
        g0 = r0 == INFINITY ? 0.f : pa_exp2(top - r0);
        g1 = r1 == INFINITY ? 0.f : pa_exp2(top - r1);
        const float sum = a0 * g0 + a1 * g1;  // without a reference: 0, or NaN if every score was
        if (it.slot < 0) {
          const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // no visible key: zeros; NaN stays
          g0 *= inv;
          g1 *= inv;
        } else if (quad == 0 && lane < nb * 8 && mine < it.rows) {
          p.part_ml[(long)it.slot * p.part_rows + mine] = make_float2(-top, sum);
        }
      }
      const int d = key;
      const bool whole = it.slot < 0, store = whole ? d < p.D : d < DP;
      int row = first, tok = pa_div(p, it.rem + row), h = it.rem + row - tok * p.group;
      long at = whole ? (long)(it.row0 + tok) * p.o_tok + (long)(it.hk * p.group + h) * p.o_head + d
                      : ((long)it.slot * p.part_rows + row) * DP + d;
      const long go = whole ? p.o_head : DP, wrap = whole ? p.o_tok - p.group * p.o_head : 0;
#pragma unroll 1
      for (int j0 = 0; j0 < nb * 8 && row < it.rows; j0 += 8) {
        uint32_t o0[8], o1[8] = {};
        pa_tmem_ld8(t_lane + O_COL + row, o0, 0);
        if (n > 1) pa_tmem_ld8(t_lane + O_COL + R + row, o1, 0);
        sb::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j, ++row) {
          const float ga = __shfl_sync(0xffffffffu, g0, j0 + j), gb = __shfl_sync(0xffffffffu, g1, j0 + j);
          const float v = fmaf(__uint_as_float(o0[j]), ga, __uint_as_float(o1[j]) * gb);
          if (row < it.rows && store) {
            if (whole) reinterpret_cast<uint16_t*>(p.out)[at] = (uint16_t)pa_pack<F16>(v, 0.f);
            else p.part_o[at] = v;
          }
          at += go;
          if (++h == p.group) {
            h = 0;
            at += wrap;
          }
        }
      }
      sb::tc_fence_before();
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&c.epi_done);
    }
  }
  pa_end(p, c, warp);
}

// ============================================================================ joining the partial results
// Zeros for the sequences of a kernel that refused the call's work: nothing else writes there, and the memory may hold
// older tensors.  Called from the last kernel, as a function: inside the kernels that refuse, the code took 5 % of a decoding
// step's time although it does not run (147 -> 154 us), inlined in the last one 1 us.
template <int ROWS> __device__ __noinline__ void pa_zero_refused(const PaParams& p) {
  const int per_head = p.D / 8, per_token = p.Hkv * p.group * per_head;
  for (int b = 0; b < p.batch; ++b) {
    const PaSeq s = pa_seq(p, b);
    if (pa_items<ROWS>(p, s.n) == 0) continue;
    for (int t = blockIdx.x; t < s.n; t += gridDim.x)
      for (int i = threadIdx.x; i < per_token; i += PA_COMBINE_THREADS) {
        const int h = i / per_head;
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + (long)(s.row0 + t) * p.o_tok + (long)h * p.o_head +
                                  (i - h * per_head) * 8) = make_uint4(0, 0, 0, 0);
      }
  }
}

// A task is a block of rows of an item that several CTAs worked on: PG rows (8, or 16 where a head has up to 64 columns) with a
// thread per four columns, or, with PG parts and more, one row whose parts are dealt to PG groups of threads that are joined in
// order.  Every block lists the tasks (one descriptor per CTA) and takes every gridDim-th, so the launch is one wave whatever the
// items are.
template <int PANELS, bool F16>
__global__ void __launch_bounds__(PA_COMBINE_THREADS, 4)
    pa_combine_kernel(const __grid_constant__ PaParams pn, const __grid_constant__ PaParams pw, int narrow_ctas, int ctas) {
  constexpr int DP = PANELS * 64, QUADS = DP / 4, PG = PA_COMBINE_THREADS / QUADS, WARPS = PA_COMBINE_THREADS / 32;
  __shared__ float4 so[PG][QUADS];
  __shared__ float2 sml[PG];
  __shared__ int swarp[WARPS];
  __shared__ int stask[3], srefused[2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int quad = threadIdx.x % QUADS, pg = threadIdx.x / QUADS;
  int before = 0;  // tasks of the descriptors before `base`
  for (int base = 0; base < ctas; base += PA_COMBINE_THREADS) {
    const int mine = base + threadIdx.x;
    int tasks = 0;
    if (mine < ctas) {
      const int local = mine < narrow_ctas ? mine : mine - narrow_ctas;
      const int* desc = (mine < narrow_ctas ? pn : pw).part_desc + 8 * local;
      const int head = desc[0];
      if (mine == 0) srefused[0] = head < 0;
      if (mine == narrow_ctas) srefused[1] = head < 0;
      if (head > 0) tasks = desc[5] - local < PG ? (desc[4] + PG - 1) / PG : desc[4];
    }
    const int inc = pa_scan(tasks, lane);
    __syncthreads();
    if (lane == 31) swarp[warp] = inc;
    __syncthreads();
    int lo = before + inc - tasks, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) lo += swarp[w];
      all += swarp[w];
    }
    // tasks of this block inside [before, before + all)
    int task = (int)blockIdx.x + (before > (int)blockIdx.x ? (before - (int)blockIdx.x + gridDim.x - 1) / gridDim.x * gridDim.x : 0);
    for (; task < before + all; task += gridDim.x) {
      __syncthreads();
      if (task >= lo && task < lo + tasks) {
        stask[0] = mine;
        stask[1] = task - lo;
      }
      __syncthreads();
      const bool wide = stask[0] >= narrow_ctas;
      const int cta = wide ? stask[0] - narrow_ctas : stask[0], block = stask[1];
      const PaParams& p = wide ? pw : pn;
      const int* desc = p.part_desc + 8 * cta;
      const int row0 = desc[1], rem = desc[2], hk = desc[3], rows = desc[4], last = desc[5];
      const bool few = last - cta < PG;
      const int row = few ? block * PG + pg : block, step = few ? 1 : PG;
      float ref = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows) {
#pragma unroll 4
        for (int c = few ? cta : cta + pg; c <= last; c += step) {
          const long prow = (long)(2 * c + (c == cta ? 1 : 0)) * p.part_rows + row;
          const float2 ml = p.part_ml[prow];
          const float4 v = *reinterpret_cast<const float4*>(p.part_o + prow * DP + quad * 4);
          if (ml.x == -INFINITY && ml.y == 0.f) continue;  // a part without a visible key
          const float next = fmaxf(ref, ml.x);
          const float a = ref == -INFINITY ? 0.f : exp2f(ref - next), b = exp2f(ml.x - next);
          l = l * a + ml.y * b;
          o.x = o.x * a + v.x * b; o.y = o.y * a + v.y * b; o.z = o.z * a + v.z * b; o.w = o.w * a + v.w * b;
          ref = next;
        }
      }
      if (!few) {
        so[pg][quad] = o;
        if (quad == 0) sml[pg] = make_float2(ref, l);
        __syncthreads();
        if (pg > 0) continue;
        ref = -INFINITY;
#pragma unroll
        for (int g = 0; g < PG; ++g) ref = fmaxf(ref, sml[g].x);
        l = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < PG; ++g) {
          const float2 ml = sml[g];
          if (ml.x == -INFINITY && ml.y == 0.f) continue;
          const float f = exp2f(ml.x - ref);
          const float4 v = so[g][quad];
          l += ml.y * f;
          o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
        }
      }
      if (row < rows && quad * 4 < p.D) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const int tok = pa_div(p, rem + row), head = hk * p.group + (rem + row - tok * p.group);
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (long)(row0 + tok) * p.o_tok + (long)head * p.o_head + quad * 4;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pa_pack<F16>(o.x * inv, o.y * inv), pa_pack<F16>(o.z * inv, o.w * inv));
      }
    }
    before += all;
  }
  if (srefused[0]) pa_zero_refused<PA_NARROW_ROWS>(pn);
  if (ctas > narrow_ctas && srefused[1]) pa_zero_refused<PA_WIDE_ROWS>(pw);
}

typedef CUresult (*PaEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
PaEncodeFn pa_encode() {
  static PaEncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult st;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &st) != cudaSuccess) f = nullptr;
    return (PaEncodeFn)f;
  }();
  return fn;
}
// A cache seen as [head][8-row group][64-column panel][row of the group][column]: one copy brings the panels of up to 128
// rows of a page as the 1024-byte blocks that the matrix descriptors step over.  With a head size that is no multiple of
// 64 there is one panel dimension of true width, so that columns beyond the head read zeros.
int pa_tmap(CUtensorMap* m, const void* base, int D, int heads, int page_size, int pages, long page, long row, long head,
            bool f16, bool joined, int* page8, int* outside) {
  if (!pa_encode()) return SB_ERR_DRIVER;
  if (row <= 0 || (pages > 1 && page % (8 * row))) return SB_ERR_BAD_ARG;
  const long step = pages == 1 ? page_size / 8 : page / (8 * row), groups = (pages - 1) * step + page_size / 8;
  if (step < 0 || groups > (1L << 30)) return SB_ERR_TOO_LARGE;
  *page8 = (int)step;
  *outside = (int)groups;
  cuuint64_t dims[5] = {(cuuint64_t)(joined ? 64 : D), 8, (cuuint64_t)(joined ? 2 : 1), (cuuint64_t)groups, (cuuint64_t)heads};
  cuuint64_t strides[4] = {(cuuint64_t)row * 2, 128, (cuuint64_t)row * 16, (cuuint64_t)head * 2};
  cuuint32_t box[5] = {64, 8, (cuuint32_t)(joined ? 2 : 1), (cuuint32_t)((page_size < PA_TILE ? page_size : PA_TILE) / 8), 1};
  cuuint32_t es[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      pa_encode()(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base),
                  dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? SB_OK : SB_ERR_DRIVER;
}

// CTAs of a launch: one per SM, fewer when not even the table's full length gives each of them two key tiles
long pa_ctas(long T, int batch, int Hq, int Hkv, long cap, int item_rows, bool whole, int sms) {
  const long items = (T * (Hq / Hkv) + item_rows - 1) / item_rows + batch;
  const long tiles = (cap + PA_TILE - 1) / PA_TILE + 1;
  const long want = whole ? items * Hkv : (items * Hkv * tiles + 1) / 2;
  return want < 1 ? 1 : want < sms ? want : sms;
}
long pa_align(long v) { return (v + 255) & ~255L; }

// Which kernels a call takes, and their places in its workspace.  Sequences with at most 64 rows (new tokens x heads per KV
// head) are narrow; with no more new tokens than sequences, as in a decoding step, all of them are, whatever their length:
// the wide launch would find nothing and cost its 3 us, and a sequence that does have more rows is read once per 64 of them.
struct PaPlan {
  bool wide, whole;
  int narrow_max, narrow_rows, narrow_ctas, wide_ctas, sms;
  long narrow_at, wide_at, bytes;
};
PaPlan pa_plan(long T, int batch, int Hq, int Hkv, int D, long cap, int sms) {
  PaPlan w = {};
  w.sms = sms;
  const long rows = T * (Hq / Hkv), dp = D <= 64 ? 64 : 128;
  w.wide = rows > PA_NARROW_ROWS && T > batch;
  // with up to eight tiles per item, dividing them costs more (a second launch, partial results) than it balances
  w.whole = !w.wide && cap <= 8 * PA_TILE;
  w.narrow_max = w.wide ? PA_NARROW_ROWS : 0x7fffffff;
  w.narrow_rows = (int)(rows < PA_NARROW_ROWS ? rows : PA_NARROW_ROWS);
  w.narrow_ctas = (int)pa_ctas(T, batch, Hq, Hkv, cap, PA_NARROW_ROWS, w.whole, sms);
  w.wide_ctas = w.wide ? (int)pa_ctas(T, batch, Hq, Hkv, cap, PA_WIDE_ROWS, false, sms) : 0;
  auto size = [&](long ctas, long r) { return pa_align(2 * ctas * r * dp * 4) + pa_align(2 * ctas * r * 8) + pa_align(ctas * 32); };
  w.narrow_at = 0;
  w.wide_at = size(w.narrow_ctas, w.narrow_rows);
  w.bytes = w.wide_at + (w.wide ? size(w.wide_ctas, PA_WIDE_ROWS) : 0);
  return w;
}
void pa_place(PaParams* p, uint8_t* ws, long ctas, int rows, long dp) {
  p->part_rows = rows;
  p->part_o = reinterpret_cast<float*>(ws);
  ws += pa_align(2 * ctas * rows * dp * 4);
  p->part_ml = reinterpret_cast<float2*>(ws);
  ws += pa_align(2 * ctas * rows * 8);
  p->part_desc = reinterpret_cast<int*>(ws);
}

template <int PANELS, bool F16>
int pa_launch(const CUtensorMap& tmK, const CUtensorMap& tmV, PaParams p, const PaPlan& w, uint8_t* ws, cudaStream_t stream) {
  constexpr int SMEM = PaCfg<PANELS>::SMEM;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  static bool set[64] = {};  // the attribute belongs to a device
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(pa_wide_kernel<PANELS, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(pa_narrow_kernel<PANELS, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) set[dev] = true;
  }
  p.narrow_max = w.narrow_max;
  p.whole = w.whole;
  PaParams pn = p, pw = p;
  // measured 3 to 4 us per item, and 0.7 us per tile and 64 columns of the head; with 64 columns a mixed batch of 24
  // sequences took 61 / 54 / 63 us at a cost of 2 / 4 / 8
  pn.cost = pw.cost = PANELS == 1 ? 4 : 2;
  pa_place(&pn, ws + w.narrow_at, w.narrow_ctas, w.narrow_rows, PaCfg<PANELS>::DP);
  if (w.wide) {
    pa_place(&pw, ws + w.wide_at, w.wide_ctas, PA_WIDE_ROWS, PaCfg<PANELS>::DP);
    pa_wide_kernel<PANELS, F16><<<w.wide_ctas, PA_THREADS, SMEM, stream>>>(tmK, tmV, pw);
    SB_CHECK_LAUNCH();
  }
  // Launches that may start while the kernel before still runs: the narrow kernel reads nothing that the wide one writes,
  // its CTAs follow as SMs become free; the last kernel waits on the device.
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(w.narrow_ctas);
  cfg.blockDim = dim3(PA_THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = w.wide ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, pa_narrow_kernel<PANELS, F16>, tmK, tmV, pn);
  if (e != cudaSuccess) return (int)e;
  if (w.whole) return SB_OK;
  const int ctas = w.narrow_ctas + w.wide_ctas;
  // one wave of the four blocks per SM that fit; fewer for few descriptors (an item of the wide kernel has up to 32 tasks)
  cfg.gridDim = dim3(std::min(4 * w.sms, (w.wide ? 32 : 4) * ctas));
  cfg.blockDim = dim3(PA_COMBINE_THREADS);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, pa_combine_kernel<PANELS, F16>, pn, pw, w.narrow_ctas, ctas);
  return e == cudaSuccess ? SB_OK : (int)e;
}

}  // namespace

// Bytes of workspace of one call (contents need not be initialised); `cap` = positions that the page table can hold.
SB_API long sb200_paged_attention_workspace(int T, int batch, int Hq, int Hkv, int D, long cap, int sms) {
  if (T <= 0 || batch < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || sms <= 0) return 0;
  return pa_plan(T, batch, Hq, Hkv, D, cap, sms).bytes;
}

// out[t, h] for the new tokens of `batch` sequences, q / out [T, Hq, D] (token and head strides in elements), caches
// [num_pages, page_size, Hkv, D] (page, row and head strides; a page stride is a multiple of 8 row strides), bf16 or fp16.
// Sequence b: rows cu[b] .. cu[b + 1] of q, its last new token at position lens[b] - 1; position j in row j % page_size of
// page table[b][j / page_size].  A query at position i sees keys j <= i (causal), |i - j| <= window (window >= 0).  page_size is a power of two from 8, D a
// multiple of 8 up to 128; pointers and strides are multiples of 16 bytes.  Rows behind the last sequence are left as
// they are, or zeroed with zero_tail (as rows before the first).  Visible pages outside the
// cache, lengths outside the table and sequences that do not follow one another inside the T rows set *status.
SB_API int sb200_paged_attention(const void* q, const void* k_cache, const void* v_cache, void* out, const int* table,
                                 const int* cu, const int* lens, void* workspace, long workspace_bytes, int T, int batch,
                                 int Hq, int Hkv, int D, int num_pages, int page_size, int cols, long table_ld, long q_tok,
                                 long q_head, long o_tok, long o_head, long k_page, long k_row, long k_head, long v_page,
                                 long v_row, long v_head, int causal, int window, float scale, int zero_tail, int dtype,
                                 int sms, int* status, cudaStream_t stream) {
  if (T == 0) return SB_OK;
  if (T < 0 || batch < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || !status || !workspace || sms <= 0) return SB_ERR_BAD_ARG;
  if (D < 8 || D > 128 || D % 8 || num_pages < 1 || cols < 0) return SB_ERR_BAD_ARG;
  if (page_size < 8 || (page_size & (page_size - 1)) || !(scale > 0.f && scale < 1e30f)) return SB_ERR_BAD_ARG;
  if (dtype != SB_DT_BF16 && dtype != SB_DT_F16) return SB_ERR_BAD_ARG;
  const long cap = (long)cols * page_size;
  // 2^26 positions: an item then takes less time than the bound of a wait (PA_WAIT_NS)
  if ((long)T * Hq > (1L << 30) || cap > (1L << 26) || batch > (1 << 17) || Hq / Hkv > (1 << 15)) return SB_ERR_TOO_LARGE;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return SB_ERR_BAD_ARG;
  if ((q_tok | q_head | o_tok | o_head | k_page | k_row | k_head | v_page | v_row | v_head) % 8) return SB_ERR_BAD_ARG;
  if (workspace_bytes < sb200_paged_attention_workspace(T, batch, Hq, Hkv, D, cap, sms)) return SB_ERR_BAD_ARG;
  const bool f16 = dtype == SB_DT_F16;
  CUtensorMap tmK, tmV;
  int rc;
  PaParams p = {};
  const bool joined = D == 128;
  if ((rc = pa_tmap(&tmK, k_cache, D, Hkv, page_size, num_pages, k_page, k_row, k_head, f16, joined, &p.k_page8, &p.k_outside)))
    return rc;
  if ((rc = pa_tmap(&tmV, v_cache, D, Hkv, page_size, num_pages, v_page, v_row, v_head, f16, joined, &p.v_page8, &p.v_outside)))
    return rc;
  p.group_step = joined ? 2048 : 1024;
  p.panel_step = joined ? 1024 : PA_PANEL;
  p.boxes = joined || D <= 64 ? 1 : 2;
  const PaPlan w = pa_plan(T, batch, Hq, Hkv, D, cap, sms);
  p.q = q; p.out = out; p.table = table; p.cu = cu; p.lens = lens;
  p.table_ld = table_ld; p.q_tok = q_tok; p.q_head = q_head; p.o_tok = o_tok; p.o_head = o_head;
  p.T = T; p.batch = batch; p.Hkv = Hkv; p.group = Hq / Hkv;
  p.group_inv = (uint32_t)((1UL << 32) / p.group + 1);
  p.D = D; p.cols = cols; p.num_pages = num_pages;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.causal = causal; p.window = window < (1 << 30) ? window : 1 << 30; p.sl2 = scale * 1.4426950408889634f;
  p.zero_tail = zero_tail; p.status = status;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  if (D <= 64) return f16 ? pa_launch<1, true>(tmK, tmV, p, w, ws, stream) : pa_launch<1, false>(tmK, tmV, p, w, ws, stream);
  return f16 ? pa_launch<2, true>(tmK, tmV, p, w, ws, stream) : pa_launch<2, false>(tmK, tmV, p, w, ws, stream);
}
