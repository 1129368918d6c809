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
// One kernel serves decoding, which is a stream over K and V, and chunks, which are matrix products:
//  * An item is up to 256 query rows (tokens x heads that share a KV head, token-major) of one sequence and KV head.  All
//    items together are a line of 128-key tiles that is cut into equal pieces, one per CTA (one CTA per SM): ragged lengths
//    are balanced without the host knowing them.  A piece that starts or ends inside an item leaves an unnormalised
//    partial result; a second kernel joins them in the order of the CTAs, so results do not depend on timing.
//  * Two groups of four softmax warps (thread = query row = TMEM lane) work on different S = Q K^T at any time, so that
//    the tensor core computes for one while the other takes exponentials.  Items of more than 128 rows give each group
//    128 rows of its own ("two_q"); smaller items give both groups the same rows and every second key tile, and join the
//    two states at the end of the item.
//  * S of a group takes 128 TMEM columns; its probabilities overwrite the first 64 as packed 16-bit values and are
//    the TMEM operand of O += P V.  O stays in TMEM over the whole item.
//  * K and V tiles come by TMA through a ring that does not know items: the loader runs ahead into the next ones.
// Warp roles: 0-3 and 4-7 softmax groups, 8 and 11 TMA loaders of K and of V (a page of 16 tokens is a copy of its own, and
// one warp alone issues them no faster than the memory delivers), 9 MMA issuer, 10 scheduler, which also copies the queries.
//
// Rounding: scores, sums and outputs are fp32; P is rounded to the 16-bit element type for the second product (half a
// step per probability, averaged over the row), the output once.
#include <cuda.h>

#include "common.cuh"

namespace {

constexpr int PA_TILE = 128;
constexpr int PA_ITEM_ROWS = 256;
constexpr int PA_WARPS = 12;
constexpr int PA_THREADS = PA_WARPS * 32;
// registers per thread after the roles part: 128 x 80 + 256 x 208 = 63488 of the 384 x 168 that the launch holds
constexpr int PA_REGS_FEW = 80, PA_REGS_MANY = 208;
constexpr int PA_PANEL = 16384;   // 128 rows x 128 bytes
constexpr int PA_ITEMS = 4;       // descriptors in flight
constexpr int PA_COMBINE_THREADS = 256;

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
  // columns `panel_step` bytes behind the first.  boxes: copies per page (1: both panels at once); page_groups8: 8-row
  // groups of the tensor maps from one page to the next, and outside: a group beyond the cache
  uint32_t group_step, panel_step;
  int boxes, k_page8, v_page8, k_outside, v_outside;
  int causal, window;  // window < 0: unlimited
  float sl2;
  float* part_o;       // [2 slots per CTA][part_rows][DP]
  float2* part_ml;     // [2 slots per CTA][part_rows]: reference (log2 domain) and sum
  int* part_desc;      // [CTAs][8]: item that starts in this CTA and ends in a later one
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
  static constexpr int STAGES = PANELS == 2 ? 5 : 12;
  static constexpr int DATA = TILE_BYTES * (2 + STAGES);  // 224 KiB
  static constexpr int SMEM = DATA + 2048 + 1024;         // (m, l) exchange and control words
};

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
// Bounded wait of a whole warp: every lane gets the same answer, also when the wait gives up, so that no lane is missing
// from the warp-wide instructions that follow.
__device__ __forceinline__ bool pa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, sb::mbar_wait(bar, parity, abort_flag));
}
// tcgen05 instructions of one elected lane, predicated instead of branched around: the warp stays converged, so that
// descriptors and addresses, which are the same in all lanes, live in uniform registers.
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void pa_umma_ss(uint32_t leader, uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: A holds two 16-bit values of a row per 32-bit column
__device__ __forceinline__ void pa_umma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "setp.ne.b32 q, %5, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
// the barrier is reached once all MMAs issued so far by the leader are complete
__device__ __forceinline__ void pa_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(sb::smem_u32(bar)), "r"(leader)
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

// ------------------------------------------------------------------------------------------------ work line
struct PaSeq { int row0, n, L; };

__device__ __forceinline__ PaSeq pa_seq(const PaParams& p, int b) {
  PaSeq s;
  s.row0 = min(max(p.cu[b], 0), p.T);
  s.n = min(max(p.cu[b + 1], s.row0), p.T) - s.row0;
  const long cap = (long)p.cols << p.page_shift;
  int L = p.lens[b];
  if (L < 0 || L > cap) {  // a length that the table does not cover: reported, cut to what it covers
    *p.status = SB_ERR_BAD_ARG;
    L = L < 0 ? 0 : (int)cap;
  }
  s.L = L;
  return s;
}
// n / group for n < group + 256
__device__ __forceinline__ int pa_div(const PaParams& p, int n) { return p.group == 1 ? n : (int)__umulhi(n, p.group_inv); }
// keys that some row of item m sees
__device__ __forceinline__ void pa_item_keys(const PaParams& p, int n, int L, int m, int& lo, int& hi) {
  const int rows = n * p.group;
  const int first = m * PA_ITEM_ROWS / p.group, last = (min(rows, (m + 1) * PA_ITEM_ROWS) - 1) / p.group;
  const int pos0 = L - n + first, pos1 = L - n + last;
  lo = p.window >= 0 ? max(0, pos0 - p.window) : 0;
  hi = p.causal ? pos1 + 1 : (p.window >= 0 ? (int)min((long)L, (long)pos1 + p.window + 1) : L);
  hi = max(min(hi, L), 0);
}
// key tiles of item m, at least one: a row without keys still has to be written
__device__ __forceinline__ int pa_item_tiles(const PaParams& p, int n, int L, int m) {
  int lo, hi;
  pa_item_keys(p, n, L, m, lo, hi);
  return max((hi + PA_TILE - 1) / PA_TILE - lo / PA_TILE, 1);
}
__device__ __forceinline__ int pa_items(const PaParams& p, int n) {
  return (n * p.group + PA_ITEM_ROWS - 1) / PA_ITEM_ROWS;
}
__device__ __forceinline__ int pa_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ int pa_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }
// Tiles of all items of one KV head of sequence 32 * chunk + lane (0 beyond the last sequence); the whole warp calls.
__device__ __forceinline__ int pa_chunk_tiles(const PaParams& p, int chunk, int lane, PaSeq& s) {
  const int b = chunk * 32 + lane;
  s = PaSeq{0, 0, 0};
  if (b < p.batch) s = pa_seq(p, b);
  const int items = pa_items(p, s.n);
  int tiles = items == 1 ? pa_item_tiles(p, s.n, s.L, 0) : 0;
  unsigned many = __ballot_sync(0xffffffffu, items > 1);
  while (many) {  // long chunks: the warp shares the items of one sequence
    const int src = __ffs(many) - 1;
    many &= many - 1;
    const int n = __shfl_sync(0xffffffffu, s.n, src), L = __shfl_sync(0xffffffffu, s.L, src);
    const int cnt = pa_items(p, n);
    int sum = 0;
    for (int m = lane; m < cnt; m += 32) sum += pa_item_tiles(p, n, L, m);
    sum = pa_sum(sum);
    if (lane == src) tiles = sum;
  }
  return tiles;
}

// The line of `total` tiles is cut into `ctas` pieces of `per` tiles, the first `rest` of them one longer.
struct PaCut {
  int total, ctas, per, rest;
  __device__ __forceinline__ int start(int c) const { return c * per + min(c, rest); }
  __device__ __forceinline__ int owner(int tile) const {
    const int longer = rest * (per + 1);
    return tile < longer ? tile / (per + 1) : rest + (tile - longer) / per;
  }
};
struct PaCursor {  // where a CTA's piece of the line starts, and how long it is
  PaSeq s;
  int seq, hk, m, tile, left, unit;
  PaCut cut;
};

// The whole warp; sums[c] = tiles per KV head of sequences 32 c .. 32 c + 31.
__device__ __forceinline__ void pa_find(const PaParams& p, const int* sums, int chunks, int lane, PaCursor& c) {
  long long all = 0;
  for (int i = lane; i < chunks; i += 32) all += sums[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  all *= p.Hkv;
  c = PaCursor{};
  if (all > 0x7fffffff) {  // months of work
    if (lane == 0) *p.status = SB_ERR_TOO_LARGE;
    return;
  }
  PaCut& cut = c.cut;
  cut.total = (int)all;
  cut.ctas = min((int)gridDim.x, (cut.total + 1) / 2);  // two tiles per CTA at least: one for each softmax group
  if ((int)blockIdx.x >= cut.ctas) return;
  cut.per = cut.total / cut.ctas;
  cut.rest = cut.total - cut.per * cut.ctas;
  c.unit = cut.start(blockIdx.x);
  c.left = cut.per + ((int)blockIdx.x < cut.rest);
  int off = c.unit, chunk = 0;
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
  }
  PaSeq s;
  const int tiles = pa_chunk_tiles(p, chunk, lane, s), v = tiles * p.Hkv, inc = pa_scan(v, lane);
  const int k = __ffs(__ballot_sync(0xffffffffu, inc > off)) - 1;
  off -= __shfl_sync(0xffffffffu, inc - v, k);
  const int per_head = __shfl_sync(0xffffffffu, tiles, k);
  c.s = PaSeq{__shfl_sync(0xffffffffu, s.row0, k), __shfl_sync(0xffffffffu, s.n, k), __shfl_sync(0xffffffffu, s.L, k)};
  c.seq = chunk * 32 + k;
  c.hk = off / per_head;
  off -= c.hk * per_head;
  const int items = pa_items(p, c.s.n);
  c.tile = off;
  if (items > 1) {
    for (int base = 0; base < items; base += 32) {
      const int t = base + lane < items ? pa_item_tiles(p, c.s.n, c.s.L, base + lane) : 0, ti = pa_scan(t, lane);
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

// Places of K and V tiles of an item in the ring: `lead` K tiles run ahead of V (1 with two_q, else 2: both groups need
// their first S before the first V), then V and K alternate - the order in which the MMA warp takes them.
__device__ __forceinline__ uint32_t pa_k_place(int t, int lead) { return t < lead ? t : 2 * t - lead + 1; }
__device__ __forceinline__ uint32_t pa_v_place(int t, int lead, int count) { return t + min(t + lead, count); }

// ============================================================================ main kernel
template <int PANELS, bool F16>
__global__ void __launch_bounds__(PA_THREADS, 1)
    pa_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const PaParams p) {
  using Cfg = PaCfg<PANELS>;
  constexpr int DP = Cfg::DP, TILE_BYTES = Cfg::TILE_BYTES, STAGES = Cfg::STAGES;
  constexpr uint32_t S_COL = 0, O_COL = 256;  // two S buffers of 128 columns, two O of DP
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;                          // two slots of 128 rows
  uint8_t* sRing = smem + 2 * TILE_BYTES;
  float2* xml = reinterpret_cast<float2*>(smem + Cfg::DATA);  // [group][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::DATA + 2048);
  uint64_t* full = bars;                       // STAGES
  uint64_t* empty = full + STAGES;             // STAGES
  uint64_t* q_full = empty + STAGES;           // 2
  uint64_t* q_empty = q_full + 2;              // 2
  uint64_t* s_full = q_empty + 2;              // 2
  uint64_t* p_full = s_full + 2;               // 2
  uint64_t* o_full = p_full + 2;               // 2
  uint64_t* epi_done = o_full + 2;             // 1
  uint64_t* merge = epi_done + 1;              // [group][quadrant]
  uint64_t* item_full = merge + 8;             // PA_ITEMS
  uint64_t* item_empty = item_full + PA_ITEMS; // PA_ITEMS
  PaItem* items = reinterpret_cast<PaItem*>(item_empty + PA_ITEMS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + PA_ITEMS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * STAGES + 11 + 8 + 2 * PA_ITEMS) * 8 + PA_ITEMS * sizeof(PaItem) + 8 <= 1024, "control words");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (sb::smem_u32(smem) & 1023) {  // the swizzled tiles need it; dynamic shared memory starts on such a boundary
    if (threadIdx.x == 0) *p.status = SB_ERR_BAD_ARG;
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      sb::mbar_init(&full[i], 1);
      sb::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      sb::mbar_init(&q_full[i], 1);
      sb::mbar_init(&q_empty[i], 1);
      sb::mbar_init(&s_full[i], 1);
      sb::mbar_init(&p_full[i], 4);
      sb::mbar_init(&o_full[i], 1);
    }
    sb::mbar_init(epi_done, 8);
    for (int i = 0; i < 8; ++i) sb::mbar_init(&merge[i], 1);
    for (int i = 0; i < PA_ITEMS; ++i) {
      sb::mbar_init(&item_full[i], 1);
      sb::mbar_init(&item_empty[i], 10);
    }
    *abort_flag = 0;
    sb::mbar_fence_init();
  }
  if (warp == 9) {
    sb::tmem_alloc(tmem_slot, 512);
    sb::tmem_relinquish();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // tiles of 32 sequences at a time, where the scheduler puts the queries afterwards
  int* sums = reinterpret_cast<int*>(sQ);
  const int chunks = (p.batch + 31) / 32;
  for (int c = warp; c < chunks; c += PA_WARPS) {
    PaSeq s;
    const int t = pa_sum(pa_chunk_tiles(p, c, lane, s));
    if (lane == 0) sums[c] = t;
  }
  sb::tc_fence_before();
  __syncthreads();
  sb::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= 8) {
  pa_regs_dec<PA_REGS_FEW>();  // one instruction for the whole warpgroup
  if (warp == 10) {
    // ------------------------------------------------------------------ scheduler and query loads
    PaCursor cur;
    pa_find(p, sums, chunks, lane, cur);
    __syncwarp();
    int* desc = p.part_desc + 8 * blockIdx.x;
    bool starts = false, ok = true;
    int q_cnt = 0;
    for (int i = 0; ok; ++i) {
      const int slot = i % PA_ITEMS;
      if (!pa_wait(&item_empty[slot], ((i / PA_ITEMS) & 1) ^ 1, abort_flag)) break;
      PaItem it = {};
      int tiles = 0;
      if (cur.left > 0) {
        int lo, hi;
        pa_item_keys(p, cur.s.n, cur.s.L, cur.m, lo, hi);
        tiles = max((hi + PA_TILE - 1) / PA_TILE - lo / PA_TILE, 1);
        const int take = min(tiles - cur.tile, cur.left);
        const bool first = cur.tile == 0, last = cur.tile + take == tiles;
        const int tok0 = cur.m * PA_ITEM_ROWS / p.group;
        it = PaItem{cur.s.row0 + tok0, cur.s.L - cur.s.n + tok0, cur.s.L, cur.seq, cur.hk,
                    min(cur.s.n * p.group - cur.m * PA_ITEM_ROWS, PA_ITEM_ROWS), cur.m * PA_ITEM_ROWS - tok0 * p.group,
                    lo / PA_TILE + cur.tile, take, lo, hi,
                    first && last ? -1 : 2 * (int)blockIdx.x + (first ? 1 : 0)};
        if (first && !last) {  // the CTA that starts an item names the one that ends it
          starts = true;
          if (lane == 0) {
            desc[1] = it.row0; desc[2] = it.rem; desc[3] = it.hk; desc[4] = it.rows;
            desc[5] = cur.cut.owner(cur.unit + tiles - 1);
          }
        }
        cur.left -= take;
        cur.unit += take;
      }
      if (lane == 0) {
        items[slot] = it;
        sb::mbar_arrive(&item_full[slot]);
      }
      if (it.count == 0) break;
      // queries of the item: one slot, or two of them, as 16-byte chunks in the swizzled K-major layout
      const int slots = it.rows > PA_TILE ? 2 : 1;
      for (int x = 0; x < slots; ++x) {
        const int qs = (q_cnt + x) & 1;
        ok = pa_wait(&q_empty[qs], (((q_cnt + x) >> 1) & 1) ^ 1, abort_flag);
        if (!ok) break;
        constexpr int CH = DP / 8;  // chunks per row
        const int ch = lane % CH, live = min(it.rows - x * PA_TILE, PA_TILE), end = (live + 31) & ~31;
        const uint32_t dst = sb::smem_u32(sQ + qs * TILE_BYTES) + (ch >> 3) * PA_PANEL;
        const uint16_t* base = reinterpret_cast<const uint16_t*>(p.q) + (long)it.row0 * p.q_tok +
                               (long)it.hk * p.group * p.q_head + ch * 8;
        // whole warps of rows: lanes without a row read zeros
#pragma unroll 4
        for (int r = lane / CH; r < end; r += 32 / CH) {
          const int row = it.rem + x * PA_TILE + r, t = pa_div(p, row), h = row - t * p.group;
          const bool take = r < live && ch * 8 < p.D;
          pa_cp16(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                  take ? base + (long)t * p.q_tok + (long)h * p.q_head : reinterpret_cast<const uint16_t*>(p.q), take);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        sb::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) sb::mbar_arrive(&q_full[qs]);
      }
      q_cnt += slots;
      cur.tile = 0;
      if (cur.left > 0 && ++cur.m == pa_items(p, cur.s.n)) {
        cur.m = 0;
        if (++cur.hk == p.Hkv) {
          cur.hk = 0;
          do { cur.s = pa_seq(p, ++cur.seq); } while (cur.s.n == 0 && cur.seq + 1 < p.batch);
        }
      }
    }
    if (lane == 0) desc[0] = starts && ok;
  } else if (warp != 9) {
    // ------------------------------------------------------------------ K tiles (warp 8), V tiles (warp 11)
    const bool is_v = warp == 11;
    const CUtensorMap* tm = is_v ? &tmV : &tmK;
    if (lane == 0) sb::tma_prefetch_desc(tm);
    const int page = 1 << p.page_shift;
    const int box = min(page, PA_TILE), per_tile = PA_TILE / box;  // rows per copy, pages per tile
    const int bi = lane % per_tile, pn = lane / per_tile;          // this lane's page of the tile, and its panel
    const int page8 = is_v ? p.v_page8 : p.k_page8, outside = is_v ? p.v_outside : p.k_outside;
    const uint32_t dst = sb::smem_u32(sRing) + bi * (box >> 3) * p.group_step + pn * p.panel_step;
    uint32_t ring = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const int slot = i % PA_ITEMS;
      if (!pa_wait(&item_full[slot], (i / PA_ITEMS) & 1, abort_flag)) break;
      const PaItem it = items[slot];
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&item_empty[slot]);
      if (it.count == 0) break;
      const int lead = it.rows > PA_TILE ? 1 : 2;
      const int* trow = p.table + (long)it.seq * p.table_ld;
      int win = -64, where = 0;  // 32 pages at a time: their first 8-row group in the tensor map
      for (int t = 0; t < it.count; ++t) {
        const int key0 = (it.tile0 + t) * PA_TILE, page0 = key0 >> p.page_shift;
        if (page0 + per_tile > win + 32) {
          win = page0;
          const int idx = page0 + lane;
          where = outside;  // a copy from outside the cache reads zeros
          if (idx < p.cols && ((idx + 1) << p.page_shift) > it.lo && (idx << p.page_shift) < it.hi) {
            const int got = trow[idx];
            if (got >= 0 && got < p.num_pages) where = got * page8;
            else *p.status = SB_ERR_BAD_ARG;  // a visible page outside the cache: reported, its keys read as zeros
          }
        }
        const int first8 = __shfl_sync(0xffffffffu, where, page0 - win + bi);
        const uint32_t e = ring + (is_v ? pa_v_place(t, lead, it.count) : pa_k_place(t, lead)), st = e % STAGES;
        ok = pa_wait(&empty[st], ((e / STAGES) & 1) ^ 1, abort_flag);
        if (!ok) break;
        if (lane == 0) sb::mbar_expect_tx(&full[st], TILE_BYTES);
        __syncwarp();
        if (pn < p.boxes)
          pa_tma_5d(dst + st * TILE_BYTES, tm, &full[st], pn * 64, first8 + ((key0 & (page - 1)) >> 3), it.hk);
      }
      ring += 2 * it.count;
    }
  } else {
    // ------------------------------------------------------------------ MMA issue
    const uint32_t leader = lane == 0;
    const uint32_t idesc_s = sb::umma_idesc_f16(PA_TILE, PA_TILE, F16 ? 0 : 1, 0, 0);  // K-major both
    const uint32_t idesc_o = sb::umma_idesc_f16(PA_TILE, DP, F16 ? 0 : 1, 0, 1);       // V is MN-major
    const uint64_t q_desc = sb::umma_smem_desc(sb::smem_u32(sQ), 16, 1024);
    const uint64_t k_desc = sb::umma_smem_desc(sb::smem_u32(sRing), 16, p.group_step);
    const uint64_t v_desc = sb::umma_smem_desc(sb::smem_u32(sRing), p.panel_step, p.group_step);
    const uint32_t k_panel = p.panel_step >> 4, v_step = (2 * p.group_step) >> 4;  // descriptors count 16-byte units
    uint32_t ring = 0, p_cnt0 = 0, p_cnt1 = 0;
    int q_cnt = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const int slot = i % PA_ITEMS;
      if (!pa_wait(&item_full[slot], (i / PA_ITEMS) & 1, abort_flag)) break;
      const int count = __shfl_sync(0xffffffffu, items[slot].count, 0);
      const int two_q = __shfl_sync(0xffffffffu, items[slot].rows > PA_TILE, 0);
      if (lane == 0) sb::mbar_arrive(&item_empty[slot]);
      if (count == 0) break;
      const int lead = two_q ? 1 : 2, n = two_q ? 2 * count : count;
      ok = pa_wait(&q_full[q_cnt & 1], (q_cnt >> 1) & 1, abort_flag);
      if (ok && two_q) ok = pa_wait(&q_full[(q_cnt + 1) & 1], ((q_cnt + 1) >> 1) & 1, abort_flag);
      if (!ok) break;
      // virtual tile v: group v & 1; key tile v (one query slot) or v / 2 (two)
      auto issue_s = [&](int v) -> bool {
        const uint32_t e = ring + pa_k_place(two_q ? v >> 1 : v, lead), st = e % STAGES;
        if (!pa_wait(&full[st], (e / STAGES) & 1, abort_flag)) return false;
        sb::tc_fence_after();
        const int qs = (q_cnt + (two_q ? v & 1 : 0)) & 1;
        const uint64_t qd = q_desc + qs * (TILE_BYTES >> 4), kd = k_desc + st * (TILE_BYTES >> 4);
        const uint32_t d = tmem_base + S_COL + (v & 1) * PA_TILE;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          pa_umma_ss(leader, d, qd + (kk >> 2) * (PA_PANEL >> 4) + (kk & 3) * 2, kd + (kk >> 2) * k_panel + (kk & 3) * 2,
                     idesc_s, kk != 0);
        pa_commit(leader, &s_full[v & 1]);
        if (!two_q || (v & 1)) pa_commit(leader, &empty[st]);
        if (two_q ? v >= n - 2 : v == n - 1) pa_commit(leader, &q_empty[qs]);
        return true;
      };
      ok = issue_s(0);
      if (ok && n > 1) ok = issue_s(1);
      for (int v = 0; v < n && ok; ++v) {
        const int x = v & 1;
        const uint32_t e = ring + pa_v_place(two_q ? v >> 1 : v, lead, count), st = e % STAGES;
        ok = pa_wait(&p_full[x], (x ? p_cnt1 : p_cnt0) & 1, abort_flag) && pa_wait(&full[st], (e / STAGES) & 1, abort_flag);
        if (ok && v == 0 && i > 0) ok = pa_wait(epi_done, (i - 1) & 1, abort_flag);  // O of the item before is read
        if (!ok) break;
        if (x) ++p_cnt1; else ++p_cnt0;
        sb::tc_fence_after();
        const uint64_t vd = v_desc + st * (TILE_BYTES >> 4);
        const uint32_t pa = tmem_base + S_COL + x * PA_TILE, d = tmem_base + O_COL + x * DP;
#pragma unroll
        for (int kk = 0; kk < PA_TILE / 16; ++kk)
          pa_umma_ts(leader, d, pa + kk * 8, vd + kk * v_step, idesc_o, v > 1 || kk != 0);
        if (!two_q || x) pa_commit(leader, &empty[st]);
        if (v + 2 >= n) pa_commit(leader, &o_full[x]);
        if (v + 2 < n) ok = issue_s(v + 2);
      }
      ring += 2 * count;
      q_cnt += 1 + two_q;
    }
  }
  } else {
    // ------------------------------------------------------------------ softmax and output
    pa_regs_inc<PA_REGS_MANY>();
    const int x = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = t_lane + S_COL + x * PA_TILE, o_addr = t_lane + O_COL + x * DP;
    const float sl2 = p.sl2;
    uint32_t ring = 0, s_cnt = 0, o_cnt = 0, merges = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const int islot = i % PA_ITEMS;
      if (!pa_wait(&item_full[islot], (i / PA_ITEMS) & 1, abort_flag)) break;
      const PaItem it = items[islot];
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(&item_empty[islot]);
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
      const int n = two_q ? 2 * it.count : it.count;
      for (int v = x; v < n; v += 2) {
        const int t = two_q ? v >> 1 : v;
        const int key0 = (it.tile0 + t) * PA_TILE;
        if (!pa_wait(&s_full[x], s_cnt & 1, abort_flag)) { ok = false; break; }
        ++s_cnt;
        sb::tc_fence_after();
        if (warp_rows > 0) {
          uint32_t s[PA_TILE];
#pragma unroll
          for (int c = 0; c < 4; ++c) sb::tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(s + c * 32));
          sb::tmem_ld_wait();
          if (!__all_sync(0xffffffffu, key0 >= lo && key0 + PA_TILE <= hi)) {
#pragma unroll
            for (int c = 0; c < PA_TILE; ++c)
              if (key0 + c < lo || key0 + c >= hi) s[c] = 0xff800000u;  // -inf, whatever the score was
          }
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < PA_TILE; ++c) m4[c & 3] = fmaxf(m4[c & 3], __uint_as_float(s[c]));
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          const bool move = (mx - ref) * sl2 > 8.f || (ref == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xffffffffu, move)) {
            const float next = move ? mx : ref;
            const float alpha = move ? (ref == -INFINITY ? 0.f : pa_exp2((ref - next) * sl2)) : 1.f;
            ref = next;
            l *= alpha;
            if (v >= 2) {  // O holds the tiles before (complete: their MMAs precede this S)
#pragma unroll
              for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[32];
                sb::tmem_ld32(o_addr + c * 32, o);
                sb::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                pa_tmem_st32(o_addr + c * 32, o);
              }
            }
          }
          const float neg = ref == -INFINITY ? 0.f : -ref * sl2;
          float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float a = pa_exp2(fmaf(__uint_as_float(s[c * 64 + 2 * j]), sl2, neg));
              const float b = pa_exp2(fmaf(__uint_as_float(s[c * 64 + 2 * j + 1]), sl2, neg));
              sum4[(2 * j) & 3] += a;
              sum4[(2 * j + 1) & 3] += b;
              pk[j] = pa_pack<F16>(a, b);
            }
            pa_tmem_st32(s_addr + c * 32, pk);
          }
          l += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
          sb::tmem_st_wait();
        }
        if (key0 + PA_TILE > it.hi) {
          // Values behind the last visible key may be anything, NaN included, and 0 * NaN is NaN: their rows of the
          // V tile are zeroed (twice with two_q, which does no harm).  Thread = key row.
          const uint32_t e = ring + pa_v_place(t, lead, it.count), st = e % STAGES;
          if (!pa_wait(&full[st], (e / STAGES) & 1, abort_flag)) { ok = false; break; }
          if (key0 + r >= it.hi) {
            uint8_t* dst = sRing + st * TILE_BYTES + (r >> 3) * p.group_step + (r & 7) * 128;
#pragma unroll
            for (int c = 0; c < PANELS * 8; ++c)
              *reinterpret_cast<uint4*>(dst + (c >> 3) * p.panel_step + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          sb::fence_proxy_async_smem();
        }
        sb::tc_fence_before();
        __syncwarp();
        if (lane == 0) sb::mbar_arrive(&p_full[x]);
      }
      ring += 2 * it.count;
      if (!ok) break;
      const bool mine = x < n;  // this group had a tile
      if (mine) {
        if (!pa_wait(&o_full[x], o_cnt & 1, abort_flag)) break;
        ++o_cnt;
        sb::tc_fence_after();
      }
      // the two states of a row: fa, fb scale the groups' outputs to a common reference
      float fa = x == 0 ? 1.f : 0.f, fb = 1.f - fa;
      int c0 = 0, c1 = DP / 32;
      const bool both = !two_q && n > 1;
      if (!two_q) {
        if (i > 0 && !pa_wait(epi_done, (i - 1) & 1, abort_flag)) break;  // xml of the item before is read
        xml[x * PA_TILE + r] = make_float2(ref, l);
        sb::tc_fence_before();
        __syncwarp();
        if (lane == 0) sb::mbar_arrive(&merge[x * 4 + quad]);
        if (!pa_wait(&merge[(x ^ 1) * 4 + quad], merges & 1, abort_flag)) break;
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
        for (int c = c0; c < c1; ++c) {
          uint32_t a[32], b[32];
          float o[32];
          if (both) {
            sb::tmem_ld32(t_lane + O_COL + c * 32, a);
            sb::tmem_ld32(t_lane + O_COL + DP + c * 32, b);
            sb::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = fmaf(__uint_as_float(a[j]), ga, __uint_as_float(b[j]) * gb);
          } else {  // one state: this group's (two_q), or group 0's
            sb::tmem_ld32((two_q ? o_addr : t_lane + O_COL) + c * 32, a);
            sb::tmem_ld_wait();
            const float f = two_q && x ? gb : ga;
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __uint_as_float(a[j]) * f;
          }
          if (row >= rows) {
          } else if (it.slot < 0) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              if (c * 32 + j < p.D) {
                uint4 u;
                u.x = pa_pack<F16>(o[j], o[j + 1]);
                u.y = pa_pack<F16>(o[j + 2], o[j + 3]);
                u.z = pa_pack<F16>(o[j + 4], o[j + 5]);
                u.w = pa_pack<F16>(o[j + 6], o[j + 7]);
                *reinterpret_cast<uint4*>(dst + c * 32 + j) = u;
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(p.part_o + prow * DP + c * 32 + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
          __syncwarp();
        }
        if (it.slot >= 0 && row < rows && (two_q || x == 0))
          p.part_ml[prow] = make_float2(ref == -INFINITY ? -INFINITY : ref * sl2, l);
      }
      sb::tc_fence_before();
      __syncwarp();
      if (lane == 0) sb::mbar_arrive(epi_done);
    }
  }

  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies and MMAs in flight end
  }
  sb::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    sb::tc_fence_after();
    sb::tmem_dealloc(tmem_base, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) *p.status = SB_ERR_WAIT_TIMEOUT;
}

// ============================================================================ joining the partial results
// blockIdx.x: the CTA that started an item; blockIdx.y strides over the item's rows.  Thread = (part group, four columns):
// each group runs over every PG-th part with an online reference, the groups are joined in order.
template <int PANELS, bool F16>
__global__ void __launch_bounds__(PA_COMBINE_THREADS) pa_combine_kernel(const PaParams p) {
  constexpr int DP = PANELS * 64, QUADS = DP / 4, PG = PA_COMBINE_THREADS / QUADS;
  __shared__ float4 so[PG][QUADS];
  __shared__ float2 sml[PG];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.zero_tail) {  // rows behind the last sequence
    const long first = p.batch > 0 ? min(max(p.cu[p.batch], 0), p.T) : 0, heads = (long)p.Hkv * p.group;
    const long chunks = (p.T - first) * heads * (p.D / 8);
    const long step = (long)gridDim.x * gridDim.y * PA_COMBINE_THREADS;
    for (long c = ((long)blockIdx.y * gridDim.x + blockIdx.x) * PA_COMBINE_THREADS + threadIdx.x; c < chunks; c += step) {
      const long row = c / (p.D / 8), t = row / heads;
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + (first + t) * p.o_tok + (row - t * heads) * p.o_head +
                                (c - row * (p.D / 8)) * 8) = make_uint4(0, 0, 0, 0);
    }
  }
  const int* desc = p.part_desc + 8 * blockIdx.x;
  if (!desc[0]) return;
  const int row0 = desc[1], rem = desc[2], hk = desc[3], rows = desc[4], last = desc[5];
  const int quad = threadIdx.x % QUADS, pg = threadIdx.x / QUADS;
  for (int row = blockIdx.y; row < rows; row += gridDim.y) {
    float ref = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = (int)blockIdx.x + pg; c <= last; c += PG) {
      const long prow = (long)(2 * c + (c == (int)blockIdx.x ? 1 : 0)) * p.part_rows + row;
      const float2 ml = p.part_ml[prow];
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + prow * DP + quad * 4);
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // a part without a visible key
      const float next = fmaxf(ref, ml.x);
      const float a = ref == -INFINITY ? 0.f : exp2f(ref - next), b = exp2f(ml.x - next);
      l = l * a + ml.y * b;
      o.x = o.x * a + v.x * b; o.y = o.y * a + v.y * b; o.z = o.z * a + v.z * b; o.w = o.w * a + v.w * b;
      ref = next;
    }
    __syncthreads();
    so[pg][quad] = o;
    if (quad == 0) sml[pg] = make_float2(ref, l);
    __syncthreads();
    if (pg == 0) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int g = 0; g < PG; ++g) top = fmaxf(top, sml[g].x);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int g = 0; g < PG; ++g) {
        const float2 ml = sml[g];
        if (ml.x == -INFINITY && ml.y == 0.f) continue;
        const float f = exp2f(ml.x - top);
        const float4 v = so[g][quad];
        sum += ml.y * f;
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
      }
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      const int tok = pa_div(p, rem + row), head = hk * p.group + (rem + row - tok * p.group);
      if (quad * 4 < p.D) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (long)(row0 + tok) * p.o_tok + (long)head * p.o_head + quad * 4;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pa_pack<F16>(acc.x * inv, acc.y * inv), pa_pack<F16>(acc.z * inv, acc.w * inv));
      }
    }
  }
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

// CTAs of the main launch: one per SM, fewer when not even the table's full length gives each of them two key tiles
long pa_ctas(long T, int batch, int Hq, int Hkv, long cap, int sms) {
  const long items = (T * (Hq / Hkv) + PA_ITEM_ROWS - 1) / PA_ITEM_ROWS + batch;
  const long tiles = (cap + PA_TILE - 1) / PA_TILE + 1;
  const long want = (items * Hkv * tiles + 1) / 2;
  return want < 1 ? 1 : want < sms ? want : sms;
}
int pa_part_rows(long T, int group) { return T * group < PA_ITEM_ROWS ? (int)(T * group) : PA_ITEM_ROWS; }
long pa_align(long v) { return (v + 255) & ~255L; }

template <int PANELS, bool F16>
int pa_launch(const CUtensorMap& tmK, const CUtensorMap& tmV, const PaParams& p, int ctas, cudaStream_t stream) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  static bool set[64] = {};  // the attribute belongs to a device
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(pa_kernel<PANELS, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, PaCfg<PANELS>::SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) set[dev] = true;
  }
  pa_kernel<PANELS, F16><<<ctas, PA_THREADS, PaCfg<PANELS>::SMEM, stream>>>(tmK, tmV, p);
  SB_CHECK_LAUNCH();
  // launched while the main kernel still runs; waits for it on the device
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, p.part_rows < 16 ? p.part_rows : 16);
  cfg.blockDim = dim3(PA_COMBINE_THREADS);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, pa_combine_kernel<PANELS, F16>, p);
  return e == cudaSuccess ? SB_OK : (int)e;
}

}  // namespace

// Bytes of workspace of one call (contents need not be initialised); `cap` = positions that the page table can hold.
SB_API long sb200_paged_attention_workspace(int T, int batch, int Hq, int Hkv, int D, long cap, int sms) {
  if (T <= 0 || batch < 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || D <= 0 || sms <= 0) return 0;
  const long slots = 2 * pa_ctas(T, batch, Hq, Hkv, cap, sms), rows = pa_part_rows(T, Hq / Hkv), dp = D <= 64 ? 64 : 128;
  return pa_align(slots * rows * dp * 4) + pa_align(slots * rows * 8) + slots / 2 * 32;
}

// out[t, h] for the new tokens of `batch` sequences, q / out [T, Hq, D] (token and head strides in elements), caches
// [num_pages, page_size, Hkv, D] (page, row and head strides; a page stride is a multiple of 8 row strides), bf16 or fp16.  Sequence b: rows cu[b] .. cu[b + 1] of q, its
// last new token at position lens[b] - 1; position j in row j % page_size of page table[b][j / page_size].  A query at
// position i sees keys j <= i (causal), |i - j| <= window (window >= 0).  page_size is a power of two from 8, D a
// multiple of 8 up to 128; pointers and strides are multiples of 16 bytes.  Rows behind the last sequence are left as
// they are, or zeroed with zero_tail.  Visible pages outside the cache and lengths outside the table set *status.
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
  if ((long)T * Hq > (1L << 30) || cap > (1L << 30) || batch > (1 << 17) || Hq / Hkv > (1 << 15)) return SB_ERR_TOO_LARGE;
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
  const int ctas = (int)pa_ctas(T, batch, Hq, Hkv, cap, sms), dp = D <= 64 ? 64 : 128;
  p.q = q; p.out = out; p.table = table; p.cu = cu; p.lens = lens;
  p.table_ld = table_ld; p.q_tok = q_tok; p.q_head = q_head; p.o_tok = o_tok; p.o_head = o_head;
  p.T = T; p.batch = batch; p.Hkv = Hkv; p.group = Hq / Hkv;
  p.group_inv = (uint32_t)((1UL << 32) / p.group + 1);
  p.D = D; p.cols = cols; p.num_pages = num_pages;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.causal = causal; p.window = window < (1 << 30) ? window : 1 << 30; p.sl2 = scale * 1.4426950408889634f;
  p.part_rows = pa_part_rows(T, p.group);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  ws += pa_align(2L * ctas * p.part_rows * dp * 4);
  p.part_ml = reinterpret_cast<float2*>(ws);
  ws += pa_align(2L * ctas * p.part_rows * 8);
  p.part_desc = reinterpret_cast<int*>(ws);
  p.zero_tail = zero_tail; p.status = status;
  if (D <= 64) return f16 ? pa_launch<1, true>(tmK, tmV, p, ctas, stream) : pa_launch<1, false>(tmK, tmV, p, ctas, stream);
  return f16 ? pa_launch<2, true>(tmK, tmV, p, ctas, stream) : pa_launch<2, false>(tmK, tmV, p, ctas, stream);
}
