// Per-head norm and rotary embedding of queries and keys in one pass over the projections, forward and backward, and
// the same forward pass writing keys and values into a paged cache.
//
// A row is one head of one token, x[0 .. D).  With r = 1 / sqrt(mean((x - mu)^2) + eps) (mu = 0 for RMS) and
// xhat = (x - mu) r:
//   y = xhat * w + b,  out = R(pos) y        R rotates the pairs of the first `rot` elements by pos * base^(-2 i / rot)
//   dy = R(pos)^T dout,  db = sum_rows dy,  dw = sum_rows dy * xhat,  g = dy * w,
//   dx = r (g - [mean(g)] - xhat mean(g xhat))                          (mean(g) for LayerNorm only)
// (src/scaling/core/nn/attention/attention.py:812-850 norms, transposes and rotates in separate passes.)
//
// The work is a stream: every element is read and written once (x twice over a training step, because the backward
// pass recomputes mu and r from x instead of reading stored ones).  A row is held by G lanes in registers, each with two
// 16-byte chunks A and B that are chosen so that every rotary pair lies inside one lane: for the rotate-half convention
// A = [l V, l V + V) and B = A + rot / 2, for interleaved pairs and the unrotated rest A and B are neighbours.  So the
// rotation needs no exchange; only the row sums go through shuffles.  Statistics, weights, sines and products stay in
// fp32 and are rounded once, at the store.
//
// Measured on one B200 (copy 6.57 TB/s), device time in a captured graph, forward and backward together: 8192 tokens, 32 + 8
// heads of 128, RMS, interleaved rotation, bf16: 115 us = 3.6 TB/s (0.55 of the copy); 16384 tokens, 12 + 12 heads of 64, layer
// norm with biases, packed projection: 83 us (0.46); a decoding step's append 6.5 us; an append of some 6000 prompt tokens,
// 40 + 1 heads: 39 us (0.51).  Eager calls take 165, 183, 32 and 41 us: the first three are bound by the enqueue.
// Bound by latency at the occupancy that the registers leave (three blocks per SM forward, two backward; 51 and 39 % of the
// issue slots, 35 % of the DRAM cycles).  Per element there are conversions, the norm's shuffles and three passes of fp32
// arithmetic; hence the packed fp32 forms, weights in registers, code of its own per kind of row and per common head size.
//
// Angles: a position of 10^5 times a frequency near 1 in fp32 is off by 10^-2 rad.  The host computes turns per position
// base^(-2 i / rot) / (2 pi) in fp64; a thread multiplies by the position, drops the whole turns in fp64 and takes
// sincospi of what is left in fp32.  One thread per (token, pair) fills a table in shared memory that all heads of the
// token read.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace {

constexpr int QN_THREADS = 256;
constexpr int QN_FWD_BLOCKS = 3;          // per SM (4 of them, with fewer registers: 150 us where the 7B step took 134)
constexpr int QN_MAX_D = 256;
constexpr int QN_MAX_SLOTS = 64;          // tokens per tile
constexpr int QN_TABLE_BYTES = 24 * 1024; // sine table of a tile

struct QnRows {  // one of q, k, v: the heads of every token
  const void* x;
  void* y;       // forward: out, backward: dx
  const void* dy;
  const void* w; // null: no norm
  const void* b;
  long x_tok, x_head, y_tok, y_head, dy_tok, dy_head;
  int heads;
  uint32_t inv;  // floor(2^32 / heads) + 1 (heads > 1): (n * inv) >> 32 = n / heads for the row numbers of a tile
};

struct QnParams {
  QnRows q, k, v;
  const int* pos;   // [T], or null in the paged form: the token's place in its sequence
  int T, D, rot, interleaved, rms, w_dtype;
  float eps;
  int tile, tile_k; // tokens per tile (backward: of q and of k)
  int log_g;        // lanes per row, as a power of two
  // paged form: k.y / v.y are the caches, y_head the stride between heads of a slot
  const int* table;
  const int* cu;
  const int* lens;
  long table_ld, k_page, k_slot, v_page, v_slot;
  int batch, cols, num_pages, page_shift;
  int* status;
  // backward
  float* partial;   // [blocks][2 * D]: sums of dw and db of each block
  int q_blocks;     // blocks 0 .. q_blocks - 1 take q, the others k
  double turns[QN_MAX_D / 2];
};

__device__ __forceinline__ float qn_load_any(const void* p, int i, int dtype) {
  if (dtype == SB_DT_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == SB_DT_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ int qn_token(const QnRows& r, int row) { return r.heads == 1 ? row : (int)__umulhi(row, r.inv); }

// Asks L2 for row `row` of a tile that starts at token t0: the lanes' 32-byte pieces of x (and of dy).  Registers hold the
// rows of one round ahead and no more; two further rounds under way take the 7B training step from 122 to 116 us (four:
// 118, eight: 125).  Only where a lane's piece is 16-byte chunks: with two-element accesses the addresses cost more.
constexpr int QN_AHEAD = 2;
template <typename T, int V>
__device__ __forceinline__ void qn_ask(const QnRows& r, int t0, int row, int rows, int D, int lane, bool grad) {
  if constexpr (V * sizeof(T) == 16) {
    if (row >= rows || lane * (2 * V) >= D) return;
    const int tl = qn_token(r, row), h = row - tl * r.heads;
    const T* x = reinterpret_cast<const T*>(r.x) + (long)(t0 + tl) * r.x_tok + (long)h * r.x_head + lane * (2 * V);
    asm volatile("prefetch.global.L2 [%0];" ::"l"(x));
    if (grad) {
      const T* dy = reinterpret_cast<const T*>(r.dy) + (long)(t0 + tl) * r.dy_tok + (long)h * r.dy_head + lane * (2 * V);
      asm volatile("prefetch.global.L2 [%0];" ::"l"(dy));
    }
  }
}

// N consecutive elements as one access
template <typename T, int N> struct alignas(sizeof(T) * N) QnVec { T e[N]; };

// Arithmetic on a chunk, two fp32 operations per instruction: the kernels are close to bound by instructions.
__device__ __forceinline__ void qn_fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void qn_mul2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void qn_add2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
template <int V> __device__ __forceinline__ void qn_mul(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) d[0] = a[0] * b[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) qn_mul2(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
}
template <int V> __device__ __forceinline__ void qn_scale(float (&d)[V], float b) {
  if constexpr (V == 1) d[0] *= b;
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) qn_mul2(d[i], d[i + 1], d[i], d[i + 1], b, b);
}
// d = a * b + c
template <int V>
__device__ __forceinline__ void qn_fma(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) d[0] = fmaf(a[0], b[0], c[0]);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) qn_fma2(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
}
// d = a * b + d with one factor for all
template <int V> __device__ __forceinline__ void qn_axpy(float (&d)[V], const float (&a)[V], float b) {
  if constexpr (V == 1) d[0] = fmaf(a[0], b, d[0]);
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) qn_fma2(d[i], d[i + 1], a[i], a[i + 1], b, b, d[i], d[i + 1]);
}
template <int V> __device__ __forceinline__ void qn_shift(float (&d)[V], float b) {
  if constexpr (V == 1) d[0] += b;
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) qn_add2(d[i], d[i + 1], d[i], d[i + 1], b, b);
}
template <int V> __device__ __forceinline__ void qn_add(float (&d)[V], const float (&a)[V]) {
  if constexpr (V == 1) d[0] += a[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 2) qn_add2(d[i], d[i + 1], d[i], d[i + 1], a[i], a[i + 1]);
}
// sum of a * b over the chunk
template <int V> __device__ __forceinline__ float qn_dot(const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) return a[0] * b[0];
  else {
    float s0, s1;
    qn_mul2(s0, s1, a[0], a[1], b[0], b[1]);
#pragma unroll
    for (int i = 2; i < V; i += 2) qn_fma2(s0, s1, a[i], a[i + 1], b[i], b[i + 1], s0, s1);
    return s0 + s1;
  }
}
template <int V> __device__ __forceinline__ float qn_total(const float (&a)[V]) {
  if constexpr (V == 1) return a[0];
  else {
    float s0 = a[0], s1 = a[1];
#pragma unroll
    for (int i = 2; i < V; i += 2) qn_add2(s0, s1, s0, s1, a[i], a[i + 1]);
    return s0 + s1;
  }
}
// A chunk of eight 16-bit elements lies in registers as its four even elements and then its four odd ones: the halves of a
// 32-bit word are taken apart anyway, and the rotation of interleaved pairs becomes packed arithmetic.
template <int V> __device__ __forceinline__ constexpr int qn_reg(int e) { return V == 8 ? (e >> 1) + (e & 1) * 4 : e; }
template <int V> __device__ __forceinline__ constexpr int qn_elem(int r) { return V == 8 ? (r & 3) * 2 + (r >> 2) : r; }
template <typename T, int V> __device__ __forceinline__ void qn_unpack(const QnVec<T, V>& v, float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = sb::to_f(v.e[qn_elem<V>(i)]);
}
template <typename T, int V> __device__ __forceinline__ void qn_pack(const float (&f)[V], QnVec<T, V>& v) {
  if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        *reinterpret_cast<__nv_bfloat162*>(&v.e[i]) = __floats2bfloat162_rn(f[qn_reg<V>(i)], f[qn_reg<V>(i + 1)]);
      else
        *reinterpret_cast<__half2*>(&v.e[i]) = __floats2half2_rn(f[qn_reg<V>(i)], f[qn_reg<V>(i + 1)]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v.e[i] = sb::from_f<T>(f[qn_reg<V>(i)]);
  }
}

// What a lane holds of a row: NP pairs of chunks of V elements.  Pair p of lane l is number c = l + p G:
//   rotate-half and c < rot / (2 V): A = c, B = c + rot / (2 V); otherwise A = 2 c, B = 2 c + 1.
template <int V> struct QnChunks {
  int a, b;
  __device__ __forceinline__ QnChunks(int c, int rot, int interleaved) {
    const int half = rot / (2 * V);
    const bool split = !interleaved && c < half;
    a = split ? c : 2 * c;
    b = split ? c + half : 2 * c + 1;
  }
};

// Place of the cosine of angle i (< V; of the register for rotate-half) of pair c in the table of one token, in floats.  A 16-byte word holds the cosines and
// then the sines of two neighbours, consecutive lanes touch consecutive words (no bank conflicts); np = pairs per row that
// the table covers.  The sine lies qn_sine<V>() behind.
template <int V> __device__ __forceinline__ int qn_table_slot(int c, int i, int np) {
  return V == 1 ? 2 * c : (((i >> 1) * np + c) << 2) + (i & 1);
}
template <int V> __device__ __forceinline__ constexpr int qn_sine() { return V == 1 ? 1 : 2; }
// Place of element e of a weight vector in shared memory: four consecutive registers stay together, chunks interleave.
template <int V> __device__ __forceinline__ int qn_weight_slot(int e, int chunks) {
  if (V < 4) return e;
  const int c = e / V, j = qn_reg<V>(e % V);
  return ((j >> 2) * chunks + c) * 4 + (j & 3);
}

template <int V> __device__ __forceinline__ void qn_read_weights(const float* s, int chunk, int chunks, float (&w)[V]) {
  if constexpr (V < 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = s[chunk * V + i];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(s + ((i >> 2) * chunks + chunk) * 4);
      w[i] = t.x; w[i + 1] = t.y; w[i + 2] = t.z; w[i + 3] = t.w;
    }
  }
}

// Rotation of a chunk pair by the table's angles, BACK: the transposed one.
template <int V, bool BACK>
__device__ __forceinline__ void qn_rotate(float (&a)[V], float (&b)[V], const float* tbl, int c, int np, int rot,
                                          int interleaved) {
  if constexpr (V == 1) {  // both conventions: the pair is (a, b)
    if (c < (rot >> 1)) {
      const float cs = tbl[2 * c], sn = BACK ? -tbl[2 * c + 1] : tbl[2 * c + 1], x = a[0], y = b[0];
      a[0] = x * cs - y * sn;
      b[0] = y * cs + x * sn;
    }
  } else {
    if (c * 2 * V >= rot) return;  // neither chunk is rotated (rotate-half: c >= rot / (2 V) is the same test)
    float cs[V], sn[V];
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float4 u = *reinterpret_cast<const float4*>(tbl + ((i >> 1) * np + c) * 4);
      cs[i] = u.x;
      cs[i + 1] = u.y;
      sn[i] = BACK ? -u.z : u.z;
      sn[i + 1] = BACK ? -u.w : u.w;
    }
    if (!interleaved) {
      float x[V], ns[V];
      qn_mul<V>(x, a, sn);  // the part of b that comes from a
#pragma unroll
      for (int i = 0; i < V; ++i) ns[i] = -sn[i];
      qn_mul<V>(a, a, cs);
      qn_fma<V>(a, b, ns, a);
      qn_fma<V>(b, b, cs, x);
    } else {
      constexpr int E = V / 2;
      auto turn = [&](float (&z)[V], int i, int j) {
        const int at = qn_reg<V>(2 * i), to = qn_reg<V>(2 * i + 1);
        const float x = z[at], y = z[to];
        z[at] = x * cs[j] - y * sn[j];
        z[to] = y * cs[j] + x * sn[j];
      };
      if (V == 8 && rot % (2 * V) == 0) {  // whole chunks, even and odd elements side by side
        auto turn2 = [&](float (&z)[V], int i, int j) {
          float t0, t1;
          qn_mul2(t0, t1, z[i], z[i + 1], sn[j], sn[j + 1]);
          qn_mul2(z[i], z[i + 1], z[i], z[i + 1], cs[j], cs[j + 1]);
          qn_fma2(z[i], z[i + 1], z[E + i], z[E + i + 1], -sn[j], -sn[j + 1], z[i], z[i + 1]);
          qn_fma2(z[E + i], z[E + i + 1], z[E + i], z[E + i + 1], cs[j], cs[j + 1], t0, t1);
        };
#pragma unroll
        for (int i = 0; i < E; i += 2) {
          turn2(a, i, i);
          turn2(b, i, E + i);
        }
      } else if (rot % (2 * V) == 0) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          turn(a, i, i);
          turn(b, i, V / 2 + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          if (2 * c * V + 2 * i < rot) turn(a, i, i);
          if ((2 * c + 1) * V + 2 * i < rot) turn(b, i, V / 2 + i);
        }
      }
    }
  }
}

// LG >= 0: a row is exactly 2^LG lanes with both chunks, known when compiling (heads of 64 and 128); else anything.
// Sum over the g lanes of a row.
template <int LG> __device__ __forceinline__ float qn_group_sum(float v, int g) {
  if constexpr (LG >= 0) {
#pragma unroll
    for (int o = (1 << LG) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
    for (int o = g >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

// Sines and cosines of a tile's tokens; positions come from `spos`.
template <int V>
__device__ __forceinline__ void qn_fill_table(const QnParams& p, float* tbl, const int* spos, int n_tok, int np) {
  const int angles = p.rot >> 1;
  for (int i = threadIdx.x; i < n_tok * angles; i += QN_THREADS) {
    const int t = i / angles, a = i - t * angles;
    const double turns = (double)spos[t] * p.turns[a];
    const float rest = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.f * rest, &s, &c);
    float* at = tbl + t * np * V * 2 + qn_table_slot<V>(a / V, p.interleaved ? a % V : qn_reg<V>(a % V), np);
    at[0] = c;
    at[qn_sine<V>()] = s;
  }
}

// Takes the mean off x (not for RMS) and returns the reciprocal deviation r.  x is held as NP pairs; chunks beyond the row
// (ha / hb false) hold zeros and keep them.
template <int V, int NP, int LG>
__device__ __forceinline__ float qn_stats(float (&a)[NP][V], float (&b)[NP][V], const bool (&ha)[NP], const bool (&hb)[NP],
                                          float inv_d, int rms, float eps, int g) {
  if (!rms) {
    float s = 0.f;
#pragma unroll
    for (int p = 0; p < NP; ++p) s += qn_total<V>(a[p]) + qn_total<V>(b[p]);
    const float mu = qn_group_sum<LG>(s, g) * inv_d;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if (ha[p]) qn_shift<V>(a[p], -mu);
      if (hb[p]) qn_shift<V>(b[p], -mu);
    }
  }
  float ss = 0.f;  // around the mean, from registers: no cancellation
#pragma unroll
  for (int p = 0; p < NP; ++p) ss += qn_dot<V>(a[p], a[p]) + qn_dot<V>(b[p], b[p]);
  return rsqrtf(fmaf(qn_group_sum<LG>(ss, g), inv_d, eps));
}

// ============================================================================ forward
// One CTA per tile of tokens.  PAGED: k and v go to their slots of the cache, positions come from the sequence lengths.
template <typename T, int V, int NP, int LG, bool PAGED>
__global__ void __launch_bounds__(QN_THREADS, QN_FWD_BLOCKS) qn_fwd_kernel(const __grid_constant__ QnParams p) {
  extern __shared__ __align__(16) float smem[];
  using Vec = QnVec<T, V>;
  const int D = p.D, chunks = (D + V - 1) / V, np = (p.rot + 2 * V - 1) / (2 * V);
  float* sw = smem;                                     // q weight, q bias, k weight, k bias
  float* tbl = smem + 4 * QN_MAX_D;
  __shared__ int spos[QN_MAX_SLOTS];
  __shared__ int spage[QN_MAX_SLOTS], sslot[QN_MAX_SLOTS];  // spage -1: nothing to write, -2: behind the last sequence
  const int t0 = blockIdx.x * p.tile, n_tok = min(p.tile, p.T - t0);
  const int log_g = LG >= 0 ? LG : p.log_g, g = 1 << log_g, lane = threadIdx.x & (g - 1), grp = threadIdx.x >> log_g;
  const int n_grp = QN_THREADS >> log_g;
  const float inv_d = 1.f / D;

  for (int i = threadIdx.x; i < D; i += QN_THREADS) {
    const int s = qn_weight_slot<V>(i, chunks);
    if (p.q.w) sw[s] = qn_load_any(p.q.w, i, p.w_dtype);
    if (p.q.b) sw[QN_MAX_D + s] = qn_load_any(p.q.b, i, p.w_dtype);
    if (p.k.w) sw[2 * QN_MAX_D + s] = qn_load_any(p.k.w, i, p.w_dtype);
    if (p.k.b) sw[3 * QN_MAX_D + s] = qn_load_any(p.k.b, i, p.w_dtype);
  }
  if (threadIdx.x < n_tok) {
    const int t = t0 + threadIdx.x;
    if constexpr (PAGED) {
      int lo = 0, hi = p.batch;  // first b with cu[b + 1] > t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.cu[mid + 1] > t) hi = mid; else lo = mid + 1;
      }
      int page = -2, slot = 0, at = 0;
      if (lo < p.batch && p.cu[lo] <= t) {
        const long long pos = (long long)p.lens[lo] - p.cu[lo + 1] + t;  // the new tokens are the sequence's last
        page = -1;
        if (pos >= 0 && (pos >> p.page_shift) < p.cols) {
          const int id = p.table[lo * p.table_ld + (pos >> p.page_shift)];
          if (id >= 0 && id < p.num_pages) page = id;
          slot = (int)(pos & ((1 << p.page_shift) - 1));
          at = (int)pos;
        }
        if (page < 0) *p.status = SB_ERR_BAD_ARG;  // the token has no place in the cache: reported, nothing written
      }
      spage[threadIdx.x] = page;
      sslot[threadIdx.x] = slot;
      spos[threadIdx.x] = p.pos ? p.pos[t] : at;
    } else {
      spos[threadIdx.x] = p.pos ? p.pos[t] : 0;
    }
  } else if (PAGED && blockIdx.x == 0 && threadIdx.x >= QN_MAX_SLOTS) {  // threads without a token
    for (int b = threadIdx.x - QN_MAX_SLOTS; b < p.batch; b += QN_THREADS - QN_MAX_SLOTS)
      if (p.cu[b] < 0 || p.cu[b + 1] < p.cu[b] || p.cu[b + 1] > p.T) *p.status = SB_ERR_BAD_ARG;
  }
  int ca[NP], cb[NP];
  bool ha[NP], hb[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const QnChunks<V> c(lane + i * g, p.rot, p.interleaved);
    ca[i] = c.a; cb[i] = c.b;
    ha[i] = LG >= 0 || c.a < chunks; hb[i] = LG >= 0 || c.b < chunks;
  }
  __syncthreads();
  if (p.rot) qn_fill_table<V>(p, tbl, spos, n_tok, np);
  __syncthreads();
  // The rows of q, then of k, then of v, each kind with its code (its addresses and strides are constants of the launch).
  // The loads of a round of the row groups are issued a round ahead; weights stay in registers over the rounds.
  auto all_rows = [&](auto kind_of, const QnRows& R) {
    constexpr int kind = decltype(kind_of)::value;
    const int rows = n_tok * R.heads;
    const float* ws = sw + kind * 2 * QN_MAX_D;
    const bool norm = kind < 2 && R.w;
    float w1[NP][V], w2[NP][V];
    if (norm) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (ha[i]) qn_read_weights<V>(ws, ca[i], chunks, w1[i]);
        if (hb[i]) qn_read_weights<V>(ws, cb[i], chunks, w2[i]);
      }
    }
    Vec na[NP] = {}, nb[NP] = {};  // chunks beyond the row stay zeros
    auto load = [&](int row) {
      if (row < rows) {
        const int tl = qn_token(R, row), h = row - tl * R.heads;
        const T* x = reinterpret_cast<const T*>(R.x) + (long)(t0 + tl) * R.x_tok + (long)h * R.x_head;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (ha[i]) na[i] = *reinterpret_cast<const Vec*>(x + ca[i] * V);
          if (hb[i]) nb[i] = *reinterpret_cast<const Vec*>(x + cb[i] * V);
        }
      }
    };
    load(grp);
#pragma unroll 1
    for (int base = 0; base < rows; base += n_grp) {  // the same trip count for every lane: the shuffles name all of them
      const int row = base + grp;
      const bool live = row < rows;
      const int tl = live ? qn_token(R, row) : 0, h = row - tl * R.heads;
      Vec va[NP], vb[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        va[i] = na[i];
        vb[i] = nb[i];
      }
      load(row + n_grp);
      qn_ask<T, V>(R, t0, row + QN_AHEAD * n_grp, rows, D, lane, false);
      if (norm || (kind < 2 && p.rot)) {  // else a copy, bit by bit
        float a[NP][V], b[NP][V];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          qn_unpack<T, V>(va[i], a[i]);
          qn_unpack<T, V>(vb[i], b[i]);
        }
        if (norm) {
          const float r = qn_stats<V, NP, LG>(a, b, ha, hb, inv_d, p.rms, p.eps, g);
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            qn_scale<V>(a[i], r);
            qn_scale<V>(b[i], r);
            if (R.b) {
              float t[V];
              if (ha[i]) {
                qn_read_weights<V>(ws + QN_MAX_D, ca[i], chunks, t);
                qn_fma<V>(a[i], a[i], w1[i], t);
              }
              if (hb[i]) {
                qn_read_weights<V>(ws + QN_MAX_D, cb[i], chunks, t);
                qn_fma<V>(b[i], b[i], w2[i], t);
              }
            } else {
              if (ha[i]) qn_mul<V>(a[i], a[i], w1[i]);
              if (hb[i]) qn_mul<V>(b[i], b[i], w2[i]);
            }
          }
        }
        if (p.rot) {
#pragma unroll
          for (int i = 0; i < NP; ++i)
            qn_rotate<V, false>(a[i], b[i], tbl + tl * np * V * 2, lane + i * g, np, p.rot, p.interleaved);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          qn_pack<T, V>(a[i], va[i]);
          qn_pack<T, V>(b[i], vb[i]);
        }
      }
      T* y = reinterpret_cast<T*>(R.y);
      bool store = live;
      if (PAGED && live) {
        const int page = spage[tl];
        if (kind == 0) {
          y += (long)(t0 + tl) * R.y_tok + (long)h * R.y_head;
          if (page == -2) {  // behind the last sequence: zeros
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
              for (int j = 0; j < V; ++j) va[i].e[j] = vb[i].e[j] = sb::from_f<T>(0.f);
          }
        } else {
          store = page >= 0;
          y += (long)page * (kind == 1 ? p.k_page : p.v_page) + (long)sslot[tl] * (kind == 1 ? p.k_slot : p.v_slot) +
               (long)h * R.y_head;
        }
      } else if (live) {
        y += (long)(t0 + tl) * R.y_tok + (long)h * R.y_head;
      }
      if (store) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (ha[i]) *reinterpret_cast<Vec*>(y + ca[i] * V) = va[i];
          if (hb[i]) *reinterpret_cast<Vec*>(y + cb[i] * V) = vb[i];
        }
      }
    }
  };
  all_rows(std::integral_constant<int, 0>(), p.q);
  all_rows(std::integral_constant<int, 1>(), p.k);
  if constexpr (PAGED) all_rows(std::integral_constant<int, 2>(), p.v);
}

// ============================================================================ backward
// A block takes either q or k, walks over tiles of tokens and keeps its share of dw and db in registers (each lane owns
// the same chunks in every row); the block's sums go to one row of `partial`, added up in a fixed order afterwards.
// RMS: no mean, and no biases whose gradients would have to be kept.
template <typename T, int V, int NP, int LG, bool RMS>
__device__ __forceinline__ void qn_bwd_rows(const QnParams& p, const QnRows& R, const int blk, const int n_blk,
                                            const int per_tile) {
  extern __shared__ __align__(16) float smem[];
  using Vec = QnVec<T, V>;
  const int D = p.D, chunks = (D + V - 1) / V, np = (p.rot + 2 * V - 1) / (2 * V);
  float* sw = smem;
  float* tbl = smem + QN_MAX_D;
  __shared__ int spos[QN_MAX_SLOTS];
  const int log_g = LG >= 0 ? LG : p.log_g, g = 1 << log_g, lane = threadIdx.x & (g - 1), grp = threadIdx.x >> log_g;
  const int n_grp = QN_THREADS >> log_g;
  const float inv_d = 1.f / D;
  for (int i = threadIdx.x; i < D; i += QN_THREADS) sw[qn_weight_slot<V>(i, chunks)] = qn_load_any(R.w, i, p.w_dtype);
  int ca[NP], cb[NP];
  bool ha[NP], hb[NP];
  float dwa[NP][V], dwb[NP][V], dba[NP][V], dbb[NP][V];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const QnChunks<V> c(lane + i * g, p.rot, p.interleaved);
    ca[i] = c.a; cb[i] = c.b;
    ha[i] = LG >= 0 || c.a < chunks; hb[i] = LG >= 0 || c.b < chunks;
#pragma unroll
    for (int j = 0; j < V; ++j) dwa[i][j] = dwb[i][j] = dba[i][j] = dbb[i][j] = 0.f;
  }
  const int tiles = (p.T + per_tile - 1) / per_tile;
#pragma unroll 1
  for (int tile = blk; tile < tiles; tile += n_blk) {
    const int t0 = tile * per_tile, n_tok = min(per_tile, p.T - t0);
    const int rows = n_tok * R.heads, iters = (rows + n_grp - 1) / n_grp;
    Vec na[NP] = {}, nb[NP] = {}, ma[NP] = {}, mb[NP] = {};  // x and dy of the next round; zeros beyond the row
    auto load = [&](int row) {
      if (row < rows) {
        const int tl = qn_token(R, row), h = row - tl * R.heads;
        const T* x = reinterpret_cast<const T*>(R.x) + (long)(t0 + tl) * R.x_tok + (long)h * R.x_head;
        const T* dy = reinterpret_cast<const T*>(R.dy) + (long)(t0 + tl) * R.dy_tok + (long)h * R.dy_head;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (ha[i]) {
            na[i] = *reinterpret_cast<const Vec*>(x + ca[i] * V);
            ma[i] = *reinterpret_cast<const Vec*>(dy + ca[i] * V);
          }
          if (hb[i]) {
            nb[i] = *reinterpret_cast<const Vec*>(x + cb[i] * V);
            mb[i] = *reinterpret_cast<const Vec*>(dy + cb[i] * V);
          }
        }
      }
    };
    load(grp);
    __syncthreads();  // the table of the tile before is no longer read
    if (p.rot) {
      if (threadIdx.x < n_tok) spos[threadIdx.x] = p.pos[t0 + threadIdx.x];
      __syncthreads();
      qn_fill_table<V>(p, tbl, spos, n_tok, np);
    }
    __syncthreads();
#pragma unroll 1
    for (int it = 0; it < iters; ++it) {
      const int row = grp + it * n_grp;
      const bool live = row < rows;
      const int tl = live ? qn_token(R, row) : 0, h = row - tl * R.heads;
      Vec va[NP], vb[NP], ya[NP], yb[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        va[i] = na[i];
        vb[i] = nb[i];
        ya[i] = ma[i];
        yb[i] = mb[i];
      }
      if (it + 1 < iters) load(row + n_grp);
      qn_ask<T, V>(R, t0, row + QN_AHEAD * n_grp, rows, D, lane, true);
      float a[NP][V], b[NP][V], da[NP][V], db[NP][V];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        qn_unpack<T, V>(va[i], a[i]);
        qn_unpack<T, V>(vb[i], b[i]);
        qn_unpack<T, V>(ya[i], da[i]);
        qn_unpack<T, V>(yb[i], db[i]);
      }
      if (p.rot) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
          qn_rotate<V, true>(da[i], db[i], tbl + tl * np * V * 2, lane + i * g, np, p.rot, p.interleaved);
      }
      const float r = qn_stats<V, NP, LG>(a, b, ha, hb, inv_d, RMS, p.eps, g);
      float s1 = 0.f, s2 = 0.f;  // sums of g and of g * xhat
      const bool keep = live;    // a group without a row works on what it loaded last (or zeros): it must not count
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        float w[V];
        auto chunk = [&](float (&x)[V], float (&dy)[V], float (&dw)[V], float (&dbias)[V], int c) {
          qn_scale<V>(x, r);
          if (keep) {
            qn_fma<V>(dw, dy, x, dw);
            if (!RMS) qn_add<V>(dbias, dy);
          }
          qn_read_weights<V>(sw, c, chunks, w);
          qn_mul<V>(dy, dy, w);
          if (!RMS) s1 += qn_total<V>(dy);
          s2 += qn_dot<V>(dy, x);
        };
        if (ha[i]) chunk(a[i], da[i], dwa[i], dba[i], ca[i]);
        if (hb[i]) chunk(b[i], db[i], dwb[i], dbb[i], cb[i]);
      }
      s2 = qn_group_sum<LG>(s2, g) * inv_d;
      s1 = RMS ? 0.f : qn_group_sum<LG>(s1, g) * inv_d;
      T* y = reinterpret_cast<T*>(R.y) + (long)(t0 + tl) * R.y_tok + (long)h * R.y_head;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (!RMS) {
          qn_shift<V>(da[i], -s1);
          qn_shift<V>(db[i], -s1);
        }
        qn_axpy<V>(da[i], a[i], -s2);
        qn_axpy<V>(db[i], b[i], -s2);
        qn_scale<V>(da[i], r);
        qn_scale<V>(db[i], r);
        qn_pack<T, V>(da[i], va[i]);
        qn_pack<T, V>(db[i], vb[i]);
        if (live && ha[i]) *reinterpret_cast<Vec*>(y + ca[i] * V) = va[i];
        if (live && hb[i]) *reinterpret_cast<Vec*>(y + cb[i] * V) = vb[i];
      }
    }
  }
  if (!p.partial) return;
  // sums over the row groups of a warp, then over the warps, in a fixed order
  float* red = smem;  // [warps][2][QN_MAX_D], after the last use of weights and table
  __syncthreads();
  const int warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      for (int o = g; o < 32; o <<= 1) {
        dwa[i][j] += __shfl_xor_sync(0xffffffffu, dwa[i][j], o);
        dwb[i][j] += __shfl_xor_sync(0xffffffffu, dwb[i][j], o);
        if (!RMS) {
          dba[i][j] += __shfl_xor_sync(0xffffffffu, dba[i][j], o);
          dbb[i][j] += __shfl_xor_sync(0xffffffffu, dbb[i][j], o);
        }
      }
      if ((threadIdx.x & 31) < g) {
        float* dst = red + warp * 2 * QN_MAX_D;
        const int ea = ca[i] * V + qn_elem<V>(j), eb = cb[i] * V + qn_elem<V>(j);
        if (ha[i]) { dst[ea] = dwa[i][j]; dst[QN_MAX_D + ea] = dba[i][j]; }
        if (hb[i]) { dst[eb] = dwb[i][j]; dst[QN_MAX_D + eb] = dbb[i][j]; }
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += QN_THREADS) {
    const int which = i >= D, e = which ? i - D : i;
    float s = 0.f;
    for (int wp = 0; wp < QN_THREADS / 32; ++wp) s += red[wp * 2 * QN_MAX_D + which * QN_MAX_D + e];
    p.partial[(size_t)blockIdx.x * 2 * D + i] = s;
  }
}

template <typename T, int V, int NP, int LG, bool RMS>
__global__ void __launch_bounds__(QN_THREADS, 2) qn_bwd_kernel(const __grid_constant__ QnParams p) {
  // code of its own for q and for k: addresses and strides are constants of the launch
  if ((int)blockIdx.x < p.q_blocks) qn_bwd_rows<T, V, NP, LG, RMS>(p, p.q, blockIdx.x, p.q_blocks, p.tile);
  else qn_bwd_rows<T, V, NP, LG, RMS>(p, p.k, blockIdx.x - p.q_blocks, gridDim.x - p.q_blocks, p.tile_k);
}

// Sums of the blocks' partial rows: blockIdx.y = 0 q, 1 k; 32 columns per block (of 2 D: dw then db), 32 row lanes.
template <typename W>
__global__ void __launch_bounds__(1024) qn_bwd_sum_kernel(const float* __restrict__ partial, int D, int q_blocks,
                                                          int blocks, W* dwq, W* dbq, W* dwk, W* dbk, int accumulate) {
  __shared__ float red[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  const int b0 = blockIdx.y ? q_blocks : 0, b1 = blockIdx.y ? blocks : q_blocks;
  float s = 0.f;
  if (col < 2 * D)
    for (int b = b0 + threadIdx.y; b < b1; b += 32) s += partial[(size_t)b * 2 * D + col];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sb::warp_sum(red[threadIdx.x][threadIdx.y]);  // warp y sums column y of this block
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < 2 * D) {
    W* dst = blockIdx.y ? (c < D ? dwk : dbk) : (c < D ? dwq : dbq);
    const int e = c < D ? c : c - D;
    if (dst) dst[e] = sb::from_f<W>(accumulate ? sb::to_f(dst[e]) + s : s);
  }
}

int qn_log_lanes(int pairs, int cap) {
  int l = 0;
  while ((1 << l) < pairs && (1 << l) < cap) ++l;
  return l;
}
// Bytes (a power of two up to 16) that divide every address of the rows.
long qn_align(const QnRows& r, int es) {
  if (r.heads == 0) return 16;
  const uintptr_t all = reinterpret_cast<uintptr_t>(r.x) | reinterpret_cast<uintptr_t>(r.y) | reinterpret_cast<uintptr_t>(r.dy) |
                        (uintptr_t)((r.x_tok | r.x_head | r.y_tok | r.y_head | r.dy_tok | r.dy_head) * es) | 16;
  return (long)(all & -all);
}

// Fills in what follows from the sizes; returns the elements V that a lane moves at once: 16 bytes where all rows are so
// aligned and, for rotate-half, the rotated half is whole chunks; else 2 elements; else 1 (2999 tokens x 41 heads of 80 in
// fp32, 20 dimensions rotated, forward and backward: 1152 us with V = 1, 143 us with V = 2).
int qn_plan(QnParams* p, int es, long align, double base) {
  auto fits = [&](int v) {
    return align >= (long)v * es && p->D % v == 0 && (p->rot == 0 || (p->interleaved ? v % 2 == 0 : (p->rot / 2) % v == 0));
  };
  const int V = fits(16 / es) ? 16 / es : fits(2) ? 2 : 1;
  const int chunks = (p->D + V - 1) / V, pairs = (chunks + 1) / 2;
  p->log_g = qn_log_lanes(pairs, 32);
  for (QnRows* r : {&p->q, &p->k, &p->v}) r->inv = r->heads ? (uint32_t)((1UL << 32) / r->heads + 1) : 0;
  // every eighth by pow, the others as products of at most seven factors: off by a few 2^-53, and a call takes 2 us less
  const double step = p->rot ? pow(base, -2.0 / p->rot) : 1.0;
  for (int i = 0; i < p->rot / 2; ++i)
    p->turns[i] = i % 8 ? p->turns[i - 1] * step : pow(base, -2.0 * i / p->rot) / 6.283185307179586476925;
  return V;
}
int qn_table_bytes_per_token(const QnParams& p, int V) { return p.rot ? ((p.rot + 2 * V - 1) / (2 * V)) * V * 8 : 0; }

}  // namespace

static int qn_check(const QnParams& p, int dtype) {
  if (dtype != SB_DT_F32 && dtype != SB_DT_BF16 && dtype != SB_DT_F16) return SB_ERR_BAD_ARG;
  if (p.w_dtype != SB_DT_F32 && p.w_dtype != SB_DT_BF16 && p.w_dtype != SB_DT_F16) return SB_ERR_BAD_ARG;
  if (p.D < 1 || p.T < 0 || p.q.heads < 0 || p.k.heads < 0) return SB_ERR_BAD_ARG;
  // the division by the head count is exact below 2^32 / heads rows, a tile has at most 64 heads of them
  if (p.D > QN_MAX_D || p.q.heads > 8000 || p.k.heads > 8000) return SB_ERR_TOO_LARGE;
  if (p.rot < 0 || p.rot % 2 || p.rot > p.D) return SB_ERR_BAD_ARG;
  return SB_OK;
}

template <typename T>
static int qn_launch_fwd(QnParams& p, bool paged, long align, double base, int sms, cudaStream_t stream) {
  const int V = qn_plan(&p, sizeof(T), align, base);
  constexpr int VF = 16 / sizeof(T);
  const int per_tok = qn_table_bytes_per_token(p, V);
  // Tokens per CTA: the launch is one wave where the table has room for that many, so that the weights, the table and
  // their barriers are paid once per CTA.
  int tile = (int)((p.T + (long)QN_FWD_BLOCKS * sms - 1) / ((long)QN_FWD_BLOCKS * sms));
  if (tile > QN_MAX_SLOTS) tile = QN_MAX_SLOTS;
  if (per_tok && tile > QN_TABLE_BYTES / per_tok) tile = QN_TABLE_BYTES / per_tok;
  p.tile = tile;
  const int smem = 4 * QN_MAX_D * 4 + tile * per_tok;
  const int grid = (p.T + tile - 1) / tile;
  const bool exact = V == VF && p.D == 2 * V << p.log_g;
  auto launch = [&](auto paged_form) {
    constexpr bool PAGED = decltype(paged_form)::value;
    if (exact && p.log_g == 2) qn_fwd_kernel<T, VF, 1, 2, PAGED><<<grid, QN_THREADS, smem, stream>>>(p);
    else if (exact && p.log_g == 3) qn_fwd_kernel<T, VF, 1, 3, PAGED><<<grid, QN_THREADS, smem, stream>>>(p);
    else if (V == VF) qn_fwd_kernel<T, VF, 1, -1, PAGED><<<grid, QN_THREADS, smem, stream>>>(p);
    else if (V == 2) qn_fwd_kernel<T, 2, 2, -1, PAGED><<<grid, QN_THREADS, smem, stream>>>(p);
    else qn_fwd_kernel<T, 1, 4, -1, PAGED><<<grid, QN_THREADS, smem, stream>>>(p);
  };
  if (paged) launch(std::true_type());
  else launch(std::false_type());
  SB_CHECK_LAUNCH();
  return SB_OK;
}

// q_out / k_out [T, heads, D] = rotated norms of q and k (token and head strides in elements, innermost stride 1).
// Null weights: no norm.  pos: int32 [T], needed when rot > 0.  base: of the rotary frequencies.
SB_API int sb200_qk_norm_rope_fwd(const void* q, const void* k, void* q_out, void* k_out, const void* q_w,
                                  const void* k_w, const void* q_b, const void* k_b, const int* pos, int T, int Hq,
                                  int Hk, int D, long q_tok, long q_head, long k_tok, long k_head, float eps, int rms,
                                  int rot, double base, int interleaved, int dtype, int w_dtype, int sms,
                                  cudaStream_t stream) {
  QnParams p = {};
  p.q = {q, q_out, nullptr, q_w, q_b, q_tok, q_head, (long)Hq * D, D, 0, 0, Hq};
  p.k = {k, k_out, nullptr, k_w, k_b, k_tok, k_head, (long)Hk * D, D, 0, 0, Hk};
  p.pos = pos; p.T = T; p.D = D; p.rot = rot; p.interleaved = interleaved; p.rms = rms; p.w_dtype = w_dtype; p.eps = eps;
  if (int rc = qn_check(p, dtype)) return rc;
  if (rot && (!pos || !(base > 0.0))) return SB_ERR_BAD_ARG;
  if (T == 0 || Hq + Hk == 0) return SB_OK;
  const int es = dtype == SB_DT_F32 ? 4 : 2;
  const long align = std::min(qn_align(p.q, es), qn_align(p.k, es));
  SB_DISPATCH_DTYPE(dtype, E, { return qn_launch_fwd<E>(p, false, align, base, sms, stream); });
  return SB_OK;
}

// The paged form.  Row t belongs to the sequence b with cu[b] <= t < cu[b + 1]; its position is
// lens[b] - cu[b + 1] + t, and k / v go to row pos % page_size of page table[b][pos / page_size] of the caches
// [num_pages, page_size, Hk, D] (page, row and head strides in elements, page_size a power of two).  A position outside
// the table or a page outside the cache writes nothing and sets *status, as do sequences that do not follow one another
// inside the T rows.  Rows behind the last sequence give zeros in
// q_out and touch no page.  pos may override the rotation angles; q may be null (Hq = 0).
SB_API int sb200_paged_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache,
                              const void* q_w, const void* k_w, const void* q_b, const void* k_b, const int* pos,
                              const int* table, const int* cu, const int* lens, int T, int batch, int Hq, int Hk, int D,
                              long q_tok, long q_head, long k_tok, long k_head, long v_tok, long v_head, long k_page,
                              long k_slot, long kc_head, long v_page, long v_slot, long vc_head, long table_ld,
                              int cols, int num_pages, int page_size, float eps, int rms, int rot, double base,
                              int interleaved, int dtype, int w_dtype, int sms, int* status, cudaStream_t stream) {
  QnParams p = {};
  p.q = {q, q_out, nullptr, q_w, q_b, q_tok, q_head, (long)Hq * D, D, 0, 0, Hq};
  p.k = {k, k_cache, nullptr, k_w, k_b, k_tok, k_head, 0, kc_head, 0, 0, Hk};
  p.v = {v, v_cache, nullptr, nullptr, nullptr, v_tok, v_head, 0, vc_head, 0, 0, Hk};
  p.pos = pos; p.T = T; p.D = D; p.rot = rot; p.interleaved = interleaved; p.rms = rms; p.w_dtype = w_dtype; p.eps = eps;
  if (int rc = qn_check(p, dtype)) return rc;
  if (batch < 0 || cols < 0 || num_pages < 0 || page_size < 1 || (page_size & (page_size - 1)) || !status || Hk < 1)
    return SB_ERR_BAD_ARG;
  if (rot && !(base > 0.0)) return SB_ERR_BAD_ARG;
  if (T == 0) return SB_OK;
  p.table = table; p.cu = cu; p.lens = lens; p.table_ld = table_ld; p.batch = batch; p.cols = cols;
  p.num_pages = num_pages; p.status = status;
  p.k_page = k_page; p.k_slot = k_slot; p.v_page = v_page; p.v_slot = v_slot;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  const int es = dtype == SB_DT_F32 ? 4 : 2;
  const uintptr_t slots = (uintptr_t)((k_page | k_slot | v_page | v_slot) * es) | 16;
  const long align = std::min({qn_align(p.q, es), qn_align(p.k, es), qn_align(p.v, es), (long)(slots & -slots)});
  SB_DISPATCH_DTYPE(dtype, E, { return qn_launch_fwd<E>(p, true, align, base, sms, stream); });
  return SB_OK;
}

// Blocks of the backward launch = rows of its workspace (2 D floats each).
SB_API int sb200_qk_norm_rope_bwd_blocks(int T, int sms) {
  const long want = 2L * sms;
  return (int)(want < T ? (want < 2 ? 2 : want) : (T < 2 ? 2 : T));
}

template <typename T>
static int qn_launch_bwd(QnParams& p, long align, double base, int blocks, cudaStream_t stream) {
  const int V = qn_plan(&p, sizeof(T), align, base);
  constexpr int VF = 16 / sizeof(T);
  const int per_tok = qn_table_bytes_per_token(p, V);
  // blocks shared out by rows, at least one each
  int qb = (int)(((long)blocks * p.q.heads + (p.q.heads + p.k.heads) / 2) / (p.q.heads + p.k.heads));
  p.q_blocks = qb < 1 ? 1 : qb > blocks - 1 ? blocks - 1 : qb;
  // Each block takes its tokens in as few and as even tiles as the table allows.
  int cap = QN_MAX_SLOTS;
  if (per_tok && cap > QN_TABLE_BYTES / per_tok) cap = QN_TABLE_BYTES / per_tok;
  auto even = [&](int n_blocks) {
    const int mine = (p.T + n_blocks - 1) / n_blocks, tiles = (mine + cap - 1) / cap;
    return (mine + tiles - 1) / tiles;
  };
  p.tile = even(p.q_blocks);
  p.tile_k = even(blocks - p.q_blocks);
  const int tile = p.tile > p.tile_k ? p.tile : p.tile_k;
  int smem = QN_MAX_D * 4 + tile * per_tok;
  const int red = (QN_THREADS / 32) * 2 * QN_MAX_D * 4;
  if (smem < red) smem = red;
  const bool exact = V == VF && p.D == 2 * V << p.log_g;
  auto launch = [&](auto rms_form) {
    constexpr bool RMS = decltype(rms_form)::value;
    if (exact && p.log_g == 2) qn_bwd_kernel<T, VF, 1, 2, RMS><<<blocks, QN_THREADS, smem, stream>>>(p);
    else if (exact && p.log_g == 3) qn_bwd_kernel<T, VF, 1, 3, RMS><<<blocks, QN_THREADS, smem, stream>>>(p);
    else if (V == VF) qn_bwd_kernel<T, VF, 1, -1, RMS><<<blocks, QN_THREADS, smem, stream>>>(p);
    else if (V == 2) qn_bwd_kernel<T, 2, 2, -1, RMS><<<blocks, QN_THREADS, smem, stream>>>(p);
    else qn_bwd_kernel<T, 1, 4, -1, RMS><<<blocks, QN_THREADS, smem, stream>>>(p);
  };
  if (p.rms) launch(std::true_type());
  else launch(std::false_type());
  SB_CHECK_LAUNCH();
  return SB_OK;
}

// dq / dk [T, heads, D] (contiguous) from d_q_out / d_k_out and the inputs; dwq .. dbk (any may be null) in w_dtype,
// written, or added to with accumulate.  partial: [blocks, 2 D] floats, or null when no weight gradient is wanted;
// blocks as sb200_qk_norm_rope_bwd_blocks says.
SB_API int sb200_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k, const void* q_w,
                                  const void* k_w, const int* pos, void* dq, void* dk, void* dwq, void* dwk, void* dbq,
                                  void* dbk, float* partial, int blocks, int T, int Hq, int Hk, int D, long dqo_tok,
                                  long dqo_head, long dko_tok, long dko_head, long q_tok, long q_head, long k_tok,
                                  long k_head, float eps, int rms, int rot, double base, int interleaved,
                                  int accumulate, int dtype, int w_dtype, cudaStream_t stream) {
  QnParams p = {};
  p.q = {q, dq, dq_out, q_w, nullptr, q_tok, q_head, (long)Hq * D, D, dqo_tok, dqo_head, Hq};
  p.k = {k, dk, dk_out, k_w, nullptr, k_tok, k_head, (long)Hk * D, D, dko_tok, dko_head, Hk};
  p.pos = pos; p.T = T; p.D = D; p.rot = rot; p.interleaved = interleaved; p.rms = rms; p.w_dtype = w_dtype; p.eps = eps;
  p.partial = partial;
  if (int rc = qn_check(p, dtype)) return rc;
  if ((rot && (!pos || !(base > 0.0))) || !q_w || !k_w || T < 1 || Hq < 1 || Hk < 1 || blocks < 2) return SB_ERR_BAD_ARG;
  const int es = dtype == SB_DT_F32 ? 4 : 2;
  const long align = std::min(qn_align(p.q, es), qn_align(p.k, es));
  int rc = SB_ERR_BAD_ARG;
  SB_DISPATCH_DTYPE(dtype, E, { rc = qn_launch_bwd<E>(p, align, base, blocks, stream); });
  if (rc || !partial) return rc;
  SB_DISPATCH_DTYPE(w_dtype, W, {
    qn_bwd_sum_kernel<W><<<dim3((2 * D + 31) / 32, 2), dim3(32, 32), 0, stream>>>(
        partial, D, p.q_blocks, blocks, (W*)dwq, (W*)dbq, (W*)dwk, (W*)dbk, accumulate);
  });
  SB_CHECK_LAUNCH();
  return SB_OK;
}
