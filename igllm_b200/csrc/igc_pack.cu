// igc_pack.cu - the key/value cache held in 4 bits: rows written to it and
// read back, and attention over its codes.
//
// Storage.  For each (slot, key/value head, position) `size` columns in
// groups of 32.  A group of values x has one f16 scale and 32 codes,
//
//   scale = f16(min(max|x| / 7, 8188)),  code = clamp(rint(x / scale), -8, 7) + 8,
//
// two codes a byte, low nibble first, and reads back as (code - 8) * scale:
// 0.5625 bytes a value, the form of the library's 4-bit weights.  The cap on
// the scale keeps 8 * scale within f16 (65504), so a decoded value always is;
// larger magnitudes and infinities saturate and a NaN stores 0, so that the
// cache never holds a value that a masked weight of 0 would turn into a NaN.
//
// Attention of row i of a sequence at p = fill + i, a query q of one of the
// `group` heads that share a key/value head:
//
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q.k_j - max),
//   j in [0, p], with a window only j > p - window or j < sinks.
//
// Rows at negative positions are padding: not written, and zeros out.
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>

#include "igc_device.cuh"
#include "igc_pack.h"

namespace igc {

// ---------------------------------------------------------------------------
// the rows of a call

struct SeqAt {
  int first, n, fill, slot;  // n 0: not to be run; slot -1: outside the cache
};

__device__ __forceinline__ void pack_trouble(const PackView &c) {
  if (c.trouble) atomicOr(c.trouble, 1);
}

__device__ __forceinline__ SeqAt seq_at(const PackView &c, const PackRows &r, int s) {
  SeqAt q;
  int a = s * r.per, b = a + r.per;
  if (r.starts) {
    a = r.starts[s];
    b = r.starts[s + 1];
  }
  const bool bad = a < 0 || b < a || b > r.rows || b - a > r.most;
  q.first = bad ? 0 : a;
  q.n = bad ? 0 : b - a;
  q.fill = min(max(r.fill[s], -(1 << 30)), 1 << 30);
  q.slot = r.slots ? r.slots[s] : s;
  if (q.slot < 0 || q.slot >= c.slots) q.slot = -1;
  if (bad) pack_trouble(c);
  return q;
}

// The sequence that holds `row`, or -1: the last whose rows start at or
// before it, if they reach it.
__device__ __forceinline__ int seq_of_row(const PackRows &r, int row) {
  if (!r.starts) return row / r.per;
  int lo = 0, hi = r.count;  // starts[lo] <= row < starts[hi], where that holds at all
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (r.starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// rows of values

// Eight values at `p` (of type 1 f32, 2 f16, 3 bf16) as floats; `wide`: the
// address is a multiple of 16.
__device__ __forceinline__ void load8(const void *base, int type, size_t at, bool wide, float (&x)[8]) {
  if (type == 1) {
    const float *p = static_cast<const float *>(base) + at;
    if (wide) {
      const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
    return;
  }
  uint32_t w[4];
  const uint16_t *p = static_cast<const uint16_t *>(base) + at;
  if (wide) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (type == 2) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ void store8(void *base, int type, size_t at, bool wide, const float (&x)[8]) {
  if (type == 1) {
    float *p = static_cast<float *>(base) + at;
    if (wide) {
      reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (type == 2) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  uint16_t *p = static_cast<uint16_t *>(base) + at;
  if (wide) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[2 * i] = (uint16_t)w[i], p[2 * i + 1] = (uint16_t)(w[i] >> 16);
  }
}

// Whether every group of eight values of these rows starts on 16 bytes.
__device__ __forceinline__ bool wide_rows(const PackData &d) {
  const long per = d.type == 1 ? 4 : 8;
  return ((size_t)d.data & 15) == 0 && d.row_stride % per == 0 && d.head_stride % per == 0;
}

// ---------------------------------------------------------------------------
// write and read: one thread a code word (8 columns), four threads a group.
// Both are one pass over their rows, bound by HBM.

constexpr int PK_THREADS = 256, PK_ITEMS = 4;

struct PackIo {
  PackView c;
  PackRows r;
  PackData k, v;
};

template <bool WRITE>
__global__ void __launch_bounds__(PK_THREADS) pack_rows_kernel(PackIo a) {
  const int words = a.c.size / 8, row_words = 2 * a.c.heads * words;
  const long first = (long)blockIdx.x * (PK_THREADS * PK_ITEMS);
  const int row0 = (int)(first / row_words), rem0 = (int)(first - (long)row0 * row_words);
  const bool kwide = wide_rows(a.k), vwide = wide_rows(a.v);
  int s = -1;
  SeqAt q = {0, 0, 0, -1};
#pragma unroll
  for (int it = 0; it < PK_ITEMS; ++it) {
    const int off = rem0 + it * PK_THREADS + threadIdx.x;
    const int row = row0 + off / row_words;
    if (row >= a.r.rows) return;  // whole groups leave together: a row is a multiple of four words
    int rest = off % row_words;
    const int side = rest / (a.c.heads * words);
    rest -= side * a.c.heads * words;
    const int head = rest / words, w = rest - head * words;
    if (s < 0 || row < q.first || row >= q.first + q.n) {
      s = seq_of_row(a.r, row);
      q = seq_at(a.c, a.r, s);
    }
    if (row < q.first || row >= q.first + q.n) continue;  // no sequence's row
    const int p = q.fill + (row - q.first);
    if (p < 0) {  // padding
      if (!WRITE) {
        const float zero[8] = {};
        const PackData &d = side ? a.v : a.k;
        store8(d.data, d.type, (size_t)row * d.row_stride + (size_t)head * d.head_stride + 8 * w, side ? vwide : kwide,
               zero);
      }
      continue;
    }
    const bool out = q.slot < 0 || p >= a.c.positions;
    if (out) {
      pack_trouble(a.c);
      if (WRITE) continue;
    }
    const PackData &d = side ? a.v : a.k;
    const size_t at = (size_t)row * d.row_stride + (size_t)head * d.head_stride + 8 * w;
    const size_t place = ((size_t)(out ? 0 : q.slot) * a.c.heads + head) * a.c.positions + (out ? 0 : p);
    uint32_t *code = reinterpret_cast<uint32_t *>(side ? a.c.vc : a.c.kc) + place * words + w;
    uint16_t *scale = (side ? a.c.vs : a.c.ks) + place * (words / 4) + (w >> 2);
    float x[8];
    if (WRITE) {
      load8(d.data, d.type, at, side ? vwide : kwide, x);
      float big = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(x[i]));  // a NaN does not take part
      const uint32_t four = 0xfu << (threadIdx.x & 28);
      big = fmaxf(big, __shfl_xor_sync(four, big, 1));
      big = fmaxf(big, __shfl_xor_sync(four, big, 2));
      const __half h = __float2half_rn(fminf(__fdiv_rn(big, 7.0f), 8188.0f));
      const float step = __half2float(h);
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float n = step > 0.0f && x[i] == x[i] ? rintf(__fdiv_rn(x[i], step)) : 0.0f;
        n = fminf(fmaxf(n, -8.0f), 7.0f);
        word |= (uint32_t)((int)n + 8) << (4 * i);
      }
      *code = word;
      if ((w & 3) == 0) *scale = __half_as_ushort(h);
    } else {
      const uint32_t word = out ? 0x88888888u : *code;
      const float step = out ? 0.0f : __half2float(__ushort_as_half(*scale));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)((int)((word >> (4 * i)) & 15u) - 8) * step;
      store8(d.data, d.type, at, side ? vwide : kwide, x);
    }
  }
}

// ---------------------------------------------------------------------------
// attention over the codes on mma.sync tiles
//
// A block holds RB = 16 MT query rows of one (sequence, key/value head): row
// rr is the sequence's row rr / group, head rr % group of the group, so a
// token's heads share each tile of codes.  Four warps walk tiles of 64
// positions that cp.async brings three tiles deep:
//
//   scores  warp w takes positions 16 w .. 16 w + 15.  A code nibble n in the
//           low bits of a half is the f16 number n 2^-24 (or 16 n 2^-24 four
//           bits up, its query column kept as q / 16), exact without any
//           conversion, so a code word costs five integer instructions.  The
//           -8 of every code is the products' starting accumulator,
//           -8 sum q over the group; the group's sum times its scale is an
//           f32 multiply-add.  Which column of a group a thread's product
//           slot holds is free as long as the query fragments agree.
//   softmax the running maximum and sum per row in 32 bits; the block's
//           maximum is merged through shared memory once a tile.
//   values  warp w takes 64 of the head's columns (or, of a narrow head, a
//           share of the positions).  A value enters as f16((code - 8) scale),
//           rounded once (2^-11 at most); pairs of positions are zipped by byte
//           permutes, so codes are used as they lie, with no transpose.  A
//           thread ends with 16 consecutive columns of its rows.
//
// A query row is scaled by the power of two that puts its largest magnitude
// in [2^13, 2^14) and kept as f16, exact for bf16 and f16 rows but for
// magnitudes 2^38 below the largest.  Weights are scaled by 2^12 (the sum
// alike) and rounded to f16, 2^-11 at most each; the results are rounded to 16
// bits anyway.
// For f32 rows (SP) queries, weights and values are each kept as f16 hi and lo
// parts, the products left out (lo x lo) below f32's own rounding.

template <int HDP, int MT, bool SP>
struct PackTile {
  static constexpr int RB = 16 * MT;
  static constexpr int C = HDP / 32;                     // groups
  static constexpr int CB = HDP / 2;                     // code bytes a position
  static constexpr int NS = 3;                           // tiles in flight
  static constexpr int WC = HDP >= 256 ? 4 : HDP / 64;   // warps across the columns
  static constexpr int WP = 4 / WC;                      // warps across a tile's positions
  static constexpr int NB = HDP / 64 / WC;               // 64-column blocks a warp
  static constexpr int SCP = 72;                         // scales a group row (64 and a bank shift)
  static constexpr int PARTS = SP ? 2 : 1;
  static constexpr int QF = C * 2 * MT * 512;            // bytes of one part's query fragments
  static constexpr int OFF_QOFF = QF * PARTS;
  static constexpr int OFF_FR = OFF_QOFF + C * RB * 4;
  static constexpr int OFF_MAX = OFF_FR + RB * 4;
  static constexpr int OFF_SUM = OFF_MAX + 4 * RB * 4;
  static constexpr int PF = 4 * MT * 512;                // bytes of one part's weight fragments
  static constexpr int OFF_P = OFF_SUM + 4 * RB * 4;
  static constexpr int OFF_SC = OFF_P + PF * PARTS;      // [NS][key, value][C][SCP] f16
  static constexpr int SC_SIDE = C * SCP * 2;
  static constexpr int OFF_CODE = (OFF_SC + NS * 2 * SC_SIDE + 127) / 128 * 128;
  static constexpr int CODE_SIDE = 64 * CB;
  static constexpr int OUT_BYTES = WP > 1 ? RB * HDP * 4 : 0;
  static constexpr int RING = NS * 2 * CODE_SIDE;
  static constexpr int SMEM = OFF_CODE + (RING > OUT_BYTES ? RING : OUT_BYTES);
};

// 16-byte piece j of position row r sits at piece pk_swz<C>(r, j): rows that
// share banks keep the same group apart.
template <int C>
__device__ __forceinline__ int pk_swz(int r, int j) {
  if (C >= 8) return j ^ (r & 7);
  if (C == 4) return j ^ ((r >> 1) & 3);
  return j ^ ((r >> 2) & 1);
}

__device__ __forceinline__ void cp16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// The tiles a block of rows [t0, t1] (of a sequence) reads: tiles [0, head)
// of the first positions, then [from, from + rest).
struct TileSpan {
  int head, from, rest;
  int lo, hi;  // positions any row sees: [lo, hi) and those below `sinks`
  __device__ __forceinline__ int count() const { return head + rest; }
  __device__ __forceinline__ int tile(int k) const { return k < head ? k : from + (k - head); }
};

__device__ __forceinline__ TileSpan span_of(const PackAttend &a, const SeqAt &q, int t0, int t1) {
  TileSpan s = {0, 0, 0, 0, 0};
  const int p0 = max(q.fill + t0, 0), p1 = min(q.fill + t1, a.c.positions - 1);
  if (q.slot < 0 || p1 < p0) return s;
  s.hi = p1 + 1;
  s.lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
  s.from = s.lo / PACK_TILE;
  s.rest = (s.hi + PACK_TILE - 1) / PACK_TILE - s.from;
  s.head = min((min(a.sinks, s.hi) + PACK_TILE - 1) / PACK_TILE, s.from);
  return s;
}

// Block b (of RB rows) of a sequence: its tokens.
__device__ __forceinline__ TileSpan block_span(const PackAttend &a, const SeqAt &q, int b, int rb) {
  const int t0 = b * rb / a.group, t1 = min(q.n - 1, ((b + 1) * rb - 1) / a.group);
  return span_of(a, q, t0, t1);
}

__device__ __forceinline__ int blocks_of(const PackAttend &a, const SeqAt &q, int rb) {
  return (q.n * a.group + rb - 1) / rb;
}

// Sums over the block (every thread gets the total); `red` holds a word a
// warp and two more.
__device__ __forceinline__ int block_total(int v, int *red) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

// The exclusive sum of `v` over the block's threads, and the total.
__device__ __forceinline__ int block_scan(int v, int *red, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  int before = 0, t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
    if (w < warp) before += red[w];
    t += red[w];
  }
  *total = t;
  return before + x - v;
}

// A sequence's weight in the list that blocks share out: its tiles over all
// its blocks and key/value heads (spread), or its blocks.
__device__ __forceinline__ int seq_weight(const PackAttend &a, int s, int rb, bool spread) {
  if (s >= a.r.count) return 0;
  const SeqAt q = seq_at(a.c, a.r, s);
  const int nb = blocks_of(a, q, rb);
  if (!spread) return nb;
  int w = 0;
  for (int b = 0; b < nb; ++b) w += block_span(a, q, b, rb).count();
  return w * a.c.heads;
}

// The total weight and, for `want` in [0, total), the sequence that holds it
// and the weight before that sequence.
struct ListAt {
  int total, s, before;
};
__device__ __forceinline__ ListAt list_at(const PackAttend &a, int rb, bool spread, int want, int *red) {
  ListAt at = {0, -1, 0};
  int *found = red + 8;
  if (threadIdx.x == 0) found[0] = -1;
  for (int base = 0; base < a.r.count; base += blockDim.x) {
    int t;
    const int w = seq_weight(a, base + threadIdx.x, rb, spread);
    const int before = at.total + block_scan(w, red, &t);
    if (want >= before && want - before < w) {
      found[0] = base + threadIdx.x;
      found[1] = before;
    }
    at.total += t;
  }
  __syncthreads();
  at.s = found[0];
  at.before = found[1];
  __syncthreads();
  return at;
}
// The weight of all sequences, and of those before `s`.
__device__ __forceinline__ int list_total(const PackAttend &a, int rb, bool spread, int s, int *before, int *red) {
  int w = 0, b = 0;
  for (int i = threadIdx.x; i < a.r.count; i += blockDim.x) {
    const int x = seq_weight(a, i, rb, spread);
    w += x;
    if (i < s) b += x;
  }
  if (before) *before = block_total(b, red);
  return block_total(w, red);
}

// Tiles a block takes of a list of `total`.
constexpr int PACK_SHARE_LEAST = 1;
__device__ __forceinline__ int share_of(int total, int grid) {
  return max(PACK_SHARE_LEAST, (total + grid - 1) / grid);
}

template <int HDP, int MT, bool SP>
__global__ void __launch_bounds__(128) pack_attend_kernel(PackAttend a, int spread, int parts) {
  using L = PackTile<HDP, MT, SP>;
  constexpr int RB = L::RB, C = L::C, NS = L::NS, WC = L::WC, WP = L::WP, NB = L::NB, SCP = L::SCP;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int red[16];
  float *qoff = reinterpret_cast<float *>(sm + L::OFF_QOFF);
  float *fr = reinterpret_cast<float *>(sm + L::OFF_FR);
  float *wmax = reinterpret_cast<float *>(sm + L::OFF_MAX);
  float *wsum = reinterpret_cast<float *>(sm + L::OFF_SUM);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int size = a.c.size, chd = size / 32, group = a.group;
  const int wc = warp % WC, wp = warp / WC;

  pdl_wait();
  // which tiles this block takes
  int at = 0, end = 0, s = 0, b = 0, h = 0, part = 0, share = 0;
  SeqAt q;
  if (spread) {
    const int total = list_total(a, RB, true, 0, nullptr, red);
    share = share_of(total, gridDim.x);
    at = blockIdx.x * share;
    end = min(total, at + share);
    pdl_release();
    if (at >= end) return;
    const ListAt f = list_at(a, RB, true, at, red);
    s = f.s;
    if (s < 0) return;
    q = seq_at(a.c, a.r, s);
    int left = at - f.before;
    for (;; ++b) {
      if (b >= blocks_of(a, q, RB)) return;
      const int n = block_span(a, q, b, RB).count() * a.c.heads;
      if (left < n) {
        h = left / (n / a.c.heads);
        part = left - h * (n / a.c.heads);  // the tile of the unit it starts at
        break;
      }
      left -= n;
    }
  } else {
    const int u = blockIdx.x / parts;
    part = blockIdx.x - u * parts;
    h = u % a.c.heads;
    const int total = list_total(a, RB, false, 0, nullptr, red);
    const int vb = total - 1 - u / a.c.heads;  // the rows at the end see the most: first
    pdl_release();
    if (vb < 0) return;
    const ListAt f = list_at(a, RB, false, vb, red);
    s = f.s;
    if (s < 0) return;
    b = vb - f.before;
    q = seq_at(a.c, a.r, s);
  }

  for (;;) {  // one unit, or a piece of it, a turn
    const TileSpan sp = block_span(a, q, b, RB);
    const int n = sp.count();
    int ka, kb;
    bool whole;
    size_t place = 0;  // of the partial sums
    if (spread) {
      ka = part;
      kb = min(n, part + (end - at));
      whole = ka == 0 && kb == n;
      place = 2 * blockIdx.x + (ka == 0 ? 1 : 0);
    } else {
      ka = (int)((long)n * part / parts);
      kb = (int)((long)n * (part + 1) / parts);
      whole = parts == 1;
      place = blockIdx.x;
      if (!whole && ka == kb) return;
    }

    // ---- the query rows, as fragments
    __syncthreads();
    {
      const bool wide = wide_rows(a.q);
      constexpr int WPL = HDP >= 256 ? HDP / 256 : 1;  // code words a lane
      for (int r = warp; r < RB; r += 4) {
        const int rr = b * RB + r, token = rr / group, hq = h * group + rr % group;
        const bool live = rr < q.n * group;
        float x[WPL][8];
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < WPL; ++i) {
          const int w = lane + 32 * i;
          if (live && w < size / 8) {
            load8(a.q.data, a.q.type,
                  (size_t)(q.first + token) * a.q.row_stride + (size_t)hq * a.q.head_stride + 8 * w, wide, x[i]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[i][e]));
        }
        big = warp_max(big);
        int ex = 0;
        if (big > 0.0f && big <= 3.4e38f) {
          frexpf(big, &ex);
          ex = 14 - ex;  // big 2^ex in [2^13, 2^14)
        }
        if (lane == 0) fr[r] = ldexpf(a.scale * 1.4426950408889634f, 24 - ex);
#pragma unroll
        for (int i = 0; i < WPL; ++i) {
          const int w = lane + 32 * i, gq = w >> 2, tq = w & 3;
          if (w >= HDP / 8) continue;  // narrow heads: the lanes past the row
          float sum = 0.0f, y[8], z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = ldexpf(x[i][e], ex);
            const float hi = __half2float(__float2half_rn(v));
            y[e] = hi;
            z[e] = SP ? __half2float(__float2half_rn(v - hi)) : 0.0f;
            sum += SP ? y[e] + z[e] : y[e];
          }
          const uint32_t four = 0xfu << (lane & 28);
          sum += __shfl_xor_sync(four, sum, 1);
          sum += __shfl_xor_sync(four, sum, 2);
          if (tq == 0) qoff[gq * RB + r] = -8.0f * 5.9604644775390625e-08f * sum;  // 2^-24
          // product m of a group: columns (2m, 2m + 4) and, an 1/16th of them, (2m + 1, 2m + 5)
#pragma unroll
          for (int pt = 0; pt < L::PARTS; ++pt) {
            const float(&v)[8] = pt ? z : y;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              uint32_t *f = reinterpret_cast<uint32_t *>(sm + pt * L::QF) +
                            (((gq * 2 + m) * MT + (r >> 4)) * 32 + (r & 7) * 4 + tq) * 4 + ((r & 8) ? 1 : 0);
              f[0] = half2_bits(v[2 * m], v[2 * m + 4]);
              f[2] = half2_bits(v[2 * m + 1] * 0.0625f, v[2 * m + 5] * 0.0625f);
            }
          }
        }
      }
      // groups past the head: their scales stay zero
      for (int i = tid; i < NS * 2 * (C - chd) * SCP; i += 128) {
        const int st = i / ((C - chd) * SCP), e = i - st * (C - chd) * SCP;
        reinterpret_cast<uint16_t *>(sm + L::OFF_SC + st * L::SC_SIDE)[chd * SCP + e] = 0;
      }
    }
    int pos[MT][2];  // the position of this thread's rows, -1 for none
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = b * RB + mt * 16 + g8 + 8 * e, p = q.fill + rr / group;
        pos[mt][e] = rr < q.n * group && p < a.c.positions ? max(p, -1) : -1;
      }
    const int p_first = q.fill + b * RB / group;  // the first row's
    const int p_last = sp.hi - 1;
    const bool past = q.fill + min(q.n - 1, ((b + 1) * RB - 1) / group) >= a.c.positions;

    if (tid == 0 && (past || q.slot < 0)) pack_trouble(a.c);

    // ---- the tiles
    const size_t unit = ((size_t)max(q.slot, 0) * a.c.heads + h) * a.c.positions;
    const uint8_t *kc = a.c.kc + unit * (size / 2), *vc = a.c.vc + unit * (size / 2);
    const uint16_t *scp = (tid >= 64 ? a.c.vs : a.c.ks) + unit * chd;
    uint32_t screg[C / 2];
    auto load_codes = [&](int k) {
      if (k < kb) {
        const size_t from = (size_t)sp.tile(k) * PACK_TILE * (size / 2);
        uint8_t *dk = sm + L::OFF_CODE + (k % NS) * 2 * L::CODE_SIDE, *dv = dk + L::CODE_SIDE;
        if (chd == C) {
#pragma unroll
          for (int i = 0; i < 64 * C / 128; ++i) {
            const int e = tid + 128 * i, r = e / C, j = e % C, o = r * L::CB + pk_swz<C>(r, j) * 16;
            cp16(dk + o, kc + from + (size_t)e * 16);
            cp16(dv + o, vc + from + (size_t)e * 16);
          }
        } else {
          for (int e = tid; e < 64 * chd; e += 128) {
            const int r = e / chd, j = e - r * chd, o = r * L::CB + pk_swz<C>(r, j) * 16;
            cp16(dk + o, kc + from + (size_t)e * 16);
            cp16(dv + o, vc + from + (size_t)e * 16);
          }
        }
      }
      cp_commit();
    };
    // scales pass through registers: position tid % 64's of the key side
    // (first half of the block) or the value side
    auto load_scales = [&](int k) {
      if (k >= kb) return;
      const uint16_t *src = scp + ((size_t)sp.tile(k) * PACK_TILE + (tid & 63)) * chd;
      if (chd == C) {
        if constexpr (C == 2) screg[0] = *reinterpret_cast<const uint32_t *>(src);
        else if constexpr (C == 4) *reinterpret_cast<uint2 *>(screg) = *reinterpret_cast<const uint2 *>(src);
        else {
#pragma unroll
          for (int i = 0; i < C / 8; ++i)
            reinterpret_cast<uint4 *>(screg)[i] = reinterpret_cast<const uint4 *>(src)[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < C / 2; ++i)
          screg[i] = (2 * i < chd ? (uint32_t)src[2 * i] : 0u) | (2 * i + 1 < chd ? (uint32_t)src[2 * i + 1] << 16 : 0u);
      }
    };
    auto keep_scales = [&](int k) {
      if (k >= kb) return;
      const int r = tid & 63, p = sp.tile(k) * PACK_TILE + r;
      // a value no row of the block sees counts as 0 whatever lies there
      const bool seen = p < sp.hi && (p >= sp.lo || p < a.sinks);
      uint16_t *dst = reinterpret_cast<uint16_t *>(sm + L::OFF_SC + ((k % NS) * 2 + (tid >> 6)) * L::SC_SIDE) + r;
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (i < chd) dst[i * SCP] = seen ? (uint16_t)(screg[i >> 1] >> (16 * (i & 1))) : (uint16_t)0;
    };

    float o[MT][NB * 8][4];
    float m_run[MT][2], l_run[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m_run[mt][e] = -INFINITY, l_run[mt][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < NB * 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.0f;
    }
    load_codes(ka);
    load_scales(ka);
    keep_scales(ka);
    load_codes(ka + 1);
    load_scales(ka + 1);
    for (int k = ka; k < kb; ++k) {
      cp_wait<1>();
      __syncthreads();
      keep_scales(k + 1);
      load_codes(k + 2);
      load_scales(k + 2);
      const uint8_t *tk = sm + L::OFF_CODE + (k % NS) * 2 * L::CODE_SIDE, *tv = tk + L::CODE_SIDE;
      const uint16_t *ksc = reinterpret_cast<const uint16_t *>(sm + L::OFF_SC + (k % NS) * 2 * L::SC_SIDE);
      const uint16_t *vsc = ksc + L::SC_SIDE / 2;

      // scores
      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][nt][e] = 0.0f;
#pragma unroll 2
      for (int gr = 0; gr < C; ++gr) {
        uint32_t qa[L::PARTS][MT][2][4];
        float off[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          off[mt][0] = qoff[gr * RB + mt * 16 + g8];
          off[mt][1] = qoff[gr * RB + mt * 16 + g8 + 8];
#pragma unroll
          for (int pt = 0; pt < L::PARTS; ++pt)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              const uint4 v = reinterpret_cast<const uint4 *>(sm + pt * L::QF)[((gr * 2 + m) * MT + mt) * 32 + lane];
              qa[pt][mt][m][0] = v.x, qa[pt][mt][m][1] = v.y, qa[pt][mt][m][2] = v.z, qa[pt][mt][m][3] = v.w;
            }
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const int r = warp * 16 + nt * 8 + g8;
          const uint32_t w = *reinterpret_cast<const uint32_t *>(tk + r * L::CB + pk_swz<C>(r, gr) * 16 + t4 * 4);
          const uint32_t w8 = w >> 8;
          const float2 step = __half22float2(
              *reinterpret_cast<const __half2 *>(ksc + gr * SCP + warp * 16 + nt * 8 + 2 * t4));
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float acc[4] = {off[mt][0], off[mt][0], off[mt][1], off[mt][1]};
#pragma unroll
            for (int pt = 0; pt < L::PARTS; ++pt) {
              mma16816(acc, qa[pt][mt][0], w & 0x000f000fu, w & 0x00f000f0u, acc);
              mma16816(acc, qa[pt][mt][1], w8 & 0x000f000fu, w8 & 0x00f000f0u, acc);
            }
            sc[mt][nt][0] = fmaf(acc[0], step.x, sc[mt][nt][0]);
            sc[mt][nt][1] = fmaf(acc[1], step.y, sc[mt][nt][1]);
            sc[mt][nt][2] = fmaf(acc[2], step.x, sc[mt][nt][2]);
            sc[mt][nt][3] = fmaf(acc[3], step.y, sc[mt][nt][3]);
          }
        }
      }

      // softmax, in powers of two
      const int tile0 = sp.tile(k) * PACK_TILE, j0 = tile0 + warp * 16 + 2 * t4;
      const bool all = !past && tile0 + PACK_TILE - 1 <= p_first &&
                       (a.window <= 0 || tile0 > p_last - a.window || tile0 + PACK_TILE <= a.sinks);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = fr[mt * 16 + g8 + 8 * e];
          float mx = -INFINITY;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float &x = sc[mt][nt][2 * e + c];
              const int j = j0 + nt * 8 + c, p = pos[mt][e];
              const bool see = all || (j <= p && (a.window <= 0 || j > p - a.window || j < a.sinks));
              x = see ? x * f : -INFINITY;
              mx = fmaxf(mx, x);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          if (t4 == 0) wmax[(mt * 16 + g8 + 8 * e) * 4 + warp] = mx;
        }
      __syncthreads();
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float al[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 w4 = *reinterpret_cast<const float4 *>(wmax + (mt * 16 + g8 + 8 * e) * 4);
          const float mx = fmaxf(fmaxf(fmaxf(w4.x, w4.y), fmaxf(w4.z, w4.w)), m_run[mt][e]);
          const float base = mx == -INFINITY ? 0.0f : mx;
          al[e] = exp2_fast(m_run[mt][e] - base);
          m_run[mt][e] = mx;
          float sum = 0.0f;
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float &x = sc[mt][nt][2 * e + c];
              x = exp2_fast(x - base + 12.0f);
              sum += x;
            }
          l_run[mt][e] = l_run[mt][e] * al[e] + sum;
        }
        // a warp's scores lie as the weights' fragment of its 16 positions does
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = sc[mt][i >> 1][2 * (i & 1)], y = sc[mt][i >> 1][2 * (i & 1) + 1];
          hi[i] = half2_bits(x, y);
          if (SP) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[i]));
            lo[i] = half2_bits(x - f.x, y - f.y);
          }
        }
        reinterpret_cast<uint4 *>(sm + L::OFF_P)[(warp * MT + mt) * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (SP)
          reinterpret_cast<uint4 *>(sm + L::OFF_P + L::PF)[(warp * MT + mt) * 32 + lane] =
              make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
          for (int j = 0; j < NB * 8; ++j) {
            o[mt][j][0] *= al[0];
            o[mt][j][1] *= al[0];
            o[mt][j][2] *= al[1];
            o[mt][j][3] *= al[1];
          }
        }
      }
      __syncthreads();

      // values
#pragma unroll
      for (int si = 0; si < 4 / WP; ++si) {
        const int st = wp * (4 / WP) + si;
        uint32_t pa[L::PARTS][MT][4];
#pragma unroll
        for (int pt = 0; pt < L::PARTS; ++pt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const uint4 v = reinterpret_cast<const uint4 *>(sm + L::OFF_P + pt * L::PF)[(st * MT + mt) * 32 + lane];
            pa[pt][mt][0] = v.x, pa[pt][mt][1] = v.y, pa[pt][mt][2] = v.z, pa[pt][mt][3] = v.w;
          }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int j = (wc * NB + nb) * 2 + (g8 >> 2);  // the 16-byte piece (one group)
          uint32_t w[4];
          __half2 step[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = st * 16 + 8 * i + 2 * t4;
            const uint8_t *row = tv + r * L::CB + (g8 & 3) * 4;
            w[2 * i] = *reinterpret_cast<const uint32_t *>(row + pk_swz<C>(r, j) * 16);
            w[2 * i + 1] = *reinterpret_cast<const uint32_t *>(row + L::CB + pk_swz<C>(r + 1, j) * 16);
            step[i] = *reinterpret_cast<const __half2 *>(vsc + j * SCP + r);
          }
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // columns 0-3, then 4-7 of the thread's eight
            uint32_t v[2][4];  // [positions 2t.., 2t + 8..][column]
#pragma unroll
            for (int i = 0; i < 2; ++i)
              dequant_i4(__byte_perm(w[2 * i], w[2 * i + 1], hf ? 0x7632 : 0x5410), v[i]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t vh[2], vl[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const __half2 n2 = *reinterpret_cast<const __half2 *>(&v[i][c]);
                const __half2 x = __hmul2(n2, step[i]);
                vh[i] = *reinterpret_cast<const uint32_t *>(&x);
                if (SP) {
                  const __half2 y = __hfma2(n2, step[i], __hneg2(x));
                  vl[i] = *reinterpret_cast<const uint32_t *>(&y);
                }
              }
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                float(&acc)[4] = o[mt][nb * 8 + hf * 4 + c];
                mma16816(acc, pa[0][mt], vh[0], vh[1], acc);
                if (SP) {
                  mma16816(acc, pa[1][mt], vh[0], vh[1], acc);
                  mma16816(acc, pa[0][mt], vl[0], vl[1], acc);
                }
              }
            }
          }
        }
      }
    }
    cp_wait<0>();

    // ---- the rows' sums, and of a narrow head the warps' shares, joined
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[mt][e];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t4 == 0) wsum[(mt * 16 + g8 + 8 * e) * 4 + warp] = l;
      }
    __syncthreads();
    if (WP > 1) {
      float *buf = reinterpret_cast<float *>(sm + L::OFF_CODE);
      for (int r = 1; r < WP; ++r) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < NB * 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float *x = buf + (((mt * WC + wc) * NB * 8 + j) * 4 + e) * 32 + lane;
              if (wp == r) *x = o[mt][j][e];
            }
        __syncthreads();
        if (wp == 0) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < NB * 8; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[mt][j][e] += buf[(((mt * WC + wc) * NB * 8 + j) * 4 + e) * 32 + lane];
        }
        __syncthreads();
      }
    }
    if (wp == 0) {
      const bool wide = wide_rows(a.out);
      float *pw = a.work + place * ((size_t)RB * (size + 2));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = mt * 16 + g8 + 8 * e, rr = b * RB + r;
          if (rr >= q.n * group) continue;
          const float4 l4 = *reinterpret_cast<const float4 *>(wsum + r * 4);
          const float l = l4.x + l4.y + l4.z + l4.w;
          const float inv = whole ? (l == 0.0f ? 0.0f : __fdividef(1.0f, l)) : 1.0f;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int col = (wc * NB + nb) * 64 + 16 * t4 + 8 * c;
              if (col >= size) continue;
              float x[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = o[mt][nb * 8 + j][2 * e + c] * inv;
              if (whole) {
                store8(a.out.data, a.out.type,
                       (size_t)(q.first + rr / group) * a.out.row_stride +
                           (size_t)(h * group + rr % group) * a.out.head_stride + col,
                       wide, x);
              } else {
                store8(pw, 1, (size_t)r * size + col, (size & 3) == 0, x);
              }
            }
          if (!whole && wc == 0 && t4 == 0) {
            pw[(size_t)RB * size + r] = m_run[mt][e];
            pw[(size_t)RB * size + RB + r] = l;
          }
        }
    }

    // ---- the next unit
    if (!spread) return;
    at += kb - ka;
    if (at >= end) return;
    part = 0;
    do {
      if (++h == a.c.heads) {
        h = 0;
        ++b;
        while (b >= blocks_of(a, q, RB)) {
          b = 0;
          if (++s >= a.r.count) return;
          q = seq_at(a.c, a.r, s);
        }
      }
    } while (block_span(a, q, b, RB).count() == 0);
  }
}

// ---------------------------------------------------------------------------
// the pieces of a unit joined, and rows that see nothing set to zero: a warp a
// row, pieces in order

struct PackMerge {
  PackAttend a;
  int rb, spread, parts, grid, blocks;
};

__global__ void __launch_bounds__(128) pack_merge_kernel(PackMerge g) {
  __shared__ int red[16];
  const PackAttend &a = g.a;
  const int RB = g.rb, size = a.c.size;
  pdl_wait();
  pdl_release();
  int u = blockIdx.x, s, b, h = u % a.c.heads, first, last, share = 0, n;
  SeqAt q;
  u /= a.c.heads;
  if (g.spread) {
    s = u / g.blocks;
    b = u - s * g.blocks;
    int before;
    const int total = list_total(a, RB, true, s, &before, red);
    share = share_of(total, g.grid);
    q = seq_at(a.c, a.r, s);
    if (b >= blocks_of(a, q, RB)) return;
    for (int i = 0; i < b; ++i) before += block_span(a, q, i, RB).count() * a.c.heads;
    n = block_span(a, q, b, RB).count();
    before += h * n;
    first = before / share;
    last = (before + max(n, 1) - 1) / share;
    if (n > 0 && first == last) return;  // one block had it all
    u = before;
  } else {
    const int total = list_total(a, RB, false, 0, nullptr, red);
    if (u >= total) return;
    const ListAt f = list_at(a, RB, false, total - 1 - u, red);
    s = f.s;
    if (s < 0) return;
    b = total - 1 - u - f.before;
    q = seq_at(a.c, a.r, s);
    n = block_span(a, q, b, RB).count();
    first = 0;
    last = g.parts - 1;
    u = blockIdx.x * g.parts;
  }
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, rr = b * RB + r;
  if (rr >= q.n * a.group) return;
  const size_t piece = (size_t)RB * (size + 2);
  float m = -INFINITY, l = 0.0f;
  float x[2][8] = {};
  if (n > 0) {
    for (int i = first; i <= last; ++i) {
      size_t place;
      if (g.spread) {
        place = 2 * (size_t)i + (i * share <= u ? 1 : 0);  // the piece with the unit's first tile
      } else {
        if ((long)n * i / g.parts == (long)n * (i + 1) / g.parts) continue;
        place = (size_t)u + i;
      }
      const float *pw = a.work + place * piece;
      const float pm = pw[(size_t)RB * size + r], pl = pw[(size_t)RB * size + RB + r];
      if (pl == 0.0f) continue;  // it saw none of the row's positions
      const float mx = fmaxf(m, pm), f0 = exp2_fast(m - mx), f1 = exp2_fast(pm - mx);
      m = mx;
      l = l * f0 + pl * f1;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = lane * 8 + e * 256;
        if (col >= size) continue;
        float y[8];
        load8(pw, 1, (size_t)r * size + col, true, y);
#pragma unroll
        for (int i2 = 0; i2 < 8; ++i2) x[e][i2] = x[e][i2] * f0 + y[i2] * f1;
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
  if (n == 0 && lane == 0 && (q.slot < 0 || q.fill + rr / a.group >= a.c.positions)) pack_trouble(a.c);
  const bool wide = wide_rows(a.out);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int col = lane * 8 + e * 256;
    if (col >= size) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[e][i] *= inv;
    store8(a.out.data, a.out.type,
           (size_t)(q.first + rr / a.group) * a.out.row_stride +
               (size_t)(h * a.group + rr % a.group) * a.out.head_stride + col,
           wide, x[e]);
  }
}

template <typename... P, typename... Q>
cudaError_t pack_launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool overlap,
                        Q... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (overlap) {
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// What a kernel form needs on the current device, looked up once a device:
// its shared memory allowed and how many blocks an SM holds.
constexpr int PACK_DEVICES = 64;

template <int HDP, int MT, bool SP>
cudaError_t pack_form_ready(int *per_sm) {
  static std::atomic<int> known[PACK_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < PACK_DEVICES && (*per_sm = known[dev].load()) > 0) return cudaSuccess;
  auto kern = pack_attend_kernel<HDP, MT, SP>;
  using L = PackTile<HDP, MT, SP>;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kern, 128, L::SMEM);
  if (e == cudaSuccess && *per_sm < 1) e = cudaErrorInvalidConfiguration;
  if (e == cudaSuccess && dev < PACK_DEVICES) known[dev].store(*per_sm);
  return e;
}

template <int HDP, int MT, bool SP>
cudaError_t pack_form_launch(const PackAttend &a, const PackPlan &p, cudaStream_t st) {
  return pack_launch(pack_attend_kernel<HDP, MT, SP>, dim3(p.grid), 128, PackTile<HDP, MT, SP>::SMEM, st, false, a,
                     p.spread, p.parts);
}

// Calls F for the form a plan names.
#define PACK_FORMS(F, p, ...)                                                                      \
  switch ((p).wide * 8 + (p).tiles16 * 2 + (p).split2) {                                          \
    case 64 * 8 + 2: return F<64, 1, false>(__VA_ARGS__);                                          \
    case 64 * 8 + 4: return F<64, 2, false>(__VA_ARGS__);                                          \
    case 64 * 8 + 8: return F<64, 4, false>(__VA_ARGS__);                                          \
    case 64 * 8 + 3: return F<64, 1, true>(__VA_ARGS__);                                           \
    case 64 * 8 + 5: return F<64, 2, true>(__VA_ARGS__);                                           \
    case 128 * 8 + 2: return F<128, 1, false>(__VA_ARGS__);                                        \
    case 128 * 8 + 4: return F<128, 2, false>(__VA_ARGS__);                                        \
    case 128 * 8 + 8: return F<128, 4, false>(__VA_ARGS__);                                        \
    case 128 * 8 + 3: return F<128, 1, true>(__VA_ARGS__);                                         \
    case 128 * 8 + 5: return F<128, 2, true>(__VA_ARGS__);                                         \
    case 256 * 8 + 2: return F<256, 1, false>(__VA_ARGS__);                                        \
    case 256 * 8 + 4: return F<256, 2, false>(__VA_ARGS__);                                        \
    case 256 * 8 + 8: return F<256, 4, false>(__VA_ARGS__);                                        \
    case 256 * 8 + 3: return F<256, 1, true>(__VA_ARGS__);                                         \
    case 256 * 8 + 5: return F<256, 2, true>(__VA_ARGS__);                                         \
    case 512 * 8 + 2: return F<512, 1, false>(__VA_ARGS__);                                        \
    case 512 * 8 + 4: return F<512, 2, false>(__VA_ARGS__);                                        \
    case 512 * 8 + 3: return F<512, 1, true>(__VA_ARGS__);                                         \
    default: return cudaErrorInvalidValue;                                                        \
  }

static cudaError_t pack_form(const PackPlan &p, int *per_sm) { PACK_FORMS(pack_form_ready, p, per_sm) }
static cudaError_t pack_run(const PackPlan &p, const PackAttend &a, cudaStream_t st) {
  PACK_FORMS(pack_form_launch, p, a, p, st)
}

static cudaError_t pack_sms(int *sms) {
  static std::atomic<int> known[PACK_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < PACK_DEVICES && (*sms = known[dev].load()) > 0) return cudaSuccess;
  e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && dev < PACK_DEVICES) known[dev].store(*sms);
  return e;
}

}  // namespace igc

using namespace igc;

static cudaError_t launch_rows(bool write, const PackView *c, const PackRows *r, const PackData *k, const PackData *v,
                               cudaStream_t st) {
  const PackIo io = {*c, *r, *k, *v};
  const long items = (long)r->rows * 2 * c->heads * (c->size / 8);
  const long blocks = (items + PK_THREADS * PK_ITEMS - 1) / (PK_THREADS * PK_ITEMS);
  if (blocks < 1 || blocks > 0x7fffffffL) return cudaErrorInvalidValue;
  return write ? pack_launch(pack_rows_kernel<true>, dim3((unsigned)blocks), PK_THREADS, 0, st, false, io)
               : pack_launch(pack_rows_kernel<false>, dim3((unsigned)blocks), PK_THREADS, 0, st, false, io);
}

cudaError_t igc_launch_pack_write(const PackView *c, const PackRows *r, const PackData *k, const PackData *v,
                                  cudaStream_t st) {
  return launch_rows(true, c, r, k, v, st);
}

cudaError_t igc_launch_pack_read(const PackView *c, const PackRows *r, const PackData *k, const PackData *v,
                                 cudaStream_t st) {
  return launch_rows(false, c, r, k, v, st);
}

cudaError_t igc_pack_plan(int count, int rows, int rows_most, int positions, int kv_heads, int group, int size,
                          int type, int window, int sinks, PackPlan *p) {
  memset(p, 0, sizeof(*p));
  p->wide = size <= 64 ? 64 : size <= 128 ? 128 : size <= 256 ? 256 : 512;
  p->split2 = type == 1 ? 1 : 0;
  const long need = (long)rows_most * group;
  const int most16 = p->wide == 512 ? (p->split2 ? 1 : 2) : (p->split2 ? 2 : 4);
  p->tiles16 = need <= 16 ? 1 : need <= 32 || most16 < 4 ? 2 : 4;
  if (p->tiles16 > most16) p->tiles16 = most16;
  const int rb = 16 * p->tiles16;
  int sms = 0, per_sm = 0;
  cudaError_t e = pack_sms(&sms);
  if (e == cudaSuccess) e = pack_form(*p, &per_sm);
  if (e != cudaSuccess) return e;
  const long blocks = (need + rb - 1) / rb;
  const long slots = (long)sms * per_sm;
  // the most tiles a unit can have: its rows' reach, wherever it starts in a tile
  const long reach = window > 0 ? (long)window + rb / group + 1 + sinks + 3 * PACK_TILE : positions;
  const long tiles = ((reach < positions ? reach : positions) + PACK_TILE - 1) / PACK_TILE;
  p->spread = blocks <= 8;
  long grid;
  if (p->spread) {
    const long units = count * blocks * kv_heads, list = units * tiles;
    grid = list < slots ? list : slots;
    p->blocks = (int)blocks;
    if (units > 0x7fffffffL) return cudaErrorInvalidValue;
    p->units = (int)units;
    p->parts = 1;
    p->work_floats = 2 * (size_t)grid * rb * (size + 2);
  } else {
    const long units = ((long)rows * group / rb + count) * kv_heads;
    long parts = (slots + units - 1) / units;
    if (parts > tiles) parts = tiles;
    grid = units * parts;
    if (grid > 0x7fffffffL) return cudaErrorInvalidValue;
    p->units = (int)units;
    p->parts = (int)parts;
    p->work_floats = parts > 1 ? (size_t)grid * rb * (size + 2) : 0;
  }
  p->grid = (int)grid;
  return cudaSuccess;
}

cudaError_t igc_launch_pack_attend(const PackAttend *a, const PackPlan *p, cudaStream_t st, int *launches) {
  *launches = 1;
  cudaError_t e = pack_run(*p, *a, st);
  if (e != cudaSuccess || (!p->spread && p->parts == 1)) return e;
  *launches = 2;
  const PackMerge g = {*a, 16 * p->tiles16, p->spread, p->parts, p->grid, p->blocks};
  return pack_launch(pack_merge_kernel, dim3((unsigned)p->units, 4 * p->tiles16), 128, 0, st, true, g);
}
