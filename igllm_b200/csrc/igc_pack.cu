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
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
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

// Four values; `wide`: eight from any multiple of eight columns start on 16 bytes.
__device__ __forceinline__ void store4(void *base, int type, size_t at, bool wide, const float (&x)[4]) {
  if (type == 1) {
    float *p = static_cast<float *>(base) + at;
    if (wide) {
      *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = x[i];
    }
    return;
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
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
    *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) p[2 * i] = (uint16_t)w[i], p[2 * i + 1] = (uint16_t)(w[i] >> 16);
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
// A block holds RB = 8 NT query rows of one (sequence, key/value head): row
// rr is the sequence's row rr / group, head rr % group of the group, so a
// token's heads share each tile of codes.  Four warps walk tiles of 64 MP
// positions that TMA brings NS deep, swizzled so that the reads below spread
// over the banks.  Positions and columns are the products' 16 rows and query
// rows their 8 columns, so eight heads fill a product.
//
//   scores  warp w takes positions 16 MP w on.  A code word becomes eight
//           n - 8, exact in f16, by nine instructions; which column of a
//           group a thread's product slot holds is free as long as the query
//           fragments agree, so words are used as they lie.  A group's sum
//           times its scale is an f32 multiply-add.  (Nibbles left in place
//           as subnormal halves, their -8 taken out of the sums, saved four
//           instructions a word and cost 2^-13 of a scale: the tensor core
//           aligns products by their exponent fields.)
//   softmax the running maximum and sum per row in 32 bits; the block's
//           maximum is merged through shared memory once a tile.
//   values  warp w takes 64 of the head's columns (or, of a narrow head, a
//           share of the positions).  Codes of two positions are zipped by a
//           byte permute, used as they lie.  For 16-bit rows the group's
//           scale goes into the weight, f16(f16(w) 8 scale), two roundings of
//           2^-11 at most, and codes enter exactly.
//
// A query row is scaled by the power of two that puts its largest magnitude
// in [2^13, 2^14) and kept as f16, exact for bf16 and f16 rows but for
// magnitudes 2^38 below the largest.  For f32 rows (SP) queries and weights
// are each kept as f16 hi and lo parts and (n - 8) scale as hi and lo, which
// hold it exactly; the products left out (lo x lo) are below f32's own
// rounding, and each step of 16 positions starts from zero accumulators, as
// the tensor core's sums round towards zero.

constexpr int PACK_TRIES = 1 << 22;  // polls a wait makes before it gives up

template <int HDP, int NT, bool SP>
struct PackTile {
  static constexpr int RB = 8 * NT;
  static constexpr int C = HDP / 32;                     // groups
  static constexpr int PITCH = HDP >= 256 ? 128 : HDP / 2;  // code bytes of a swizzled row
  static constexpr int HALVES = HDP / 2 / PITCH;         // rows of 512 columns lie in two halves
  static constexpr int MP = NT <= 2 && HDP <= 256 ? 2 : 1;
  static constexpr int TP = 64 * MP;                     // positions a step
  static constexpr int NS = MP == 2 || HDP == 512 ? 2 : 3;  // steps in flight
  static constexpr int WC = HDP >= 256 ? 4 : HDP / 64;   // warps across the columns
  static constexpr int WP = 4 / WC;                      // warps across a step's positions
  static constexpr int NB = HDP / 64 / WC;               // 64-column blocks a warp
  static constexpr int PARTS = SP ? 2 : 1;
  static constexpr int QF = C * NT * 512;                // bytes of one part's query fragments
  static constexpr int CODE64 = 64 * PITCH;              // one TMA box: 64 positions
  static constexpr int CODE_SIDE = MP * HALVES * CODE64;
  static constexpr int SC_SIDE = TP * C * 2;
  static constexpr int STAGE = 2 * CODE_SIDE + 2 * SC_SIDE;
  static constexpr int OFF_SC = 2 * CODE_SIDE;           // in a stage: keys, values, key scales, value scales
  static constexpr int RING = NS * ((STAGE + 1023) / 1024 * 1024);
  static constexpr int SLOT = RING / NS;
  static constexpr int OUT_BYTES = WP > 1 ? RB * HDP * 4 : 0;
  static constexpr int OFF_Q = RING > OUT_BYTES ? RING : OUT_BYTES;
  static constexpr int OFF_FR = OFF_Q + QF * PARTS;
  static constexpr int OFF_MAX = OFF_FR + RB * 4;
  static constexpr int OFF_SUM = OFF_MAX + 4 * RB * 4;
  static constexpr int PF = TP / 16 * NT * 256;          // bytes of one part's weight fragments
  static constexpr int OFF_P = OFF_SUM + 4 * RB * 4;
  static constexpr int SMEM = 1024 + OFF_P + PF * PARTS;
  // blocks an SM that registers are kept for
  static constexpr int PER_SM = NT == 1 ? (HDP <= 128 ? 4 : 3) : NT <= 4 && HDP <= 256 ? 3 : 2;
};

// Where the 16-byte piece j of position row r lies in a box of PITCH-byte
// rows: the 128-, 64- and 32-byte swizzles of a tensor map.
template <int PITCH>
__device__ __forceinline__ int pk_swz(int r, int j) {
  if (PITCH == 128) return r * 128 + ((j ^ (r & 7)) << 4);
  if (PITCH == 64) return r * 64 + ((j ^ ((r >> 1) & 3)) << 4);
  return r * 32 + ((j ^ ((r >> 2) & 1)) << 4);
}

// One box of a code array: 64 rows from row y, PITCH bytes from byte x.
__device__ __forceinline__ void pk_load(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// mma16816 of igc_device.cuh, free to be scheduled: d += a b.
__device__ __forceinline__ void mma_add(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
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
__device__ __forceinline__ uint32_t mul2(uint32_t x, uint32_t y) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2 *>(&x), *reinterpret_cast<const __half2 *>(&y));
  return *reinterpret_cast<const uint32_t *>(&h);
}
// c s - p, exact where p is c s rounded
__device__ __forceinline__ uint32_t rest2(uint32_t c, uint32_t s, uint32_t p) {
  const __half2 h = __hfma2(*reinterpret_cast<const __half2 *>(&c), *reinterpret_cast<const __half2 *>(&s),
                            __hneg2(*reinterpret_cast<const __half2 *>(&p)));
  return *reinterpret_cast<const uint32_t *>(&h);
}
// 2^e, e in [-126, 127]
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// The tiles a block of rows [t0, t1] (of a sequence) reads: tiles [0, head)
// of the first positions, then [from, from + rest).
struct TileSpan {
  int head, from, rest;
  int lo, hi;  // positions any row sees: [lo, hi) and those below `sinks`
  __device__ __forceinline__ int count() const { return head + rest; }
  __device__ __forceinline__ int tile(int k) const { return k < head ? k : from + (k - head); }
};

__device__ __forceinline__ TileSpan span_of(const PackAttend &a, const SeqAt &q, int t0, int t1, int tp) {
  TileSpan s = {0, 0, 0, 0, 0};
  const int p0 = max(q.fill + t0, 0), p1 = min(q.fill + t1, a.c.positions - 1);
  if (q.slot < 0 || p1 < p0) return s;
  s.hi = p1 + 1;
  s.lo = a.window > 0 ? max(0, p0 - a.window + 1) : 0;
  s.from = s.lo / tp;
  s.rest = (s.hi + tp - 1) / tp - s.from;
  s.head = min((min(a.sinks, s.hi) + tp - 1) / tp, s.from);
  return s;
}

// Block b (of RB rows) of a sequence: its tokens.
__device__ __forceinline__ TileSpan block_span(const PackAttend &a, const SeqAt &q, int b, int rb, int tp) {
  const int t0 = a.by_group.of(b * rb), t1 = min(q.n - 1, a.by_group.of((b + 1) * rb - 1));
  return span_of(a, q, t0, t1, tp);
}

__device__ __forceinline__ int blocks_of(const PackAttend &a, const SeqAt &q, int rb) {
  return (q.n * a.group + rb - 1) / rb;
}

// Sums over the block (every thread gets the total); `red` holds a word a
// warp and two more.
constexpr int PACK_WARPS = 16;  // the most of any block
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
__device__ __forceinline__ int seq_weight(const PackAttend &a, int s, int rb, int tp, bool spread) {
  if (s >= a.r.count) return 0;
  const SeqAt q = seq_at(a.c, a.r, s);
  const int nb = blocks_of(a, q, rb);
  if (!spread) return nb;
  int w = 0;
  for (int b = 0; b < nb; ++b) w += block_span(a, q, b, rb, tp).count();
  return w * a.c.heads;
}

// The total weight and, for `want` in [0, total), the sequence that holds it
// and the weight before that sequence.
struct ListAt {
  int total, s, before;
};
__device__ __forceinline__ ListAt list_at(const PackAttend &a, int rb, int tp, bool spread, int want, int *red) {
  ListAt at = {0, -1, 0};
  int *found = red + PACK_WARPS;
  if (threadIdx.x == 0) found[0] = -1;
  for (int base = 0; base < a.r.count; base += blockDim.x) {
    int t;
    const int w = seq_weight(a, base + threadIdx.x, rb, tp, spread);
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
__device__ __forceinline__ int list_total(const PackAttend &a, int rb, int tp, bool spread, int s, int *before, int *red) {
  int w = 0, b = 0;
  for (int i = threadIdx.x; i < a.r.count; i += blockDim.x) {
    const int x = seq_weight(a, i, rb, tp, spread);
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


// What each of `grid` blocks takes of the list (its total in at->total), and
// where in it block `mine` begins: one pass over the sequences where they fit
// the block, else two.
__device__ __forceinline__ int list_share(const PackAttend &a, int rb, int tp, int grid, int mine, ListAt *at,
                                          int *red) {
  if (a.r.count <= (int)blockDim.x) {
    int *found = red + PACK_WARPS;
    if (threadIdx.x == 0) found[0] = -1;
    const int w = seq_weight(a, threadIdx.x, rb, tp, true);
    const int before = block_scan(w, red, &at->total);
    const int share = share_of(at->total, grid), want = mine * share;
    if (want >= before && want - before < w) {
      found[0] = threadIdx.x;
      found[1] = before;
    }
    __syncthreads();
    at->s = found[0];
    at->before = found[1];
    return share;
  }
  const int total = list_total(a, rb, tp, true, 0, nullptr, red), share = share_of(total, grid);
  *at = list_at(a, rb, tp, true, mine * share, red);
  at->total = total;
  return share;
}

// The units of a block's share, in the order every warp walks them.
struct PackWalk {
  int at, end, s, b, h, part, n, ka, kb;
  bool whole;
  size_t place;
  SeqAt q;
  TileSpan sp;
};

// The block's first unit; false where it has none.
template <int RB, int TP>
__device__ __forceinline__ bool walk_start(const PackAttend &a, int spread, int parts, PackWalk &w, int *red) {
  w.at = w.end = w.h = w.b = w.part = 0;
  if (spread) {
    ListAt f;
    const int share = list_share(a, RB, TP, gridDim.x, blockIdx.x, &f, red);
    w.at = blockIdx.x * share;
    w.end = min(f.total, w.at + share);
    if (w.at >= w.end || f.s < 0) return false;
    w.s = f.s;
    w.q = seq_at(a.c, a.r, w.s);
    int left = w.at - f.before;
    for (;; ++w.b) {
      if (w.b >= blocks_of(a, w.q, RB)) return false;
      const int n = block_span(a, w.q, w.b, RB, TP).count() * a.c.heads;
      if (left < n) {
        w.h = left / (n / a.c.heads);
        w.part = left - w.h * (n / a.c.heads);  // the step of the unit it starts at
        return true;
      }
      left -= n;
    }
  }
  const int u = blockIdx.x / parts;
  w.part = blockIdx.x - u * parts;
  w.h = u % a.c.heads;
  const int total = list_total(a, RB, TP, false, 0, nullptr, red);
  const int vb = total - 1 - u / a.c.heads;  // the rows at the end see the most: first
  if (vb < 0) return false;
  const ListAt f = list_at(a, RB, TP, false, vb, red);
  w.s = f.s;
  if (w.s < 0) return false;
  w.b = vb - f.before;
  w.q = seq_at(a.c, a.r, w.s);
  return true;
}

// The steps [ka, kb) of the unit that are this block's.
template <int RB, int TP>
__device__ __forceinline__ void walk_unit(const PackAttend &a, int spread, int parts, PackWalk &w) {
  w.sp = block_span(a, w.q, w.b, RB, TP);
  w.n = w.sp.count();
  if (spread) {
    w.ka = w.part;
    w.kb = min(w.n, w.part + (w.end - w.at));
    w.whole = w.ka == 0 && w.kb == w.n;
    w.place = 2 * (size_t)blockIdx.x + (w.ka == 0 ? 1 : 0);
  } else {
    w.ka = (int)((long)w.n * w.part / parts);
    w.kb = (int)((long)w.n * (w.part + 1) / parts);
    w.whole = parts == 1;
    w.place = blockIdx.x;
  }
}

// On to the next unit; false at the end.
template <int RB, int TP>
__device__ __forceinline__ bool walk_next(const PackAttend &a, int spread, PackWalk &w) {
  if (!spread) return false;
  w.at += w.kb - w.ka;
  if (w.at >= w.end) return false;
  w.part = 0;
  do {
    if (++w.h == a.c.heads) {
      w.h = 0;
      ++w.b;
      while (w.b >= blocks_of(a, w.q, RB)) {
        w.b = 0;
        if (++w.s >= a.r.count) return false;
        w.q = seq_at(a.c, a.r, w.s);
      }
    }
  } while (block_span(a, w.q, w.b, RB, TP).count() == 0);
  return true;
}

template <int HDP, int NT, bool SP, bool FULL>
__global__ void __launch_bounds__(128, PackTile<HDP, NT, SP>::PER_SM)
    pack_attend_kernel(const __grid_constant__ PackAttend a, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv, int spread, int parts) {
  using L = PackTile<HDP, NT, SP>;
  constexpr int RB = L::RB, C = L::C, NS = L::NS, WC = L::WC, WP = L::WP, NB = L::NB, MP = L::MP, TP = L::TP,
                PITCH = L::PITCH;
  extern __shared__ __align__(1024) uint8_t sm_raw[];
  __shared__ int red[PACK_WARPS + 2];
  __shared__ uint64_t full[NS];
  uint8_t *sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
  float *fr = reinterpret_cast<float *>(sm + L::OFF_FR);
  float *wmax = reinterpret_cast<float *>(sm + L::OFF_MAX);
  float *wsum = reinterpret_cast<float *>(sm + L::OFF_SUM);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
  const int size = FULL ? HDP : a.c.size, chd = size / 32, group = a.group;
  const int wc = warp % WC, wp = warp / WC;
  // Places in a step's codes, the swizzle resolved: piece j of this thread's
  // key row is at kat ^ 16 j, of its two value rows at vat[.] ^ 16 j (rows a
  // multiple of 8 on are plain offsets).
  const int r0 = warp * 16 * MP + g8;
  const uint32_t kat = pk_swz<PITCH>(r0, 0) + t4 * 4;
  const uint32_t vrow = wp * (TP / WP) + 2 * t4, vj = ((wc * NB * 2) & 7) << 4;
  const uint32_t vat[2] = {(pk_swz<PITCH>(vrow, 0) + (g8 >> 1) * 4) ^ vj, (pk_swz<PITCH>(vrow + 1, 0) + (g8 >> 1) * 4) ^ vj};
  const uint32_t vhalf = (wc * NB / 4) * L::CODE64;  // of 512 columns, the half
  const uint32_t zip = g8 & 1 ? 0x7632 : 0x5410;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 1);
    mbar_init_fence();
  }

  PackWalk w;
  const bool any = walk_start<RB, TP>(a, spread, parts, w, red);
  pdl_release();
  if (!any) return;
  int step0 = 0;  // steps this block has taken: the ring's place
  bool gave_up = false;
  for (;;) {  // one unit, or a piece of it, a turn
    walk_unit<RB, TP>(a, spread, parts, w);
    const SeqAt q = w.q;
    const TileSpan sp = w.sp;
    const int b = w.b, h = w.h, ka = w.ka, kb = w.kb;
    const bool whole = w.whole;
    if (!spread && !whole && ka == kb) return;
    const size_t unit = ((size_t)max(q.slot, 0) * a.c.heads + h) * a.c.positions;
    // step k's codes and scales: 64 positions a copy, those past the last
    // position any row sees left out
    auto load = [&](int k) {
      if (k >= kb || tid != 0) return;
      const int i = (step0 + k - ka) % NS, p0 = sp.tile(k) * TP;
      const int boxes = min(MP, (sp.hi - p0 + 63) / 64);
      uint8_t *st = sm + i * L::SLOT;
      const uint32_t scales = (uint32_t)boxes * 64 * chd * 2;
      mbar_expect(&full[i], (uint32_t)boxes * 2 * L::HALVES * L::CODE64 + 2 * scales);
      for (int x = 0; x < boxes; ++x)
#pragma unroll
        for (int y = 0; y < L::HALVES; ++y) {
          pk_load(st + (x * L::HALVES + y) * L::CODE64, &tmk, y * 128, (int)unit + p0 + 64 * x, &full[i]);
          pk_load(st + L::CODE_SIDE + (x * L::HALVES + y) * L::CODE64, &tmv, y * 128, (int)unit + p0 + 64 * x,
                  &full[i]);
        }
      const uint64_t once = l2_evict_first();
      bulk_load(st + L::OFF_SC, a.c.ks + (unit + p0) * chd, scales, &full[i], once);
      bulk_load(st + L::OFF_SC + L::SC_SIDE, a.c.vs + (unit + p0) * chd, scales, &full[i], once);
    };
    __syncthreads();  // the unit before is done with the ring and the fragments
    for (int k = ka; k < ka + NS - 1; ++k) load(k);

    // ---- the query rows, as fragments
    {
      const bool wide = wide_rows(a.q);
      constexpr int WPL = HDP >= 256 ? HDP / 256 : 1;  // code words a lane
      for (int r = warp; r < RB; r += 4) {
        const int rr = b * RB + r, token = a.by_group.of(rr), hq = h * group + rr - token * group;
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
        const int e8 = (int)(__float_as_uint(big) >> 23);
        const int ex = big > 0.0f && e8 < 255 ? 140 - max(e8, 1) : 0;  // big 2^ex in [2^13, 2^14)
        const float up0 = pow2i(ex / 2), up1 = pow2i(ex - ex / 2);
        if (lane == 0) fr[r] = a.scale * 1.4426950408889634f * pow2i(-(ex / 2)) * pow2i(ex / 2 - ex);
#pragma unroll
        for (int i = 0; i < WPL; ++i) {
          const int w = lane + 32 * i, gq = w >> 2, tq = w & 3;
          if (w >= HDP / 8) continue;  // narrow heads: the lanes past the row
          float y[8], z[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = x[i][e] * up0 * up1;
            y[e] = __half2float(__float2half_rn(v));
            z[e] = v - y[e];
          }
          // product m of a group: columns (2m, 2m + 4) and (2m + 1, 2m + 5)
#pragma unroll
          for (int pt = 0; pt < L::PARTS; ++pt) {
            const float(&v)[8] = pt ? z : y;
            reinterpret_cast<uint4 *>(sm + L::OFF_Q + pt * L::QF)[(gq * NT + (r >> 3)) * 32 + (r & 7) * 4 + tq] =
                make_uint4(half2_bits(v[0], v[4]), half2_bits(v[1], v[5]), half2_bits(v[2], v[6]),
                           half2_bits(v[3], v[7]));
          }
        }
      }
    }
    int pos[NT][2];  // the position of this thread's rows, -1 for none
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = b * RB + nt * 8 + 2 * t4 + e, p = q.fill + a.by_group.of(rr);
        pos[nt][e] = rr < q.n * group && p < a.c.positions ? max(p, -1) : -1;
      }
    const int p_first = q.fill + a.by_group.of(b * RB);  // the first row's
    const int p_last = sp.hi - 1;
    const bool past = q.fill + min(q.n - 1, a.by_group.of((b + 1) * RB - 1)) >= a.c.positions;
    if (tid == 0 && (past || q.slot < 0)) pack_trouble(a.c);
    __syncthreads();

    // ---- the tiles
    float o[NT][NB * 4][4];  // [16 columns: two of them a thread][column, query row]
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m_run[nt][e] = -INFINITY, l_run[nt][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < NB * 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.0f;
    }
    for (int k = ka; k < kb; ++k) {
      const int turn = step0 + k - ka, slot = turn % NS;
      gave_up = !mbar_wait(&full[slot], (uint32_t)((turn / NS) & 1), gave_up ? PACK_TRIES / 64 : PACK_TRIES) || gave_up;
      const uint8_t *tk = sm + slot * L::SLOT, *tv = tk + L::CODE_SIDE;
      const uint16_t *ksc = reinterpret_cast<const uint16_t *>(tk + L::OFF_SC);
      const uint16_t *vsc = reinterpret_cast<const uint16_t *>(tk + L::OFF_SC + L::SC_SIDE);
      const int tile0 = sp.tile(k) * TP;
      const bool all = !past && tile0 + TP - 1 <= p_first &&
                       (a.window <= 0 || tile0 > p_last - a.window || tile0 + TP <= a.sinks);

      // scores
      float sc[MP][NT][4];
#pragma unroll
      for (int mp = 0; mp < MP; ++mp)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mp][nt][e] = 0.0f;
#pragma unroll 2
      for (int gr = 0; gr < C; ++gr) {
        uint32_t aw[MP][2][4];
        float st[MP][2];
#pragma unroll
        for (int mp = 0; mp < MP; ++mp) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(tk + (kat ^ ((gr & 7) << 4)) + (gr / 8) * L::CODE64 +
                                                                   (mp * 16 + 8 * e) * PITCH);
            uint32_t v[4];
            dequant_i4(w, v);
            aw[mp][0][e] = v[0];
            aw[mp][0][2 + e] = v[1];
            aw[mp][1][e] = v[2];
            aw[mp][1][2 + e] = v[3];
            st[mp][e] = FULL || gr < chd ? __half2float(__ushort_as_half(ksc[(r0 + mp * 16 + 8 * e) * chd + gr])) : 0.0f;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint4 qb[L::PARTS];
#pragma unroll
          for (int pt = 0; pt < L::PARTS; ++pt)
            qb[pt] = reinterpret_cast<const uint4 *>(sm + L::OFF_Q + pt * L::QF)[(gr * NT + nt) * 32 + lane];
#pragma unroll
          for (int mp = 0; mp < MP; ++mp) {
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (SP) {
              float low[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_add(low, aw[mp][0], qb[L::PARTS - 1].x, qb[L::PARTS - 1].y);
              mma_add(low, aw[mp][1], qb[L::PARTS - 1].z, qb[L::PARTS - 1].w);
              mma_add(acc, aw[mp][0], qb[0].x, qb[0].y);
              mma_add(acc, aw[mp][1], qb[0].z, qb[0].w);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[e] += low[e];
            } else {
              mma_add(acc, aw[mp][0], qb[0].x, qb[0].y);
              mma_add(acc, aw[mp][1], qb[0].z, qb[0].w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[mp][nt][e] = fmaf(acc[e], st[mp][e >> 1], sc[mp][nt][e]);
          }
        }
      }

      // softmax, in powers of two
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 f = *reinterpret_cast<const float2 *>(fr + nt * 8 + 2 * t4);
        float mx[2] = {-INFINITY, -INFINITY};
        if (all) {
#pragma unroll
          for (int mp = 0; mp < MP; ++mp)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sc[mp][nt][e] *= e & 1 ? f.y : f.x;
              mx[e & 1] = fmaxf(mx[e & 1], sc[mp][nt][e]);
            }
        } else {
#pragma unroll
          for (int mp = 0; mp < MP; ++mp)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = tile0 + r0 + mp * 16 + 8 * (e >> 1), p = pos[nt][e & 1];
              const bool see = j <= p && (a.window <= 0 || j > p - a.window || j < a.sinks);
              sc[mp][nt][e] = see ? sc[mp][nt][e] * (e & 1 ? f.y : f.x) : -INFINITY;
              mx[e & 1] = fmaxf(mx[e & 1], sc[mp][nt][e]);
            }
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], x));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], x));
        }
        if (g8 == 0) {
          wmax[(nt * 8 + 2 * t4) * 4 + warp] = mx[0];
          wmax[(nt * 8 + 2 * t4 + 1) * 4 + warp] = mx[1];
        }
      }
      __syncthreads();
      load(k + NS - 1);  // every warp is done with the step before, whose place this takes
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float al[2], base[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 w4 = *reinterpret_cast<const float4 *>(wmax + (nt * 8 + 2 * t4 + e) * 4);
          const float mx = fmaxf(fmaxf(fmaxf(w4.x, w4.y), fmaxf(w4.z, w4.w)), m_run[nt][e]);
          base[e] = mx == -INFINITY ? 0.0f : mx;
          al[e] = exp2_fast(m_run[nt][e] - base[e]);
          m_run[nt][e] = mx;
        }
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int mp = 0; mp < MP; ++mp) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // f32 rows: 2^12 the weight, so that its halves reach 2^-37 of the largest
            const float x = exp2_fast(sc[mp][nt][e] - base[e & 1]);
            sc[mp][nt][e] = SP ? x * 4096.0f : x;
            sum[e & 1] += sc[mp][nt][e];
          }
          // the weights turned to the second product's fragment: positions along its depth
          const uint32_t h0 = half2_bits(sc[mp][nt][0], sc[mp][nt][1]), h1 = half2_bits(sc[mp][nt][2], sc[mp][nt][3]);
          uint2 *p = reinterpret_cast<uint2 *>(sm + L::OFF_P) + ((warp * MP + mp) * NT + nt) * 32 + lane;
          *p = make_uint2(transpose8(h0), transpose8(h1));
          if (SP) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
            const uint32_t l0 = half2_bits(sc[mp][nt][0] - f0.x, sc[mp][nt][1] - f0.y);
            const uint32_t l1 = half2_bits(sc[mp][nt][2] - f1.x, sc[mp][nt][3] - f1.y);
            p[L::PF / 8] = make_uint2(transpose8(l0), transpose8(l1));
          }
        }
        l_run[nt][0] = l_run[nt][0] * al[0] + sum[0];
        l_run[nt][1] = l_run[nt][1] * al[1] + sum[1];
        if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f)) {
#pragma unroll
          for (int j = 0; j < NB * 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][j][e] *= al[e & 1];
        }
      }
      __syncthreads();

      // values
      constexpr int STEPS = TP / 16 / WP;
#pragma unroll(NT * NB <= 2 ? 2 : 1)
      for (int si = 0; si < STEPS; ++si) {
        const int st = wp * STEPS + si;
        const int r0v = vrow + si * 16;  // this thread's positions: r0v, + 1, + 8, + 9
        uint2 pb[L::PARTS][NT];
#pragma unroll
        for (int pt = 0; pt < L::PARTS; ++pt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            pb[pt][nt] = reinterpret_cast<const uint2 *>(sm + L::OFF_P + pt * L::PF)[(st * NT + nt) * 32 + lane];
        uint32_t live[2] = {0xffffffffu, 0xffffffffu};  // positions no row sees count as 0 whatever lies there
        if (!all) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int p = tile0 + r0v + 8 * i;
            const bool x = p < sp.hi && (p >= sp.lo || p < a.sinks);
            const bool y = p + 1 < sp.hi && (p + 1 >= sp.lo || p + 1 < a.sinks);
            live[i] = (x ? 0xffffu : 0u) | (y ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int cb = wc * NB + nb;  // 64 columns: groups 2 cb, 2 cb + 1
          uint32_t rows2[4];            // their scales at each position
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t *src = vsc + (r0v + (i & 1) + 8 * (i >> 1)) * chd + 2 * cb;
            if (FULL || (chd & 1) == 0) {
              rows2[i] = FULL || 2 * cb < chd ? *reinterpret_cast<const uint32_t *>(src) : 0u;
            } else {
              rows2[i] = (2 * cb < chd ? (uint32_t)src[0] : 0u) | (2 * cb + 1 < chd ? (uint32_t)src[1] << 16 : 0u);
            }
          }
#pragma unroll
          for (int gi = 0; gi < 2; ++gi) {
            uint32_t step[2], x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              step[i] = __byte_perm(rows2[2 * i], rows2[2 * i + 1], gi ? 0x7632 : 0x5410) & live[i];
              const uint8_t *box = tv + vhalf + (si * 16 + 8 * i) * PITCH;
              const uint32_t j = (nb * 2 + gi) << 4;
              const uint32_t w0 = *reinterpret_cast<const uint32_t *>(box + (vat[0] ^ j));
              const uint32_t w1 = *reinterpret_cast<const uint32_t *>(box + (vat[1] ^ j));
              x[i] = __byte_perm(w0, w1, zip);
            }
            // product u: columns 2u (rows 0-7) and 2u + 1 (rows 8-15) of the thread's four
            uint32_t av[2][4], al[2][4];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t v[4];
                dequant_i4(x[i], v);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const uint32_t c = v[2 * u + e];
                    if (SP) {
                      const uint32_t hi = mul2(c, step[i]);
                      av[u][2 * i + e] = hi;
                      al[u][2 * i + e] = rest2(c, step[i], hi);
                    } else {
                      av[u][2 * i + e] = c;
                    }
                  }
              }
            if (!SP) {
              step[0] = mul2(step[0], 0x48004800u);  // 8: weights of small scales stay above f16's smallest
              step[1] = mul2(step[1], 0x48004800u);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (SP) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  mma_add(acc, al[u], pb[0][nt].x, pb[0][nt].y);
                  mma_add(acc, av[u], pb[L::PARTS - 1][nt].x, pb[L::PARTS - 1][nt].y);
                  mma_add(acc, av[u], pb[0][nt].x, pb[0][nt].y);
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[nt][nb * 4 + gi * 2 + u][e] += acc[e];
                }
              } else {
                const uint32_t b0 = mul2(pb[0][nt].x, step[0]), b1 = mul2(pb[0][nt].y, step[1]);
#pragma unroll
                for (int u = 0; u < 2; ++u) mma_add(o[nt][nb * 4 + gi * 2 + u], av[u], b0, b1);
              }
            }
          }
        }
      }
    }
    step0 += kb - ka;
    if (!SP) {  // undo the 8 the weights carried
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < NB * 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][j][e] *= 0.125f;
    }

    // ---- the rows' sums, and of a narrow head the warps' shares, joined
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[nt][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        if (g8 == 0) wsum[(nt * 8 + 2 * t4 + e) * 4 + warp] = l;
      }
    __syncthreads();
    if (WP > 1) {
      float *buf = reinterpret_cast<float *>(sm);
      for (int r = 1; r < WP; ++r) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < NB * 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float *x = buf + (((nt * WC + wc) * NB * 4 + j) * 4 + e) * 32 + lane;
              if (wp == r) *x = o[nt][j][e];
            }
        __syncthreads();
        if (wp == 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < NB * 4; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][j][e] += buf[(((nt * WC + wc) * NB * 4 + j) * 4 + e) * 32 + lane];
        }
        __syncthreads();
      }
      fence_async_smem();  // the ring's next copies come after these reads
    }
    if (wp == 0) {
      const bool wide = wide_rows(a.out);
      float *pw = a.work + w.place * ((size_t)RB * (size + 2));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * t4 + e, rr = b * RB + r;
          if (rr >= q.n * group) continue;
          const float4 l4 = *reinterpret_cast<const float4 *>(wsum + r * 4);
          const float l = l4.x + l4.y + l4.z + l4.w;
          const float inv = whole ? (l == 0.0f ? 0.0f : __fdividef(1.0f, l)) : 1.0f;
          const int token = a.by_group.of(rr);
          const size_t to = (size_t)(q.first + token) * a.out.row_stride +
                            (size_t)(h * group + rr - token * group) * a.out.head_stride;
#pragma unroll
          for (int j = 0; j < NB * 2; ++j) {  // a group's four columns
            const int col = (wc * NB * 2 + j) * 32 + 4 * g8;
            if (col >= size) continue;
            const float x[4] = {o[nt][2 * j][e] * inv, o[nt][2 * j][2 + e] * inv, o[nt][2 * j + 1][e] * inv,
                                o[nt][2 * j + 1][2 + e] * inv};
            if (whole) store4(a.out.data, a.out.type, to + col, wide, x);
            else *reinterpret_cast<float4 *>(pw + (size_t)r * size + col) = make_float4(x[0], x[1], x[2], x[3]);
          }
          if (!whole && wc == 0 && g8 == 0) {
            pw[(size_t)RB * size + r] = m_run[nt][e];
            pw[(size_t)RB * size + RB + r] = l;
          }
        }
    }

    if (!walk_next<RB, TP>(a, spread, w)) break;
  }
  if (gave_up) pack_trouble(a.c);
}

// ---------------------------------------------------------------------------
// attention over the codes on tcgen05, for many 16-bit query rows
//
// A block holds 128 query rows of one (sequence, key/value head) and the
// whole of an SM's tensor memory: the rows' queries (f16, an operand), their
// results (f32), and two tiles of scores whose places the weights take.  The
// steps are tiles of 64 positions:
//
//   warps 4-7, 8-11  read a tile's key (value) codes a tile ahead into
//                    registers, turn them into f16((n - 8) scale) and store
//                    them in two operand buffers a side; rows of 64 columns
//                    (128 bytes, swizzled), one layout for both: the key
//                    operand's rows are its 8 KB blocks' rows, the value
//                    operand is read across them, so nothing is transposed.
//   warp 12          one thread issues scores (t + 1), then values (t), so
//                    that the softmax of a tile runs beside the products of
//                    its neighbours.
//   warps 0-3        a thread a row: the tile's 64 scores, their maximum, the
//                    weights back into tensor memory, the row's sum.  The
//                    results are rescaled only when the maximum has grown by
//                    more than 2^8 over the one in use; weights stay below
//                    f16's range until then.
//
// Columns of a group of eight keep the order their nibbles come out in,
// 0 4 1 5 2 6 3 7, in the queries and, undone at the end, in the results.
// A query row is scaled by an exact power of two as above; keys, values and
// weights are each rounded to f16 once (2^-11 at most).

template <int HDP>
struct PackTc {
  static constexpr int RB = 128, TP = 64, C = HDP / 32;
  static constexpr int BLOCKS = HDP / 64;               // 64-column blocks of an operand
  static constexpr int SIDE = BLOCKS * 64 * 128;        // one operand buffer
  static constexpr int T_Q = HDP, T_S = HDP + HDP / 2;  // tensor-memory columns: results, queries, scores
  static constexpr int SMEM = 1024 + (4 * SIDE > 116 * 1024 ? 4 * SIDE : 116 * 1024);  // one block an SM
  static constexpr int LW = C < 4 ? C : 4;              // groups across a warp's lanes
  static constexpr int ROWS = 32 / LW;                  // positions across them
  static constexpr int ITEMS = 64 * C / 128;            // groups a thread turns a tile
};

constexpr int TC_THREADS = 416;

__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t at, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tc_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_st32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// Operand descriptors, 128-byte swizzle, 8-row groups 1 KB apart: the key
// operand along its rows (K-major), and the value operand across them
// (MN-major: 64-column blocks 8 KB apart).
__device__ __forceinline__ uint64_t tc_desc(uint32_t at, uint32_t lead) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <int HDP>
__global__ void __launch_bounds__(TC_THREADS, 1)
    pack_attend_tc_kernel(const __grid_constant__ PackAttend a, int spread, int parts) {
  using L = PackTc<HDP>;
  constexpr int RB = L::RB, TP = L::TP, C = L::C;
  extern __shared__ __align__(1024) uint8_t tc_raw[];
  __shared__ int red[PACK_WARPS + 2];
  __shared__ uint64_t bars[14];
  __shared__ uint32_t tmem_slot;
  uint8_t *sm = tc_raw + ((1024 - (smem_u32(tc_raw) & 1023)) & 1023);
  // [side][buffer] filled by the code warps, and free again; scores ready;
  // weights ready; values added; queries ready
  uint64_t *full = bars, *empty = bars + 4, *sfull = bars + 8, *pfull = bars + 10, *vdone = bars + 12, *qfull = bars + 13;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int size = a.c.size, chd = size / 32, group = a.group;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&full[i], 128), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sfull[i], 1), mbar_init(&pfull[i], 128);
    mbar_init(vdone, 1);
    mbar_init(qfull, 128);
    mbar_init_fence();
  }
  PackWalk w;
  const bool any = walk_start<RB, TP>(a, spread, parts, w, red);
  pdl_release();
  if (any) walk_unit<RB, TP>(a, spread, parts, w);
  if (!any || (!spread && !w.whole && w.ka == w.kb)) return;
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    tc_before();
  }
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  int step0 = 0, unit = 0;  // steps and units before this one
  bool failed = false;
  auto wait = [&](uint64_t *bar, int phase) {
    if (!mbar_wait(bar, (uint32_t)(phase & 1), failed ? PACK_TRIES / 64 : PACK_TRIES)) failed = true;
  };

  for (;;) {
    const int steps = w.kb - w.ka;
    if (warp >= 12) {
      // ---- the products
      if (lane == 0 && steps > 0) {
        constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(TP >> 3) << 17) | ((uint32_t)(RB >> 4) << 24);
        constexpr uint32_t id_v =
            (1u << 4) | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | ((uint32_t)(RB >> 4) << 24);
        auto scores = [&](int t) {
          const int T = step0 + t, buf = T & 1;
          wait(&full[buf], T >> 1);
          tc_after();
          const uint32_t kb = smem_u32(sm + buf * L::SIDE);
#pragma unroll
          for (int i = 0; i < HDP / 16; ++i)
            tc_mma_ts(tmem + L::T_S + buf * 64, tmem + L::T_Q + i * 8, tc_desc(kb + (i / 4) * 8192 + (i & 3) * 32, 16),
                      id_s, i > 0);
          tc_commit(&sfull[buf]);
          tc_commit(&empty[buf]);
        };
        wait(qfull, unit);
        tc_after();
        scores(0);
        for (int t = 0; t < steps; ++t) {
          if (t + 1 < steps) scores(t + 1);
          const int T = step0 + t, buf = T & 1;
          wait(&full[2 + buf], T >> 1);
          wait(&pfull[buf], T >> 1);
          tc_after();
          const uint32_t vb = smem_u32(sm + (2 + buf) * L::SIDE);
#pragma unroll
          for (int i = 0; i < TP / 16; ++i)
            tc_mma_ts(tmem, tmem + L::T_S + buf * 64 + i * 8, tc_desc(vb + i * 2048, 8192), id_v, t > 0 || i > 0);
          tc_commit(&empty[2 + buf]);
          tc_commit(vdone);
        }
      }
      __syncwarp();
    } else if (warp >= 4) {
      // ---- codes to operands
      const int side = warp >= 8 ? 1 : 0, w4 = warp & 3;
      const int row_l = lane % L::ROWS, gr_l = lane / L::ROWS;
      const size_t base = ((size_t)max(w.q.slot, 0) * a.c.heads + w.h) * a.c.positions;
      const uint8_t *codes = (side ? a.c.vc : a.c.kc) + base * (size / 2);
      const uint16_t *scales = (side ? a.c.vs : a.c.ks) + base * chd;
      uint4 code[L::ITEMS];
      uint16_t scale[L::ITEMS];
      // item i: a position row and a group; eight neighbouring lanes hold
      // eight neighbouring rows, so that their stores spread over the banks
      auto row_of = [&](int i) { return (w4 + 4 * (i / (C / L::LW))) * L::ROWS + row_l; };
      auto group_of = [&](int i) { return gr_l + L::LW * (i % (C / L::LW)); };
      auto fetch = [&](int t) {
        if (t >= steps) return;
        const int p0 = w.sp.tile(w.ka + t) * TP;
#pragma unroll
        for (int i = 0; i < L::ITEMS; ++i) {
          const int p = p0 + row_of(i), gr = group_of(i);
          code[i] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
          scale[i] = 0;
          // a position no row sees counts as 0 whatever lies there
          if (gr < chd && p < w.sp.hi && (p >= w.sp.lo || p < a.sinks)) {
            code[i] = __ldg(reinterpret_cast<const uint4 *>(codes + (size_t)p * (size / 2)) + gr);
            scale[i] = __ldg(scales + (size_t)p * chd + gr);
          }
        }
      };
      fetch(0);
      for (int t = 0; t < steps; ++t) {
        const int T = step0 + t, buf = T & 1;
        uint4 now[L::ITEMS];
        uint32_t by[L::ITEMS];
#pragma unroll
        for (int i = 0; i < L::ITEMS; ++i) now[i] = code[i], by[i] = scale[i] | ((uint32_t)scale[i] << 16);
        fetch(t + 1);
        if (T >= 2) wait(&empty[side * 2 + buf], (T >> 1) - 1);
        uint8_t *dst = sm + (side * 2 + buf) * L::SIDE;
#pragma unroll
        for (int i = 0; i < L::ITEMS; ++i) {
          const int r = row_of(i), gr = group_of(i);
          uint8_t *to = dst + (gr >> 1) * 8192 + r * 128;
          const uint32_t words[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t v[4];
            dequant_i4(words[k], v);
            *reinterpret_cast<uint4 *>(to + ((((gr & 1) * 4 + k) ^ (r & 7)) << 4)) =
                make_uint4(mul2(v[0], by[i]), mul2(v[1], by[i]), mul2(v[2], by[i]), mul2(v[3], by[i]));
          }
        }
        fence_async_smem();  // written here, read by the tensor core (async proxy)
        mbar_arrive(&full[side * 2 + buf]);
      }
    } else {
      // ---- the softmax, a thread a row
      const int rr = w.b * RB + tid, token = a.by_group.of(rr), hq = w.h * group + rr - token * group;
      const bool live = rr < w.q.n * group;
      const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
      const int p_row = w.q.fill + token;
      const int pos = live && p_row < a.c.positions ? max(p_row, -1) : -1;
      const int t_last = min(w.q.n - 1, a.by_group.of((w.b + 1) * RB - 1));
      const bool past = w.q.fill + t_last >= a.c.positions;
      const int p_first = w.q.fill + a.by_group.of(w.b * RB), p_last = w.sp.hi - 1;
      if (tid == 0 && (past || w.q.slot < 0)) pack_trouble(a.c);
      float f = 0.0f;
      if (steps > 0) {
        const bool wide = wide_rows(a.q);
        const size_t from = (size_t)(w.q.first + token) * a.q.row_stride + (size_t)hq * a.q.head_stride;
        float big = 0.0f;
        if (live)
          for (int c = 0; c < size; c += 8) {
            float x[8];
            load8(a.q.data, a.q.type, from + c, wide, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
          }
        const int e8 = (int)(__float_as_uint(big) >> 23);
        const int ex = big > 0.0f && e8 < 255 ? 140 - max(e8, 1) : 0;  // big 2^ex in [2^13, 2^14)
        // the scale's sign goes with the queries, so that the largest score is the largest weight's
        const float up0 = pow2i(ex / 2), up1 = (a.scale < 0.0f ? -1.0f : 1.0f) * pow2i(ex - ex / 2);
        f = fabsf(a.scale) * 1.4426950408889634f * pow2i(-(ex / 2)) * pow2i(ex / 2 - ex);
        for (int c0 = 0; c0 < HDP; c0 += 64) {
          uint32_t r[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float x[8] = {};
            if (live && c0 + 8 * k < size) load8(a.q.data, a.q.type, from + c0 + 8 * k, wide, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) r[4 * k + e] = half2_bits(x[e] * up0 * up1, x[e + 4] * up0 * up1);
          }
          tc_st32(lanes + L::T_Q + c0 / 2, r);
        }
        tc_st_wait();
        tc_before();
        mbar_arrive(qfull);
      }
      float m = -INFINITY, l = 0.0f;  // the maximum in use (of scores as the products leave them)
      for (int t = 0; t < steps; ++t) {
        const int T = step0 + t, buf = T & 1;
        wait(&sfull[buf], T >> 1);
        tc_after();
        uint32_t lo[32], hi[32];
        tc_ld32(lanes + L::T_S + buf * 64, lo);
        tc_ld32(lanes + L::T_S + buf * 64 + 32, hi);
        tc_ld_wait();
        const int tile0 = w.sp.tile(w.ka + t) * TP;
        const bool all = !past && tile0 + TP - 1 <= p_first &&
                         (a.window <= 0 || tile0 > p_last - a.window || tile0 + TP <= a.sinks);
        if (!all) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int j = tile0 + i;
            if (!(j <= pos && (a.window <= 0 || j > pos - a.window || j < a.sinks))) lo[i] = 0xff800000u;
            if (!(j + 32 <= pos && (a.window <= 0 || j + 32 > pos - a.window || j + 32 < a.sinks))) hi[i] = 0xff800000u;
          }
        }
        float mx[4] = {m, m, m, m};
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          mx[0] = fmaxf(mx[0], __uint_as_float(lo[i]));
          mx[1] = fmaxf(mx[1], __uint_as_float(lo[i + 1]));
          mx[2] = fmaxf(mx[2], __uint_as_float(hi[i]));
          mx[3] = fmaxf(mx[3], __uint_as_float(hi[i + 1]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool grown = top > m && (m == -INFINITY || (top - m) * f > 8.0f);
        if (__any_sync(0xffffffffu, grown)) {
          const float back = grown ? (m == -INFINITY ? 0.0f : exp2_fast((m - top) * f)) : 1.0f;
          if (grown) m = top;
          l *= back;
          if (t > 0) {
            wait(vdone, T - 1);
            tc_after();
#pragma unroll 1
            for (int c = 0; c < HDP; c += 32) {
              uint32_t r[32];
              tc_ld32(lanes + c, r);
              tc_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * back);
              tc_st32(lanes + c, r);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t p[32];
        auto weight = [&](uint32_t x) {
          const float y = exp2_fast((__uint_as_float(x) - base) * f);  // 0 at the largest, however large
          return all || x != 0xff800000u ? y : 0.0f;
        };
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float x = weight(lo[i]), y = weight(lo[i + 1]);
          p[i / 2] = half2_bits(x, y);
          sum[0] += x;
          sum[1] += y;
          const float z = weight(hi[i]), v = weight(hi[i + 1]);
          p[16 + i / 2] = half2_bits(z, v);
          sum[2] += z;
          sum[3] += v;
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tc_st32(lanes + L::T_S + buf * 64, p);
        tc_st_wait();
        tc_before();
        mbar_arrive(&pfull[buf]);
      }
      // ---- the rows out
      if (steps > 0) {
        wait(vdone, step0 + steps - 1);
        tc_after();
      }
      const bool wide = wide_rows(a.out);
      const float inv = w.whole ? (l == 0.0f ? 0.0f : __fdividef(1.0f, l)) : 1.0f;
      float *pw = a.work + w.place * ((size_t)RB * (size + 2));
      const size_t to = (size_t)(w.q.first + token) * a.out.row_stride + (size_t)hq * a.out.head_stride;
#pragma unroll 1
      for (int c = 0; c < size; c += 32) {
        uint32_t r[32];
        if (steps > 0) {
          tc_ld32(lanes + c, r);
          tc_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        }
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x[8] = {__uint_as_float(r[8 * k]) * inv,     __uint_as_float(r[8 * k + 2]) * inv,
                              __uint_as_float(r[8 * k + 4]) * inv, __uint_as_float(r[8 * k + 6]) * inv,
                              __uint_as_float(r[8 * k + 1]) * inv, __uint_as_float(r[8 * k + 3]) * inv,
                              __uint_as_float(r[8 * k + 5]) * inv, __uint_as_float(r[8 * k + 7]) * inv};
          if (w.whole) store8(a.out.data, a.out.type, to + c + 8 * k, wide, x);
          else store8(pw, 1, (size_t)tid * size + c + 8 * k, true, x);
        }
      }
      if (!w.whole && live) {
        pw[(size_t)RB * size + tid] = m == -INFINITY ? -INFINITY : m * f;
        pw[(size_t)RB * size + RB + tid] = l;
      }
      tc_before();
    }
    step0 += steps;
    ++unit;
    if (!walk_next<RB, TP>(a, spread, w)) break;
    walk_unit<RB, TP>(a, spread, parts, w);
  }
  if (failed) pack_trouble(a.c);
  __syncthreads();
  if (warp == 12) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ---------------------------------------------------------------------------
// the pieces of a unit joined, and rows that see nothing set to zero: a block
// a row, its threads four columns each and, of narrow heads, every second or
// fourth (eighth) piece; each column's pieces are added in a fixed order

struct PackMerge {
  PackAttend a;
  int rb, tp, spread, parts, grid, blocks;
};

constexpr int PM_THREADS = 128, PM_CHUNK = 256;  // pieces whose factors are kept at a time

__global__ void __launch_bounds__(PM_THREADS) pack_merge_kernel(PackMerge g) {
  __shared__ int red[PACK_WARPS + 2];
  __shared__ float pm[PM_CHUNK], pl[PM_CHUNK];
  __shared__ float4 part4[PM_THREADS];
  const PackAttend &a = g.a;
  const int RB = g.rb, TP = g.tp, size = a.c.size, tid = threadIdx.x;
  int u = blockIdx.x, s, b, h = u % a.c.heads, first, last, share = 0, n;
  SeqAt q;
  u /= a.c.heads;
  const int r = blockIdx.y;
  if (g.spread) {
    s = u / g.blocks;
    b = u - s * g.blocks;
    q = seq_at(a.c, a.r, s);
    if (b * RB + r >= q.n * a.group) return;
    int before;
    const int total = list_total(a, RB, TP, true, s, &before, red);
    share = share_of(total, g.grid);
    for (int i = 0; i < b; ++i) before += block_span(a, q, i, RB, TP).count() * a.c.heads;
    n = block_span(a, q, b, RB, TP).count();
    before += h * n;
    first = before / share;
    last = (before + max(n, 1) - 1) / share;
    if (n > 0 && first == last) return;  // one block had it all
    u = before;
  } else {
    const int total = list_total(a, RB, TP, false, 0, nullptr, red);
    if (u >= total) return;
    const ListAt f = list_at(a, RB, TP, false, total - 1 - u, red);
    s = f.s;
    if (s < 0) return;
    b = total - 1 - u - f.before;
    q = seq_at(a.c, a.r, s);
    if (b * RB + r >= q.n * a.group) return;
    n = block_span(a, q, b, RB, TP).count();
    first = 0;
    last = g.parts - 1;
    u = blockIdx.x * g.parts;
  }
  const int rr = b * RB + r, token = a.by_group.of(rr);
  const size_t piece = (size_t)RB * (size + 2);
  auto place = [&](int i) {
    return g.spread ? 2 * (size_t)i + (i * share <= u ? 1 : 0)  // the piece with the unit's first tile
                    : (size_t)u + i;
  };
  const int lanes = size / 4, teams = PM_THREADS / lanes, team = tid / lanes, col = 4 * (tid - team * lanes);
  float m = -INFINITY, l = 0.0f;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  pdl_wait();
  for (int c0 = first; n > 0 && c0 <= last; c0 += PM_CHUNK) {
    const int cn = min(PM_CHUNK, last + 1 - c0);
    float mx = m;
    __syncthreads();
    for (int i = tid; i < cn; i += PM_THREADS) {
      const int p = c0 + i;
      const bool none = !g.spread && (long)n * p / g.parts == (long)n * (p + 1) / g.parts;
      const float *pw = a.work + place(p) * piece + (size_t)RB * size + r;
      const float y = none ? 0.0f : pw[RB];
      pl[i] = y;
      pm[i] = y == 0.0f ? -INFINITY : pw[0];  // a piece that saw none of the row's positions
    }
    __syncthreads();
    for (int i = 0; i < cn; ++i) mx = fmaxf(mx, pm[i]);
    const float base = mx == -INFINITY ? 0.0f : mx;
    const float back = exp2_fast(m - base);
    m = mx;
    l *= back;
    x.x *= back, x.y *= back, x.z *= back, x.w *= back;
    for (int i = 0; i < cn; ++i) {
      const float y = pl[i];
      if (y != 0.0f) l += y * exp2_fast(pm[i] - base);
    }
    if (team < teams) {
#pragma unroll 4
      for (int i = team; i < cn; i += teams) {
        if (pl[i] == 0.0f) continue;
        const float f = exp2_fast(pm[i] - base);
        const float4 y = *reinterpret_cast<const float4 *>(a.work + place(c0 + i) * piece + (size_t)r * size + col);
        x.x = fmaf(y.x, f, x.x);
        x.y = fmaf(y.y, f, x.y);
        x.z = fmaf(y.z, f, x.z);
        x.w = fmaf(y.w, f, x.w);
      }
    }
  }
  part4[tid] = x;
  __syncthreads();
  if (n == 0 && tid == 0 && (q.slot < 0 || q.fill + token >= a.c.positions)) pack_trouble(a.c);
  if (team != 0) return;
  for (int i = 1; i < teams; ++i) {
    const float4 y = part4[i * lanes + tid];
    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
  }
  const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
  const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
  store4(a.out.data, a.out.type,
         (size_t)(q.first + token) * a.out.row_stride +
             (size_t)(h * a.group + rr - token * a.group) * a.out.head_stride + col,
         wide_rows(a.out), y);
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

template <int HDP, int NT, bool SP, bool FULL>
cudaError_t pack_form_ready(PackPlan *plan, int *per_sm) {
  using L = PackTile<HDP, NT, SP>;
  plan->tile = L::TP;
  plan->pitch = L::PITCH;
  static std::atomic<int> known[PACK_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < PACK_DEVICES && (*per_sm = known[dev].load()) > 0) return cudaSuccess;
  auto kern = pack_attend_kernel<HDP, NT, SP, FULL>;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kern, 128, L::SMEM);
  if (e == cudaSuccess && *per_sm < 1) e = cudaErrorInvalidConfiguration;
  if (e == cudaSuccess && dev < PACK_DEVICES) known[dev].store(*per_sm);
  return e;
}

template <int HDP, int NT, bool SP, bool FULL>
cudaError_t pack_form_launch(const PackAttend &a, const PackPlan &p, const CUtensorMap &tmk, const CUtensorMap &tmv,
                             cudaStream_t st) {
  return pack_launch(pack_attend_kernel<HDP, NT, SP, FULL>, dim3(p.grid), 128, PackTile<HDP, NT, SP>::SMEM, st, false, a,
                     tmk, tmv, p.spread, p.parts);
}

// Calls F for the form a plan names.
#define PACK_FORMS(F, p, ...) \
  switch ((p).wide * 32 + (p).rows8 * 4 + (p).split2 * 2 + (p).full) { \
    case 2053: return F<64, 1, false, true>(__VA_ARGS__); \
    case 2057: return F<64, 2, false, true>(__VA_ARGS__); \
    case 2055: return F<64, 1, true, true>(__VA_ARGS__); \
    case 2059: return F<64, 2, true, true>(__VA_ARGS__); \
    case 2067: return F<64, 4, true, true>(__VA_ARGS__); \
    case 4101: return F<128, 1, false, true>(__VA_ARGS__); \
    case 4105: return F<128, 2, false, true>(__VA_ARGS__); \
    case 4103: return F<128, 1, true, true>(__VA_ARGS__); \
    case 4107: return F<128, 2, true, true>(__VA_ARGS__); \
    case 4115: return F<128, 4, true, true>(__VA_ARGS__); \
    case 8197: return F<256, 1, false, true>(__VA_ARGS__); \
    case 8201: return F<256, 2, false, true>(__VA_ARGS__); \
    case 8199: return F<256, 1, true, true>(__VA_ARGS__); \
    case 8203: return F<256, 2, true, true>(__VA_ARGS__); \
    case 8211: return F<256, 4, true, true>(__VA_ARGS__); \
    case 16389: return F<512, 1, false, true>(__VA_ARGS__); \
    case 16393: return F<512, 2, false, true>(__VA_ARGS__); \
    case 16401: return F<512, 4, false, true>(__VA_ARGS__); \
    case 16391: return F<512, 1, true, true>(__VA_ARGS__); \
    case 16395: return F<512, 2, true, true>(__VA_ARGS__); \
    case 2052: return F<64, 1, false, false>(__VA_ARGS__); \
    case 2056: return F<64, 2, false, false>(__VA_ARGS__); \
    case 2054: return F<64, 1, true, false>(__VA_ARGS__); \
    case 2066: return F<64, 4, true, false>(__VA_ARGS__); \
    case 4100: return F<128, 1, false, false>(__VA_ARGS__); \
    case 4104: return F<128, 2, false, false>(__VA_ARGS__); \
    case 4102: return F<128, 1, true, false>(__VA_ARGS__); \
    case 4114: return F<128, 4, true, false>(__VA_ARGS__); \
    case 8196: return F<256, 1, false, false>(__VA_ARGS__); \
    case 8200: return F<256, 2, false, false>(__VA_ARGS__); \
    case 8198: return F<256, 1, true, false>(__VA_ARGS__); \
    case 8210: return F<256, 4, true, false>(__VA_ARGS__); \
    case 16388: return F<512, 1, false, false>(__VA_ARGS__); \
    case 16400: return F<512, 4, false, false>(__VA_ARGS__); \
    case 16390: return F<512, 1, true, false>(__VA_ARGS__); \
    case 16394: return F<512, 2, true, false>(__VA_ARGS__); \
    default: return cudaErrorInvalidValue; \
  }

template <int HDP>
cudaError_t pack_tc_ready(PackPlan *plan) {
  static std::atomic<int> known[PACK_DEVICES];
  plan->tile = PackTc<HDP>::TP;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < PACK_DEVICES && known[dev].load())) return e;
  e = cudaFuncSetAttribute(pack_attend_tc_kernel<HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackTc<HDP>::SMEM);
  if (e == cudaSuccess && dev < PACK_DEVICES) known[dev].store(1);
  return e;
}

static cudaError_t pack_form(PackPlan *p, int *per_sm) {
  if (p->tc) {
    *per_sm = 1;
    return p->wide == 64 ? pack_tc_ready<64>(p) : p->wide == 128 ? pack_tc_ready<128>(p) : pack_tc_ready<256>(p);
  }
  PACK_FORMS(pack_form_ready, *p, p, per_sm)
}
static cudaError_t pack_run(const PackPlan &p, const PackAttend &a, const CUtensorMap &tmk, const CUtensorMap &tmv,
                            cudaStream_t st) {
  PACK_FORMS(pack_form_launch, p, a, p, tmk, tmv, st)
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
  int most8 = p->split2 ? 4 : 2;  // what registers hold, and past 16 rows the tcgen05 form takes over
  if (p->wide == 512) most8 = p->split2 ? 2 : 4;
  p->full = size == p->wide;
  p->rows8 = need <= 8 ? 1 : need <= 16 && p->full ? 2 : most8;  // fewer forms where a group's tile is part empty
  if (!p->split2 && p->wide <= 256 && need > 16) {
    p->tc = 1;
    p->rows8 = 16;
  }
  const int rb = 8 * p->rows8;
  int sms = 0, per_sm = 0;
  cudaError_t e = pack_sms(&sms);
  if (e == cudaSuccess) e = pack_form(p, &per_sm);
  if (e != cudaSuccess) return e;
  const long blocks = (need + rb - 1) / rb;
  const long slots = (long)sms * per_sm;
  // the most tiles a unit can have: its rows' reach, wherever it starts in a tile
  const long reach = window > 0 ? (long)window + rb / group + 1 + sinks + 3 * p->tile : positions;
  const long tiles = ((reach < positions ? reach : positions) + p->tile - 1) / p->tile;
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

// The tensor map of one side's codes: [slot, head, position][size / 2] bytes
// in boxes of 64 positions by `pitch` bytes, swizzled over the pitch; columns
// past the head arrive as zeros.  Host only.
static cudaError_t pack_map(const PackView &c, const void *codes, int pitch, CUtensorMap *map) {
  static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> known{nullptr};
  PFN_cuTensorMapEncodeTiled_v12000 encode = known.load();
  if (!encode) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (found != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    known.store(encode);
  }
  const cuuint64_t dims[2] = {(cuuint64_t)c.size / 2, (cuuint64_t)c.slots * c.heads * c.positions};
  const cuuint64_t strides[1] = {(cuuint64_t)c.size / 2};
  const cuuint32_t box[2] = {(cuuint32_t)pitch, 64}, step[2] = {1, 1};
  const CUtensorMapSwizzle swz = pitch == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                 : pitch == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                               : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t igc_launch_pack_attend(const PackAttend *a, const PackPlan *p, cudaStream_t st, int *launches) {
  *launches = 0;
  cudaError_t e;
  if (p->tc) {
    auto run = [&](auto kern, int smem) {
      return pack_launch(kern, dim3(p->grid), TC_THREADS, smem, st, false, *a, p->spread, p->parts);
    };
    e = p->wide == 64    ? run(pack_attend_tc_kernel<64>, PackTc<64>::SMEM)
        : p->wide == 128 ? run(pack_attend_tc_kernel<128>, PackTc<128>::SMEM)
                         : run(pack_attend_tc_kernel<256>, PackTc<256>::SMEM);
  } else {
    CUtensorMap tmk, tmv;
    e = pack_map(a->c, a->c.kc, p->pitch, &tmk);
    if (e == cudaSuccess) e = pack_map(a->c, a->c.vc, p->pitch, &tmv);
    if (e == cudaSuccess) e = pack_run(*p, *a, tmk, tmv, st);
  }
  *launches = 1;
  if (e != cudaSuccess || (!p->spread && p->parts == 1)) return e;
  *launches = 2;
  const PackMerge g = {*a, 8 * p->rows8, p->tile, p->spread, p->parts, p->grid, p->blocks};
  return pack_launch(pack_merge_kernel, dim3((unsigned)p->units, 8 * p->rows8), PM_THREADS, 0, st, true, g);
}
