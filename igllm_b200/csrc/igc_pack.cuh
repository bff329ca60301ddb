// igc_pack.cuh - device code shared by the packed cache's kernels (igc_pack.cu,
// igc_pack_tc.cu): a call's rows, rows of values, and how blocks share out
// the tiles of positions that the rows see.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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
// small things

constexpr int PACK_TRIES = 1 << 22;  // polls a wait makes before it gives up

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

// What lies at `p` in the shared memory of cluster block `rank`.
__device__ __forceinline__ uint32_t cluster_at(const float *p, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ float cluster_ld(const float *p, int rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(x) : "r"(cluster_at(p, rank)) : "memory");
  return x;
}
__device__ __forceinline__ float4 cluster_ld4(const float *p, int rank) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(cluster_at(p, rank))
               : "memory");
  return x;
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

// ---------------------------------------------------------------------------
// who takes which tiles
//
// A unit is one block of RB query rows of one (sequence, key/value head).  All
// units' tiles, in order, are one list that the launch's blocks share out
// evenly, so that sequences of any lengths load them alike; a block's run may
// begin and end inside units.  What a unit costs beside its tiles (its queries
// in, its results out) counts as `over` tiles before its own.
// A unit cut between blocks leaves partial sums (the maximum, the sum and the
// unnormalised result of each row) that pack_merge_kernel joins.

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

// The steps a unit counts for.
__device__ __forceinline__ int unit_weight(const PackAttend &a, const SeqAt &q, int b, int rb, int tp, int over) {
  return over + block_span(a, q, b, rb, tp).count();
}

__device__ __forceinline__ int seq_weight(const PackAttend &a, int s, int rb, int tp, int over) {
  if (s >= a.r.count) return 0;
  const SeqAt q = seq_at(a.c, a.r, s);
  const int nb = blocks_of(a, q, rb);
  int w = 0;
  for (int b = 0; b < nb; ++b) w += unit_weight(a, q, b, rb, tp, over);
  return w * a.c.heads;
}

// Every warp finds its place by itself: 32 sequences at a time, or (tall)
// sequence by sequence 32 of its blocks at a time.  -1 where the list weighs
// more than list_most, as a list of starts that goes back and forth gives rows
// to many sequences: none of it is run, which bounds what a call does and keeps
// every sum in 31 bits (a sequence's weight is below list_most, a lane's sum
// below twice that, and the warp's is first taken in 64ths).
__device__ __forceinline__ int list_total(const PackAttend &a, int rb, int tp, int over, int tall) {
  const int lane = threadIdx.x & 31;
  uint32_t w = 0;
  const uint32_t most = (uint32_t)a.list_most;
  if (!tall) {
    for (int i = lane; i < a.r.count; i += 32) w = min(w, most) + (uint32_t)seq_weight(a, i, rb, tp, over);
  } else {
    for (int s = 0; s < a.r.count; ++s) {
      const SeqAt q = seq_at(a.c, a.r, s);
      const int nb = blocks_of(a, q, rb);
      for (int b = lane; b < nb; b += 32) w = min(w, most) + (uint32_t)(unit_weight(a, q, b, rb, tp, over) * a.c.heads);
      if (__any_sync(0xffffffffu, w > most)) break;
    }
  }
  if (__reduce_add_sync(0xffffffffu, w >> 6) > (most >> 6)) return -1;
  w = __reduce_add_sync(0xffffffffu, w);
  return w > most ? -1 : (int)w;
}

// Among 32 weights, a lane each, after `before` in all: the lane that holds
// `want`, or -1; `before` moves on to the weight before that lane, or past all.
__device__ __forceinline__ int lane_holding(int w, int want, int *before) {
  const int lane = threadIdx.x & 31;
  int x = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  const uint32_t past = __ballot_sync(0xffffffffu, *before + x > want);
  const int l = __ffs(past) - 1;
  *before += __shfl_sync(0xffffffffu, past ? x - w : x, past ? l : 31);
  return l;
}

// A block's way through its run of the list.
struct PackWalk {
  int at, end, took;     // of the list; `took` of it by the unit
  int s, b, h, ka, kb;   // the unit, and its steps [ka, kb) that are this block's
  bool whole;            // all of them
  int first, last;       // the blocks that share its tiles
  SeqAt q;
  TileSpan sp;
};

// The unit from `part` of its weight on; false where no step of it is the block's.
template <int RB, int TP, int OVER>
__device__ __forceinline__ bool walk_piece(const PackAttend &a, PackWalk &w, int part, int share) {
  w.sp = block_span(a, w.q, w.b, RB, TP);
  const int n = w.sp.count();
  w.took = min(n + OVER - part, w.end - w.at);
  w.ka = max(0, part - OVER);
  w.kb = max(0, part + w.took - OVER);
  w.whole = w.ka == 0 && w.kb == n;
  w.first = (w.at - part + OVER) / share;
  w.last = (w.at - part + OVER + n - 1) / share;
  return w.whole || w.ka < w.kb;
}

// On to the next unit; false at the end.
template <int RB, int TP, int OVER>
__device__ __forceinline__ bool walk_next(const PackAttend &a, PackWalk &w, int share) {
  do {
    w.at += w.took;
    if (w.at >= w.end) return false;
    if (++w.h == a.c.heads) {
      w.h = 0;
      ++w.b;
      while (w.b >= blocks_of(a, w.q, RB)) {
        w.b = 0;
        if (++w.s >= a.r.count) return false;
        w.q = seq_at(a.c, a.r, w.s);
      }
    }
  } while (!walk_piece<RB, TP, OVER>(a, w, 0, share));
  return true;
}

// The block's first unit; false where it has none.
template <int RB, int TP, int OVER>
__device__ __forceinline__ bool walk_start(const PackAttend &a, int tall, PackWalk &w, int *share_out) {
  const int lane = threadIdx.x & 31;
  const int total = list_total(a, RB, TP, OVER, tall), share = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  *share_out = share;
  w.at = blockIdx.x * share;
  w.end = min(total, w.at + share);
  if (total < 0) pack_trouble(a.c);
  if (w.at >= w.end) return false;
  int before = 0, l = -1;
  if (!tall) {
    for (int base = 0; base < a.r.count && l < 0; base += 32) {
      w.s = base;
      l = lane_holding(seq_weight(a, base + lane, RB, TP, OVER), w.at, &before);
    }
    if (l < 0) return false;
    w.s += l;
    w.q = seq_at(a.c, a.r, w.s);
    const int nb = blocks_of(a, w.q, RB);
    for (w.b = 0; w.b < nb; ++w.b) {
      const int n = unit_weight(a, w.q, w.b, RB, TP, OVER) * a.c.heads;
      if (w.at - before < n) break;
      before += n;
    }
    if (w.b >= nb) return false;
  } else {
    for (w.s = 0; w.s < a.r.count; ++w.s) {
      w.q = seq_at(a.c, a.r, w.s);
      const int nb = blocks_of(a, w.q, RB);
      for (w.b = 0; w.b < nb && l < 0; w.b += 32) {
        l = lane_holding(w.b + lane < nb ? unit_weight(a, w.q, w.b + lane, RB, TP, OVER) * a.c.heads : 0, w.at, &before);
        if (l >= 0) w.b += l - 32;
      }
      if (l >= 0) break;
    }
    if (l < 0) return false;
  }
  const int n = unit_weight(a, w.q, w.b, RB, TP, OVER);
  w.h = (w.at - before) / n;
  return walk_piece<RB, TP, OVER>(a, w, w.at - before - w.h * n, share) || walk_next<RB, TP, OVER>(a, w, share);
}

// What a block leaves for the merge about the unit it begins inside (first:
// the block that holds the unit's beginning, -2 where there is none).
struct PackCut {
  int first, last, q_first, q_n, b, h, pad[2];
};
__device__ __forceinline__ void leave_cut(const PackAttend &a, const PackWalk &w, bool any) {
  PackCut c;
  c.first = any && w.ka > 0 ? w.first : -2;
  c.last = w.last;
  c.q_first = w.q.first;
  c.q_n = w.q.n;
  c.b = w.b;
  c.h = w.h;
  c.pad[0] = c.pad[1] = 0;
  reinterpret_cast<PackCut *>(a.work)[blockIdx.x] = c;
}

// Partial sums of piece `i` of `grid` blocks': [RB][size] results, [RB] maxima,
// [RB] sums.  A block leaves at most two: of the unit it begins inside (2
// block), and of the one it ends inside (2 block + 1).
__device__ __forceinline__ float *piece_at(const PackAttend &a, int grid, int rb, size_t i) {
  return a.work + (size_t)grid * (sizeof(PackCut) / 4) + i * ((size_t)rb * (a.c.size + 2));
}

// `overlap`: may start before the kernel ahead ends; `cluster`: blocks of one (0: none).
template <typename... P, typename... Q>
cudaError_t pack_launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool overlap,
                        int cluster, Q... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  cfg.attrs = at;
  if (overlap) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    at[cfg.numAttrs].val.clusterDim.y = 1;
    at[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

constexpr int PACK_DEVICES = 64;  // devices whose forms are looked up once

}  // namespace igc
