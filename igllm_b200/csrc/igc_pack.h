// igc_pack.h - host-side launchers of igc_pack.cu: the 4-bit key/value cache.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace igc {

constexpr int PACK_GROUP = 32;  // columns that share a scale
constexpr int PACK_TILE = 64;   // positions a tile; a slot holds a whole number of them

// A packed cache in device memory: codes [slot][head][position][size / 2]
// bytes, scales [slot][head][position][size / 32] f16.
struct PackView {
  uint8_t *kc, *vc;
  uint16_t *ks, *vs;
  int slots, heads, positions, size;
  int *trouble;  // set nonzero where a call names a place outside the cache (nullable)
};

// The rows of a call: sequence s has rows [starts[s], starts[s + 1]) (or, with
// no starts, s * per .. + per), at positions fill[s] + i of slot slots[s] (or s).
// No sequence has more than `most`.
struct PackRows {
  int count, rows, per, most;
  const int *starts, *fill, *slots;
};

// Rows of values, `type` 1 f32, 2 f16, 3 bf16; strides in values.
struct PackData {
  void *data;
  int type;
  long row_stride, head_stride;
};

// Quotients by a number known at the launch: n / d for 0 <= n < 2^31 as
// (hi32(n mul) + n) >> shift, mul = floor(2^32 (2^shift - d) / d) + 1, 2^shift
// the power of two from d on (Granlund and Montgomery, 1994).
struct Quotient {
  uint32_t mul, shift;
#ifdef __CUDACC__
  __device__ __forceinline__ int of(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
#endif
  static Quotient by(int d) {
    uint32_t s = 0;
    while ((1ull << s) < (uint64_t)d) ++s;
    return Quotient{(uint32_t)(((1ull << 32) * ((1ull << s) - (uint64_t)d)) / (uint64_t)d + 1), s};
  }
};

struct PackAttend {
  PackView c;
  PackRows r;
  PackData q, out;
  int group;          // query heads a key/value head
  Quotient by_group;
  int window, sinks;  // window 0: every position up to the row's own
  float scale;
  float *work;        // split units' partial sums (PackPlan::work_floats)
  int list_most;      // PackPlan::list_most
};

// How a call's attention runs, from its host-known sizes alone.
struct PackPlan {
  int rows8;     // eights of query rows a block holds (1, 2 or 4, with tc 16)
  int tc;        // the tcgen05 form
  int wide;      // head width the kernel is built for: 64, 128, 256 or 512
  int split2;    // f32 rows: hi and lo halves of both operands
  int full;      // the head fills that width
  int tile;      // positions a step
  int over;      // steps a unit costs beside its own
  int pitch;     // code bytes of a row of a TMA box
  int tall;      // some sequence has many blocks of rows; with clusters, the most of any
  int cluster;   // blocks of a cluster that share a unit, 0: the list of tiles instead
  int grid;
  int list_most;  // the most the list of tiles weighs where no two sequences hold one row
  size_t work_floats;
};

}  // namespace igc

extern "C" {
cudaError_t igc_launch_pack_write(const igc::PackView *c, const igc::PackRows *r, const igc::PackData *k,
                                  const igc::PackData *v, cudaStream_t st);
cudaError_t igc_launch_pack_read(const igc::PackView *c, const igc::PackRows *r, const igc::PackData *k,
                                 const igc::PackData *v, cudaStream_t st);
// `type` the query rows' type, `rows_most` the most rows of any sequence;
// cudaErrorNotSupported where the call's tiles are too many to count.
cudaError_t igc_pack_plan(int count, int rows, int rows_most, int positions, int kv_heads, int group, int size,
                          int type, int window, int sinks, igc::PackPlan *plan);
// igc_pack_tc.cu's part of the two calls around it.
cudaError_t igc_pack_tc_ready(igc::PackPlan *plan);
cudaError_t igc_launch_pack_tc(const igc::PackAttend *a, const igc::PackPlan *plan, const CUtensorMap *keys,
                               const CUtensorMap *values, cudaStream_t st);
cudaError_t igc_launch_pack_attend(const igc::PackAttend *a, const igc::PackPlan *plan, cudaStream_t st,
                                   int *launches);
}
