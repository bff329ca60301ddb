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
#include <cudaTypedefs.h>
#include <string.h>

#include <atomic>

#include "igc_pack.cuh"

namespace igc {

// ---------------------------------------------------------------------------
// write and read: a thread half a group (two code words), two of them a turn
// with their loads issued together, a block the rows of one side and head,
// whose places are neighbours.  Both are one pass over their rows, bound
// by HBM where instructions allow.  A code is rint(x / scale) with the quotient
// rounded as IEEE's division does, which Markstein's correction (1990) gives
// from the correctly rounded reciprocal: q = x y, then q + (x - q scale) y with
// fused multiply-adds.  A group that holds a NaN or needs the clamp divides.
// 67,000 rows of 8 x 128 in bf16: written in 142 us, read back in 77 (109 for
// both at the copy rate; a group a thread with a division a value took 400);
// 32768 rows of 256 in f16 read in 11 us.

constexpr int PK_THREADS = 256, PK_ITEMS = 2, PK_TURNS = 2, PK_COLS = 16;

struct PackIo {
  PackView c;
  PackRows r;
  PackData k, v;
  int halves, rows;              // a head's halves of groups; rows a block takes at a time
  Quotient by_halves, by_per;    // and rows a sequence
};

// The last sequence that starts at or before `row`, the same for the warp.
__device__ __forceinline__ int seq_before(const PackRows &r, int row) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int i = lane; i < r.count; i += 32) n += r.starts[i] <= row;
  return max((int)__reduce_add_sync(0xffffffffu, n) - 1, 0);
}

__device__ __forceinline__ float max_nan(float x, float y) {  // a NaN where either is one
  float z;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// The codes of 16 values, and the scale of their group (two neighbouring
// lanes hold it).
__device__ __forceinline__ uint2 encode16(const float (&x)[PK_COLS], __half *scale) {
  const uint32_t pair = 3u << (threadIdx.x & 30);
  float big = 0.0f;
#pragma unroll
  for (int i = 0; i < PK_COLS; ++i) big = max_nan(big, fabsf(x[i]));
  big = max_nan(big, __shfl_xor_sync(pair, big, 1));
  const bool odd = big != big;
  if (odd) {  // without the NaNs
    big = 0.0f;
#pragma unroll
    for (int i = 0; i < PK_COLS; ++i) big = fmaxf(big, fabsf(x[i]));
    big = fmaxf(big, __shfl_xor_sync(pair, big, 1));
  }
  const __half h = __float2half_rn(fminf(__fdiv_rn(big, 7.0f), 8188.0f));
  const float step = __half2float(h), by = __frcp_rn(step);
  *scale = h;
  uint32_t w[2] = {0, 0};
  if (!odd && big * by < 7.4f) {
#pragma unroll
    for (int i = PK_COLS - 1; i >= 0; --i) {
      const float r = x[i] * by, quotient = fmaf(fmaf(-r, step, x[i]), by, r);
      const float y = quotient + 12582920.0f;  // 1.5 2^23 + 8: rounded to a whole number, its low bits n + 8
      w[i >> 3] = w[i >> 3] * 16 + (__float_as_uint(y) & 15u);
    }
  } else {
    w[0] = w[1] = 0;
#pragma unroll 1
    for (int i = PK_COLS - 1; i >= 0; --i) {
      float v = x[0];  // x[i], with no array in memory
#pragma unroll
      for (int k = 1; k < PK_COLS; ++k) v = k == i ? x[k] : v;
      float n = step > 0.0f && v == v ? rintf(__fdiv_rn(v, step)) : 0.0f;
      n = fminf(fmaxf(n, -8.0f), 7.0f);
      const uint32_t c = (uint32_t)((int)n + 8);
      if (i >= 8) w[1] = w[1] * 16 + c;
      else w[0] = w[0] * 16 + c;
    }
  }
  return make_uint2(w[0], w[1]);
}

// Eight codes' values.
__device__ __forceinline__ void decode8(uint32_t w, float step, float (&x)[8]) {
  uint32_t v[4];
  dequant_i4(w, v);  // codes e and e + 4 together
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v[e]));
    x[e] = f.x * step;
    x[e + 4] = f.y * step;
  }
}

template <bool WRITE, int TYPE, bool WIDE>
__global__ void __launch_bounds__(PK_THREADS) pack_rows_kernel(const __grid_constant__ PackIo a) {
  const int side = blockIdx.y & 1, head = blockIdx.y >> 1;
  const int r = a.by_halves.of(threadIdx.x), w = threadIdx.x - r * a.halves;
  const PackData d = side ? a.v : a.k;
  uint2 *codes = reinterpret_cast<uint2 *>(side ? a.c.vc : a.c.kc);
  uint16_t *scales = side ? a.c.vs : a.c.ks;
  const size_t col = (size_t)head * d.head_stride + PK_COLS * w;
  int row = blockIdx.x * (a.rows * PK_ITEMS * PK_TURNS) + r;
  // every sequence that is not to be run is told, those that no row leads to among them
  if (a.r.starts && blockIdx.y == 0)
    for (int i = blockIdx.x * PK_THREADS + threadIdx.x; i < a.r.count; i += gridDim.x * PK_THREADS) seq_at(a.c, a.r, i);
  int s = a.r.starts ? seq_before(a.r, min(row - r, a.r.rows - 1)) : 0;
  if (r >= a.rows) return;  // threads past a whole number of rows
  SeqAt q = {0, 0, 0, -1};
  bool have = false;
#pragma unroll 1
  for (int turn = 0; turn < PK_TURNS; ++turn) {
    // 0 nothing to do, 1 a place of the cache, 2 zeros (padding, or outside the cache), by item
    int todo[PK_ITEMS];
    size_t at[PK_ITEMS], half_at[PK_ITEMS];
#pragma unroll
    for (int it = 0; it < PK_ITEMS; ++it, row += a.rows) {
      todo[it] = 0;
      if (row >= a.r.rows) continue;
      if (!a.r.starts) {
        const int now = a.by_per.of(row);
        if (!have || now != s) q = seq_at(a.c, a.r, s = now), have = true;
      } else {
        if (!have) q = seq_at(a.c, a.r, s), have = true;
        while (row >= a.r.starts[s + 1] && s + 1 < a.r.count) q = seq_at(a.c, a.r, ++s);
      }
      if (row < q.first || row >= q.first + q.n) continue;  // no sequence's row
      const int p = q.fill + (row - q.first);
      const bool outside = p >= a.c.positions || q.slot < 0;
      if (p >= 0 && outside) pack_trouble(a.c);
      todo[it] = p < 0 || outside ? 2 : 1;
      at[it] = (size_t)row * d.row_stride + col;
      half_at[it] = (todo[it] == 1 ? ((size_t)q.slot * a.c.heads + head) * a.c.positions + p : 0) * a.halves + w;
    }
    if (WRITE) {
      float x[PK_ITEMS][PK_COLS];
#pragma unroll
      for (int it = 0; it < PK_ITEMS; ++it) {
        if (todo[it] != 1) continue;
        load8(d.data, TYPE, at[it], WIDE, *reinterpret_cast<float(*)[8]>(&x[it][0]));
        load8(d.data, TYPE, at[it] + 8, WIDE, *reinterpret_cast<float(*)[8]>(&x[it][8]));
      }
#pragma unroll
      for (int it = 0; it < PK_ITEMS; ++it) {
        if (todo[it] != 1) continue;
        __half h;
        codes[half_at[it]] = encode16(x[it], &h);
        if ((w & 1) == 0) scales[half_at[it] >> 1] = __half_as_ushort(h);
      }
    } else {
      uint2 c[PK_ITEMS];
      float step[PK_ITEMS];
#pragma unroll
      for (int it = 0; it < PK_ITEMS; ++it) {
        c[it] = make_uint2(0x88888888u, 0x88888888u);
        step[it] = 0.0f;
        if (todo[it] == 1) {
          c[it] = codes[half_at[it]];
          step[it] = __half2float(__ushort_as_half(scales[half_at[it] >> 1]));
        }
      }
#pragma unroll
      for (int it = 0; it < PK_ITEMS; ++it) {
        if (todo[it] == 0) continue;
        float x[8];
        decode8(c[it].x, step[it], x);
        store8(d.data, TYPE, at[it], WIDE, x);
        decode8(c[it].y, step[it], x);
        store8(d.data, TYPE, at[it] + 8, WIDE, x);
      }
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
//           byte permute, used as they lie.  For 16-bit rows a weight and a
//           value are each rounded to f16 once: the value f16((n - 8) scale),
//           a whole number of 2^-24 however small the scale (2^-11 of it at
//           most), and the weight 2^15 times itself (2^-11 of it at most down
//           to 2^-29 of the row's largest, below that 2^-40 of the largest).
//           Folded into the weight instead, small scales took the product
//           below f16's range, and first positions of much weight and small
//           values took the rest of the row's result with them.
//
// A query row is scaled by the power of two that puts its largest magnitude
// in [2^13, 2^14) and kept as f16, exact for bf16 and f16 rows but for
// magnitudes 2^38 below the largest.  For f32 rows (SP) queries and weights
// are each kept as f16 hi and lo parts, a weight's lo 2^11 times itself (its
// hi 2^15 times, so that both hold to 2^-51 of the row's largest), and
// (n - 8) scale as hi and lo, which hold it exactly; the products left out
// (lo x lo) are below f32's own rounding, and each step of 16 positions starts from zero accumulators, as
// the tensor core's sums round towards zero.
//
// Bound by instruction issue: four query heads over 131071 positions of 8 x 128
// take 57 us (151 MB: 2.7 TB/s, issue 64% busy), 512 rows of 8 heads of 512
// over 8704 positions 347 us (204 TFLOP/s, 38% of the tensor pipe), 511 f32 rows
// behind a window of 512 46 us, one token at 1024 9 us.  Steps are 128 positions
// for 8 and 16 rows to 256 wide; wider tiles' registers leave room for 64.

template <int HDP, int NT, bool SP>
struct PackTile {
  static constexpr int RB = 8 * NT;
  static constexpr int C = HDP / 32;                     // groups
  static constexpr int PITCH = HDP >= 256 ? 128 : HDP / 2;  // code bytes of a swizzled row
  static constexpr int HALVES = HDP / 2 / PITCH;         // rows of 512 columns lie in two halves
  static constexpr int MP = NT <= 2 && HDP <= 256 ? 2 : 1;
  static constexpr int TP = 64 * MP;                     // positions a step
  static constexpr int OVER = 2;                         // steps a unit costs beside its own
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
  static_assert(RING >= RB * (HDP + 2) * 4, "a cluster's partial sums lie in the ring");
  static constexpr bool CLUSTERS = NT <= 2;              // may share a unit as a cluster (the wider forms have no registers for it)
  // blocks an SM that registers are kept for
  static constexpr int PER_SM = NT == 1 ? (HDP <= 128 ? 4 : 3) : NT <= 4 && HDP <= 256 ? 3 : 2;
};

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

// A cluster's partial sums, each block's in its own shared memory as pieces lie
// in global, joined; a block takes its share of the fours of columns.
template <int RB>
__device__ __forceinline__ void join_cluster(const PackAttend &a, const PackWalk &w, const float *mine, int cluster) {
  cluster_sync();
  const int size = a.c.size, fours = size / 4, all = min(RB, w.q.n * a.group - w.b * RB) * fours;
  const int rank = blockIdx.x % cluster;
  const bool wide = wide_rows(a.out);
  for (int i = rank * 128 + threadIdx.x; i < all; i += cluster * 128) {
    const int r = i / fours, col = 4 * (i - r * fours);
    float m = -INFINITY, l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < cluster; j0 += 4) {
      float pm[4], pl[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        pl[k] = 0.0f;
        pm[k] = -INFINITY;
        v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (j0 + k < cluster) {
          pm[k] = cluster_ld(mine + RB * size + r, j0 + k);
          pl[k] = cluster_ld(mine + RB * size + RB + r, j0 + k);
          v[k] = cluster_ld4(mine + r * size + col, j0 + k);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float mx = fmaxf(m, pm[k]), base = mx == -INFINITY ? 0.0f : mx;
        const float back = exp2_fast(m - base), f = exp2_fast(pm[k] - base);
        m = mx;
        l = l * back + pl[k] * f;
        x[0] = fmaf(v[k].x, f, x[0] * back);
        x[1] = fmaf(v[k].y, f, x[1] * back);
        x[2] = fmaf(v[k].z, f, x[2] * back);
        x[3] = fmaf(v[k].w, f, x[3] * back);
      }
    }
    const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
    const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    const int rr = w.b * RB + r, token = a.by_group.of(rr);
    store4(a.out.data, a.out.type,
           (size_t)(w.q.first + token) * a.out.row_stride +
               (size_t)(w.h * a.group + rr - token * a.group) * a.out.head_stride + col,
           wide, y);
  }
  cluster_sync();  // no block ends before the others have read its sums
}

template <int HDP, int NT, bool SP, bool FULL>
__global__ void __launch_bounds__(128, PackTile<HDP, NT, SP>::PER_SM)
    pack_attend_kernel(const __grid_constant__ PackAttend a, const __grid_constant__ CUtensorMap tmk,
                       const __grid_constant__ CUtensorMap tmv, int tall, int cluster) {
  using L = PackTile<HDP, NT, SP>;
  constexpr float WEIGHT = 32768.0f;  // what weights, and with them sums and results, are kept times
  constexpr float LOW = 2048.0f;      // what their low halves are kept times beside it
  constexpr int RB = L::RB, C = L::C, NS = L::NS, WC = L::WC, WP = L::WP, NB = L::NB, MP = L::MP, TP = L::TP,
                PITCH = L::PITCH;
  extern __shared__ __align__(1024) uint8_t sm_raw[];
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
  int share = 0;
  bool any;
  if (!L::CLUSTERS) cluster = 0;
  if (cluster > 0) {  // a unit a cluster: the blocks take runs of its tiles
    const int unit = blockIdx.x / cluster, rank = blockIdx.x - unit * cluster;
    const int block = unit / a.c.heads;
    w.h = unit - block * a.c.heads;
    w.s = block / tall;
    w.b = block - w.s * tall;
    w.q = seq_at(a.c, a.r, w.s);
    any = w.b < blocks_of(a, w.q, RB);
    if (any) w.sp = block_span(a, w.q, w.b, RB, TP);
    else w.sp = {0, 0, 0, 0, 0};
    w.ka = w.sp.count() * rank / cluster;
    w.kb = w.sp.count() * (rank + 1) / cluster;
    w.whole = cluster == 1;
  } else {
    any = walk_start<RB, TP, L::OVER>(a, tall, w, &share);
  }
  pdl_release();
  if (cluster == 0 && tid == 0) leave_cut(a, w, any);
  if (!any) return;
  int step0 = 0;  // steps this block has taken: the ring's place
  bool gave_up = false;
  for (;;) {  // one unit, or a piece of it, a turn
    const SeqAt q = w.q;
    const TileSpan sp = w.sp;
    const int b = w.b, h = w.h, ka = w.ka, kb = w.kb;
    const bool whole = w.whole;
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
      __syncwarp();  // lanes may leave the polls apart, and the products take the warp as one
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
            sc[mp][nt][e] = exp2_fast(sc[mp][nt][e] - base[e & 1]) * WEIGHT;
            sum[e & 1] += sc[mp][nt][e];
          }
          // the weights turned to the second product's fragment: positions along its depth
          const uint32_t h0 = half2_bits(sc[mp][nt][0], sc[mp][nt][1]), h1 = half2_bits(sc[mp][nt][2], sc[mp][nt][3]);
          uint2 *p = reinterpret_cast<uint2 *>(sm + L::OFF_P) + ((warp * MP + mp) * NT + nt) * 32 + lane;
          *p = make_uint2(transpose8(h0), transpose8(h1));
          if (SP) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
            const uint32_t l0 = half2_bits((sc[mp][nt][0] - f0.x) * LOW, (sc[mp][nt][1] - f0.y) * LOW);
            const uint32_t l1 = half2_bits((sc[mp][nt][2] - f1.x) * LOW, (sc[mp][nt][3] - f1.y) * LOW);
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
            // f32 rows: scales all below 2^-7 (0x2000) go in 2^13 times, as the tensor core aligns
            // products by their exponent fields and would cut those of subnormal values short
            float back = 1.0f;
            if (SP && __all_sync(0xffffffffu, ((step[0] | step[1]) & 0xe000e000u) == 0)) {
              step[0] = mul2(step[0], 0x70007000u);
              step[1] = mul2(step[1], 0x70007000u);
              back = 1.0f / 8192.0f;
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
                    const uint32_t c = v[2 * u + e], hi = mul2(c, step[i]);
                    av[u][2 * i + e] = hi;
                    if (SP) al[u][2 * i + e] = rest2(c, step[i], hi);
                  }
              }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (SP) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  mma_add(acc, av[u], pb[L::PARTS - 1][nt].x, pb[L::PARTS - 1][nt].y);
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[e] *= 1.0f / LOW;
                  mma_add(acc, al[u], pb[0][nt].x, pb[0][nt].y);
                  mma_add(acc, av[u], pb[0][nt].x, pb[0][nt].y);
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    o[nt][nb * 4 + gi * 2 + u][e] = fmaf(acc[e], back, o[nt][nb * 4 + gi * 2 + u][e]);
                }
              } else {
#pragma unroll
                for (int u = 0; u < 2; ++u) mma_add(o[nt][nb * 4 + gi * 2 + u], av[u], pb[0][nt].x, pb[0][nt].y);
              }
            }
          }
        }
      }
    }
    step0 += kb - ka;

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
      float *pw = cluster > 0 ? reinterpret_cast<float *>(sm)
                              : piece_at(a, gridDim.x, RB, 2 * (size_t)blockIdx.x + (ka == 0 ? 1 : 0));
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

    if (cluster > 0) {
      if (cluster > 1) join_cluster<RB>(a, w, reinterpret_cast<const float *>(sm), cluster);
      break;
    }
    if (!walk_next<RB, TP, L::OVER>(a, w, share)) break;
  }
  if (gave_up) pack_trouble(a.c);
}

// ---------------------------------------------------------------------------
// units cut between blocks, joined: block x takes the unit that attention
// block x + 1 begins inside, if that is the unit's first cut.  `some` rows a
// block: one by all its threads (a thread four columns of every second, fourth
// or eighth piece of a narrow head) where there may be many pieces, else each
// by as many threads as it has fours of columns.  The order of the additions
// is fixed.  (64 sequences of 32 rows cut over 148 blocks: 66 us with the
// attention; 79 with one row a block and its pieces read one after another.)

struct PackMerge {
  PackAttend a;
  int rb, grid, some;
};

constexpr int PM_THREADS = 128, PM_CHUNK = 128;  // pieces whose factors are kept at a time

__global__ void __launch_bounds__(PM_THREADS) pack_merge_kernel(const __grid_constant__ PackMerge g) {
  __shared__ float pm[PM_CHUNK], pl[PM_CHUNK];
  __shared__ float4 part4[PM_THREADS];
  const PackAttend &a = g.a;
  const int RB = g.rb, size = a.c.size, tid = threadIdx.x;
  const int lanes = size / 4, teams = PM_THREADS / lanes, team = tid / lanes, col = 4 * (tid - team * lanes);
  const bool wide = wide_rows(a.out);
  pdl_wait();
  const PackCut c = reinterpret_cast<const PackCut *>(a.work)[blockIdx.x + 1];
  if (c.first != (int)blockIdx.x) return;
  const int pieces = c.last - c.first + 1;
  auto at = [&](int i) { return piece_at(a, g.grid, RB, 2 * (size_t)(c.first + i) + (i == 0 ? 1 : 0)); };
  auto put = [&](int rr, float4 x, float l) {
    const int token = a.by_group.of(rr);
    const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
    const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    store4(a.out.data, a.out.type,
           (size_t)(c.q_first + token) * a.out.row_stride +
               (size_t)(c.h * a.group + rr - token * a.group) * a.out.head_stride + col,
           wide, y);
  };
  auto add = [](float4 &x, const float4 &y, float f) {
    x.x = fmaf(y.x, f, x.x);
    x.y = fmaf(y.y, f, x.y);
    x.z = fmaf(y.z, f, x.z);
    x.w = fmaf(y.w, f, x.w);
  };
  if (g.some > 1) {
    const int r = blockIdx.y * g.some + team, rr = c.b * RB + r;
    if (team >= g.some || rr >= c.q_n * a.group) return;
    float m = -INFINITY, l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i0 = 0; i0 < pieces; i0 += 4) {
      float ym[4], y[4];
      float4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = 0.0f;
        if (i0 + i < pieces) {
          const float *p = at(i0 + i);
          y[i] = p[(size_t)RB * size + RB + r];
          ym[i] = p[(size_t)RB * size + r];
          v[i] = *reinterpret_cast<const float4 *>(p + (size_t)r * size + col);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (y[i] == 0.0f) continue;  // it saw none of the row's positions
        const float mx = fmaxf(m, ym[i]), base = mx == -INFINITY ? 0.0f : mx;
        const float back = exp2_fast(m - base), f = exp2_fast(ym[i] - base);
        m = mx;
        l = l * back + y[i] * f;
        x.x *= back, x.y *= back, x.z *= back, x.w *= back;
        add(x, v[i], f);
      }
    }
    put(rr, x, l);
    return;
  }
  const int r = blockIdx.y, rr = c.b * RB + r;
  if (rr >= c.q_n * a.group) return;
  float m = -INFINITY, l = 0.0f;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int c0 = 0; c0 < pieces; c0 += PM_CHUNK) {
    const int cn = min(PM_CHUNK, pieces - c0);
    __syncthreads();
    if (tid < cn) {
      const float *p = at(c0 + tid) + (size_t)RB * size + r;
      const float y = p[RB], ym = p[0];
      pl[tid] = y;
      pm[tid] = y == 0.0f ? -INFINITY : ym;
    }
    __syncthreads();
    float mx = m;
    for (int i = 0; i < cn; ++i) mx = fmaxf(mx, pm[i]);
    const float base = mx == -INFINITY ? 0.0f : mx, back = exp2_fast(m - base);
    m = mx;
    l *= back;
    x.x *= back, x.y *= back, x.z *= back, x.w *= back;
    for (int i = 0; i < cn; ++i)
      if (pl[i] != 0.0f) l += pl[i] * exp2_fast(pm[i] - base);
    if (team < teams) {
#pragma unroll 4
      for (int i = team; i < cn; i += teams) {
        const float4 v = *reinterpret_cast<const float4 *>(at(c0 + i) + (size_t)r * size + col);
        if (pl[i] != 0.0f) add(x, v, exp2_fast(pm[i] - base));
      }
    }
  }
  part4[tid] = x;
  __syncthreads();
  if (team != 0) return;
  for (int i = 1; i < teams; ++i) {
    const float4 y = part4[i * lanes + tid];
    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
  }
  put(rr, x, l);
}

// What a kernel form needs on the current device, looked up once a device:
// its shared memory allowed and how many blocks an SM holds.
template <int HDP, int NT, bool SP, bool FULL>
cudaError_t pack_form_ready(PackPlan *plan, int *per_sm) {
  using L = PackTile<HDP, NT, SP>;
  plan->tile = L::TP;
  plan->over = L::OVER;
  plan->pitch = L::PITCH;
  static std::atomic<int> known[PACK_DEVICES];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < PACK_DEVICES && (*per_sm = known[dev].load()) > 0) return cudaSuccess;
  auto kern = pack_attend_kernel<HDP, NT, SP, FULL>;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(per_sm, kern, 128, L::SMEM);
  if (e == cudaSuccess && *per_sm < 1) e = cudaErrorInvalidConfiguration;
  if (e == cudaSuccess && dev < PACK_DEVICES) known[dev].store(*per_sm);
  return e;
}

template <int HDP, int NT, bool SP, bool FULL>
cudaError_t pack_form_launch(const PackAttend &a, const PackPlan &p, const CUtensorMap &tmk, const CUtensorMap &tmv,
                             cudaStream_t st) {
  return pack_launch(pack_attend_kernel<HDP, NT, SP, FULL>, dim3(p.grid), 128, PackTile<HDP, NT, SP>::SMEM, st, false, p.cluster,
                     a, tmk, tmv, p.tall, p.cluster);
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

static cudaError_t pack_form(PackPlan *p, int *per_sm) {
  if (p->tc) {
    *per_sm = 1;
    return igc_pack_tc_ready(p);
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

template <bool WRITE>
static cudaError_t launch_rows(const PackView *c, const PackRows *r, const PackData *k, const PackData *v,
                               cudaStream_t st) {
  if (k->type != v->type) return cudaErrorInvalidValue;
  const int halves = c->size / PK_COLS;
  const int rows = PK_THREADS / halves;
  const PackIo io = {*c, *r, *k, *v, halves, rows, Quotient::by(halves), Quotient::by(r->per > 0 ? r->per : 1)};
  const int block_rows = rows * PK_ITEMS * PK_TURNS;
  const dim3 grid((unsigned)((r->rows + block_rows - 1) / block_rows), 2 * c->heads);
  if (c->heads > 32767) return cudaErrorInvalidValue;
  // 16 bytes at a time where every eight columns of both sides start on them
  auto lies = [](const PackData &d) {
    const long per = d.type == 1 ? 4 : 8;
    return ((size_t)d.data & 15) == 0 && d.row_stride % per == 0 && d.head_stride % per == 0;
  };
  const bool wide = lies(*k) && lies(*v);
  auto run = [&](auto kern) { return pack_launch(kern, grid, PK_THREADS, 0, st, false, 0, io); };
  switch (k->type * 2 + (wide ? 1 : 0)) {
    case 2: return run(pack_rows_kernel<WRITE, 1, false>);
    case 3: return run(pack_rows_kernel<WRITE, 1, true>);
    case 4: return run(pack_rows_kernel<WRITE, 2, false>);
    case 5: return run(pack_rows_kernel<WRITE, 2, true>);
    case 6: return run(pack_rows_kernel<WRITE, 3, false>);
    default: return run(pack_rows_kernel<WRITE, 3, true>);
  }
}

cudaError_t igc_launch_pack_write(const PackView *c, const PackRows *r, const PackData *k, const PackData *v,
                                  cudaStream_t st) {
  return launch_rows<true>(c, r, k, v, st);
}

cudaError_t igc_launch_pack_read(const PackView *c, const PackRows *r, const PackData *k, const PackData *v,
                                 cudaStream_t st) {
  return launch_rows<false>(c, r, k, v, st);
}

// The most tiles a unit of blocks of `rb` rows has: the rows' reach, wherever it
// starts in a tile.
static long most_tiles(const PackPlan *p, int rb, int positions, int group, int window, int sinks) {
  const long reach = window > 0 ? (long)window + rb / group + 1 + sinks + 3 * p->tile : positions;
  return ((reach < positions ? reach : positions) + p->tile - 1) / p->tile;
}

cudaError_t igc_pack_plan(int count, int rows, int rows_most, int positions, int kv_heads, int group, int size,
                          int type, int window, int sinks, PackPlan *p) {
  memset(p, 0, sizeof(*p));
  p->wide = size <= 64 ? 64 : size <= 128 ? 128 : size <= 256 ? 256 : 512;
  p->split2 = type == 1 ? 1 : 0;
  p->full = size == p->wide;
  const long need = (long)rows_most * group;
  int sms = 0, per_sm = 0;
  cudaError_t e = pack_sms(&sms);
  // Few units of few tiles: a cluster of blocks a unit, joined there, one
  // launch and no scratch (one token at 1024 positions 11.6 -> 9.1 us, 64 tokens
  // behind a window of 512 17 -> 12.4; 4 lanes of 8 heads of 256 at 1024, in 32
  // bits 20.6 -> 8.9, in 16, against the tcgen05 form, 17.8 -> 8.7).  That holds to
  // eight tiles a block (100 tokens at 1000: 21.8 us, the list 27.9; 4 lanes at
  // 16000 28 and 41), but to four where the largest clusters of single blocks of
  // rows leave most of the device idle (one token at 8100: 17 us and 20, at 16000
  // 28 and 23).  Sixteen rows a block where eight would not do, of full heads only.
  for (int rows8 = 1; rows8 <= (p->full && need > 8 ? 2 : 1) && e == cudaSuccess; ++rows8) {
    p->rows8 = rows8;
    e = pack_form(p, &per_sm);
    const long blocks = (need + 8 * rows8 - 1) / (8 * rows8), units = (long)count * kv_heads * blocks;
    const long wave = (long)sms * per_sm, tiles = most_tiles(p, 8 * rows8, positions, group, window, sinks);
    int cluster = 1;
    while (cluster < 16 && cluster < tiles) cluster *= 2;
    while (cluster > 1 && units * cluster > wave) cluster /= 2;
    if (e == cudaSuccess && units * cluster <= wave && tiles <= (cluster == 16 && blocks == 1 ? 4 : 8) * cluster) {
      p->cluster = cluster;
      p->tall = (int)blocks;
      p->grid = (int)units * cluster;
      return cudaSuccess;
    }
  }
  if (e != cudaSuccess) return e;
  int most8 = p->split2 ? 4 : 2;  // what registers hold, and past 16 rows the tcgen05 form takes over
  if (p->wide == 512) most8 = p->split2 ? 2 : 4;
  p->rows8 = need <= 8 ? 1 : need <= 16 && p->full ? 2 : most8;  // fewer forms where a group's tile is part empty
  if (!p->split2 && p->wide <= 256 && need > 16) {
    p->tc = 1;
    p->rows8 = 16;
  }
  const int rb = 8 * p->rows8;
  e = pack_form(p, &per_sm);
  if (e != cudaSuccess) return e;
  const long blocks = (need + rb - 1) / rb, tiles = most_tiles(p, rb, positions, group, window, sinks);
  // no more units than whole blocks and a part of one for each sequence that has rows
  const double list = ((double)rows * group / rb + (count < rows ? count : rows)) * kv_heads * (tiles + p->over);
  if (list >= 2147418112.0) return cudaErrorNotSupported;  // 31 bits, with room for a share's rounding
  p->list_most = (int)list + 1;
  // blocks of at least 7 steps, were all units as long as the cache's room lets them
  // be (their depths are on the device; in a roomier cache the runs are shorter):
  // shorter runs leave more pieces to join than they save (one token at 32000 in a
  // cache of that room: 49 us by single steps, 29 by 4, 28 by 7; 100000: 60, 60, 53)
  p->grid = sms * per_sm;
  if (list / 7 < p->grid) p->grid = list < 7 ? 1 : (int)(list / 7);
  p->tall = blocks > 8;
  p->work_floats = p->grid > 1 ? (size_t)p->grid * (8 + 2 * (size_t)rb * (size + 2)) : 8;
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
  CUtensorMap tmk, tmv;
  cudaError_t e = pack_map(a->c, a->c.kc, p->pitch, &tmk);
  if (e == cudaSuccess) e = pack_map(a->c, a->c.vc, p->pitch, &tmv);
  if (e != cudaSuccess) return e;
  *launches = 1;
  e = p->tc ? igc_launch_pack_tc(a, p, &tmk, &tmv, st) : pack_run(*p, *a, tmk, tmv, st);
  if (e != cudaSuccess || p->grid == 1 || p->cluster > 0) return e;
  *launches = 2;
  const int rb = 8 * p->rows8, some = p->tc && PM_THREADS / (a->c.size / 4) >= 2 ? 2 : 1;
  const PackMerge g = {*a, rb, p->grid, some};
  return pack_launch(pack_merge_kernel, dim3((unsigned)p->grid - 1, rb / some), PM_THREADS, 0, st, true, 0, g);
}
