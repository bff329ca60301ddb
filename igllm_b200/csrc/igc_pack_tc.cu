// igc_pack_tc.cu - attention over the packed cache's codes on tcgen05, for many
// 16-bit query rows.
//
// A block holds 128 query rows of one (sequence, key/value head): their
// queries in shared memory (f16, an operand), and in tensor memory their
// results and four tiles of scores, whose places the weights take.  Its steps
// are tiles of 64 positions:
//
//   warp 17          walks the block's units, tells the others, and has their
//                    codes and scales brought into shared memory by TMA.
//   warps 8-11, 12-15 turn a tile's key (value) codes into f16((n - 8) scale)
//                    in two operand buffers a side; rows of 64 columns
//                    (128 bytes, swizzled), one layout for both: the key
//                    operand's rows are its 8 KB blocks' rows, the value
//                    operand is read across them, so nothing is transposed.
//   warp 16          one thread issues scores three tiles ahead and the values
//                    as weights come.
//   warps 0-3, 4-7   the even and the odd tiles, a thread a row: the 64 scores'
//                    maximum, the weights back into tensor memory, the row's
//                    sum.  The maximum in use is handed from tile to tile; it
//                    and the results change only when a tile's maximum is more
//                    than 2^8 over it.  Weights are kept 2^7 times, which then
//                    still fits f16.  (Following by 2^4, 2^2 or at once, with
//                    weights 2^11 to 2^15 times, takes prompts 128 us to 135,
//                    171, 180 and the windowed prompt 102 to 125.)
//
// Columns of a group of eight keep the order their nibbles come out in,
// 0 4 1 5 2 6 3 7, in the queries and, undone at the end, in the results.
// A bf16 query row is scaled by an exact power of two into f16's range; keys,
// values and weights are each rounded to f16 once: 2^-11 of a key or value at
// most, which are whole numbers of 2^-24 whatever their scale, and 2^-11 of a
// weight down to 2^-21 of the row's largest, below that 2^-32 of the largest.
//
// Bound by the products: a step of a 256-wide head is 16 score products of 53
// cycles (64 positions wide: 61% of the pipe's rate) and 4 value products of 129
// (all of it), 1360 cycles; warp 16 is busy 1400 to 1540 a step.  Wider score
// products would need 128 rows of key operands twice, which the queries leave no
// room for.  3 prompts to 4096 of 8 x 256: 124 us, 630 TFLOP/s; 8192 rows behind
// a window of 512: 101 us; 64 x 4 rows at 8192: 66 us.  The mma.sync form took
// 506, 355 and 104.  A unit's ends (queries in, results out) cost about 8 steps,
// which OVER tells the sharing (4, 7 and 10 measured: 64 x 4 in 86, 81 and 83 us,
// prompts in 164, 127 and 131, before the joining was sped up).
#include <atomic>

#include "igc_pack.cuh"

namespace igc {

template <int HDP>
struct PackTc {
  static constexpr int RB = 128, TP = 64, C = HDP / 32;
  static constexpr int OVER = 8;                        // steps a unit costs beside its own
  static constexpr int LAG = 8;                         // powers of two a maximum in use may be passed by
  static constexpr int KEEP = 15 - LAG;                 // power of two that weights, sums and results are kept times
  static constexpr int BLOCKS = HDP / 64;               // 64-column blocks of an operand
  static constexpr int SIDE = BLOCKS * 64 * 128;        // one key or value operand buffer
  static constexpr int T_S = HDP;                       // tensor-memory columns: results, then four tiles of scores
  static constexpr int SB = 4;
  static constexpr int PITCH = HDP / 2 < 128 ? HDP / 2 : 128;  // code bytes of a row
  static constexpr int NS = HDP == 256 ? 3 : 6;         // codes in flight: a side of a tile a place
  // Barriers that codes are there, one a side even where the sides take a
  // place in turns: a warp that waits for a phase has to have seen the phase
  // before it complete, which it knows of its own side's only.
  static constexpr int NF = NS % 2 ? 2 * NS : NS;
  static constexpr int CODE = 64 * PITCH + 64 * C * 2;  // codes, then scales
  static constexpr int OFF_Q = 4 * SIDE;                // the queries, 16 KB a 64-column block
  static constexpr int OFF_CODE = OFF_Q + BLOCKS * RB * 128;
  static constexpr int ALL = OFF_CODE + NS * CODE;
  static constexpr int SMEM = 1024 + (ALL > 116 * 1024 ? ALL : 116 * 1024);  // one block an SM
  static constexpr int LW = C < 4 ? C : 4;              // groups across a warp's lanes
  static constexpr int ROWS = 32 / LW;                  // positions across them
  static constexpr int ITEMS = 64 * C / 128;            // groups a thread turns a tile
  static_assert(CODE % 1024 == 0 || PITCH < 128, "swizzled boxes start on their pattern");
};

constexpr int TC_THREADS = 576;

__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
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
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 16 bytes (or, of none, zeros) into shared memory, not waited for.
__device__ __forceinline__ void pk_copy16(void *dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}

// Pairs of floats at once.
__device__ __forceinline__ uint64_t pair2(float x, float y) {
  return (uint64_t)__float_as_uint(x) | ((uint64_t)__float_as_uint(y) << 32);
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mulf2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float first2(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float second2(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// Operand descriptors, 128-byte swizzle, 8-row groups 1 KB apart: the key
// operand along its rows (K-major), and the value operand across them
// (MN-major: 64-column blocks 8 KB apart).
__device__ __forceinline__ uint64_t tc_desc(uint32_t at, uint32_t lead) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// The scores of the tile in key buffer KB into place SB of tensor memory, and
// the values of the weights there added; every operand is a constant but for
// the shared memory's base.
template <int HDP>
__device__ __forceinline__ void tc_scores(const uint8_t *sm, int kb, int sb, uint64_t *ready, uint64_t *free) {
  using L = PackTc<HDP>;
  constexpr uint32_t id = (1u << 4) | ((uint32_t)(L::TP >> 3) << 17) | ((uint32_t)(L::RB >> 4) << 24);
  const uint64_t q0 = tc_desc(smem_u32(sm) + L::OFF_Q, 16), k0 = tc_desc(smem_u32(sm) + kb * L::SIDE, 16);
  const uint32_t d = L::T_S + sb * 64;
#pragma unroll
  for (int i = 0; i < HDP / 16; ++i)
    tc_mma_ss(d, q0 + (uint64_t)(((i / 4) * 16384 + (i & 3) * 32) >> 4), k0 + (uint64_t)(((i / 4) * 8192 + (i & 3) * 32) >> 4),
              id, i > 0);
  tc_commit(ready);
  tc_commit(free);
}
template <int HDP>
__device__ __forceinline__ void tc_values(const uint8_t *sm, int vb, int sb, bool add, uint64_t *free, uint64_t *done) {
  using L = PackTc<HDP>;
  constexpr uint32_t id = (1u << 4) | (1u << 16) | ((uint32_t)(HDP >> 3) << 17) | ((uint32_t)(L::RB >> 4) << 24);
  const uint64_t v0 = tc_desc(smem_u32(sm) + (2 + vb) * L::SIDE, 8192);
  const uint32_t p = L::T_S + sb * 64;
#pragma unroll
  for (int i = 0; i < L::TP / 16; ++i)
    tc_mma_ts(0, p + i * 8, v0 + (uint64_t)(i * 2048 >> 4), id, i > 0 ? 1u : add ? 1u : 0u);
  tc_commit(free);
  tc_commit(done);
}

// A unit as the walking warp tells it to the others; steps < 0 at the end.
struct TcUnit {
  int steps, whole;
  int head, from;         // step t's tile: k = ka + t below head, else from + k - head
  int ka, hi, lo;
  int q_first, live_rows;  // the sequence's first row; how many of the block's rows are its
  int rr0, h;             // the block's first (row, head of the group), and the key/value head
  int fill, past, lost;   // past: some row stands beyond the cache; lost: no such slot
  int base;               // the first position of the slot's head among all
  float *piece;           // where partial sums go
};

template <int HDP>
__global__ void __launch_bounds__(TC_THREADS, 1)
    pack_attend_tc_kernel(const __grid_constant__ PackAttend a, const __grid_constant__ CUtensorMap tmk,
                          const __grid_constant__ CUtensorMap tmv, int tall) {
  using L = PackTc<HDP>;
  constexpr int RB = L::RB, TP = L::TP, C = L::C;
  extern __shared__ __align__(1024) uint8_t tc_raw[];
  __shared__ uint64_t bars[30 + L::NF + L::NS];
  __shared__ uint32_t tmem_slot;
  __shared__ float shared_m[2][RB], half_big[2][RB], half_sum[2][RB];
  __shared__ TcUnit units[2];
  uint8_t *sm = tc_raw + ((1024 - (smem_u32(tc_raw) & 1023)) & 1023);
  // [side][buffer] filled by the code warps, and free again; [score place]
  // scores ready, weights ready, values added; maxima told; queries ready; a
  // unit told, and done with; the last product over; the softmax warps' halves
  // of a row told (maxima, sums); codes there; [place] free again
  uint64_t *full = bars, *empty = bars + 4, *sfull = bars + 8, *pfull = bars + 12, *vdone = bars + 16, *mtold = bars + 20,
           *qfull = bars + 22, *told = bars + 23, *done = bars + 25, *over = bars + 27, *both = bars + 28, *cfull = bars + 30,
           *cfree = cfull + L::NF;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&full[i], 128), mbar_init(&empty[i], 1);
    for (int i = 0; i < L::SB; ++i) mbar_init(&sfull[i], 1), mbar_init(&pfull[i], 128), mbar_init(&vdone[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&mtold[i], 128), mbar_init(&told[i], 1), mbar_init(&done[i], 17);
    mbar_init(qfull, 256);
    mbar_init(over, 1);
    mbar_init(&both[0], 256), mbar_init(&both[1], 256);
    for (int i = 0; i < L::NF; ++i) mbar_init(&cfull[i], 1);
    for (int i = 0; i < L::NS; ++i) mbar_init(&cfree[i], 4);
    mbar_init_fence();
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    tc_before();
  }
  __syncthreads();
  tc_after();
  pdl_release();
  bool failed = tmem_slot != 0;  // all 512 columns begin at 0, which keeps the products' operands constants
  int step0 = 0;                 // steps before this unit
  auto wait = [&](uint64_t *bar, int phase) {
    if (!mbar_wait(bar, (uint32_t)(phase & 1), failed ? PACK_TRIES / 64 : PACK_TRIES)) failed = true;
    // the warp as one: lanes may leave the polls apart
    failed = __any_sync(0xffffffffu, failed);
  };
  auto tile_of = [](const TcUnit &u, int t) {
    const int k = u.ka + t;
    return k < u.head ? k : u.from + (k - u.head);
  };

  if (warp == 17) {
    // ---- the units, and their codes into shared memory
    const int chd = a.c.size / 32;
    const bool one = elect_one();
    const uint64_t policy = tall ? l2_evict_last() : l2_evict_first();  // other blocks of a prompt read them too
    PackWalk w;
    int share, issued = 0;  // copies of a side of a tile
    bool any = walk_start<RB, TP, L::OVER>(a, tall, w, &share);
    if (one) leave_cut(a, w, any);
    for (int u = 0;; ++u) {
      if (u >= 2) wait(&done[u & 1], (u >> 1) - 1);
      const int steps = any ? w.kb - w.ka : -1;
      const int base = any ? (max(w.q.slot, 0) * a.c.heads + w.h) * a.c.positions : 0;
      if (one) {
        TcUnit &n = units[u & 1];
        n.steps = failed ? -1 : steps;
        if (any) {
          n.whole = w.whole;
          n.head = w.sp.head;
          n.from = w.sp.from;
          n.ka = w.ka;
          n.hi = w.sp.hi;
          n.lo = w.sp.lo;
          n.q_first = w.q.first;
          n.rr0 = w.b * RB;
          n.live_rows = min(RB, w.q.n * a.group - n.rr0);
          n.h = w.h;
          n.fill = w.q.fill;
          n.past = w.q.fill + min(w.q.n - 1, a.by_group.of(n.rr0 + RB - 1)) >= a.c.positions;
          n.lost = w.q.slot < 0;
          n.base = base;
          n.piece = piece_at(a, gridDim.x, RB, 2 * (size_t)blockIdx.x + (w.ka == 0 ? 1 : 0));
          if (n.past || n.lost) pack_trouble(a.c);
        }
        mbar_arrive(&told[u & 1]);
      }
      __syncwarp();
      if (steps < 0 || failed) break;
      for (int t = 0; t < steps && !failed; ++t) {
        const int p0 = base + w.sp.tile(w.ka + t) * TP;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const int I = 2 * (step0 + t) + side, at = I % L::NS;
          if (I >= L::NS) wait(&cfree[at], I / L::NS - 1);
          if (failed) break;  // the place may be in use
          issued = I + 1;
          if (one) {
            uint8_t *dst = sm + L::OFF_CODE + at * L::CODE;
            uint64_t *there = &cfull[I % L::NF];
            mbar_expect(there, (uint32_t)(64 * L::PITCH + 64 * chd * 2));
            pk_load(dst, side ? &tmv : &tmk, 0, p0, there);
            bulk_load(dst + 64 * L::PITCH, (side ? a.c.vs : a.c.ks) + (size_t)p0 * chd, (uint32_t)(64 * chd * 2),
                      there, policy);
          }
          __syncwarp();
        }
      }
      step0 += steps;
      any = walk_next<RB, TP, L::OVER>(a, w, share);
    }
    // no copy is under way when the block ends, whatever ended it
    for (int I = max(0, issued - L::NS); I < issued; ++I) wait(&cfull[I % L::NF], I / L::NF);
  } else {
    int spent = 0;  // units that had steps
    for (int un = 0;; ++un) {
      wait(&told[un & 1], un >> 1);
      const TcUnit &u = units[un & 1];
      const int steps = failed ? -1 : u.steps;
      if (steps < 0) break;
      if (warp == 16) {
        // ---- the products
        if (steps > 0) {
          const bool one = elect_one();
          auto scores = [&](int t) {
            if (t >= steps) return;
            const int T = step0 + t, sb = T % L::SB;
            wait(&full[T & 1], T >> 1);
            tc_after();
            if (one) tc_scores<HDP>(sm, T & 1, sb, &sfull[sb], &empty[T & 1]);
            __syncwarp();
          };
          wait(qfull, spent);
          // three tiles of scores ahead of the values: a place's scores come
          // after the values of the weights it held, in the order issued
          for (int t = 0; t < L::SB - 1; ++t) scores(t);
          for (int t = 0; t < steps; ++t) {
            const int T = step0 + t, sb = T % L::SB;
            wait(&full[2 + (T & 1)], T >> 1);
            wait(&pfull[sb], T / L::SB);
            tc_after();
            if (one) tc_values<HDP>(sm, T & 1, sb, t > 0, &empty[2 + (T & 1)], &vdone[sb]);
            __syncwarp();
            scores(t + L::SB - 1);
          }
        }
      } else if (warp >= 8) {
        // ---- codes to operands
        const int side = warp >= 12 ? 1 : 0, w4 = warp & 3, chd = a.c.size / 32;
        const int row_l = lane % L::ROWS, gr_l = lane / L::ROWS;
        const uint8_t *ring = sm + L::OFF_CODE;
        // item i: a position row and a group; eight neighbouring lanes hold
        // eight neighbouring rows, so that their accesses spread over the
        // banks.  Items are plain offsets apart: ACROSS groups to a row, then
        // rows; the swizzles are resolved here once.
        constexpr int ACROSS = C / L::LW, DOWN = 4 * L::ROWS;
        const int r0 = w4 * L::ROWS + row_l;
        const uint32_t src0 = pk_swz<L::PITCH>(r0, gr_l), sc0 = (uint32_t)(64 * L::PITCH + (r0 * chd + gr_l) * 2);
        const uint32_t dst0 = (uint32_t)((gr_l >> 1) * 8192 + r0 * 128 + ((((gr_l & 1) * 4) ^ (r0 & 7)) << 4));
        const int hi = u.hi, lo = u.lo;
        for (int t = 0; t < steps; ++t) {
          const int T = step0 + t, buf = T & 1, I = 2 * T + side, at = I % L::NS;
          wait(&cfull[I % L::NF], I / L::NF);
          const uint8_t *src = ring + at * L::CODE;
          uint4 code[L::ITEMS];
          uint32_t by[L::ITEMS];
#pragma unroll
          for (int i = 0; i < L::ITEMS; ++i) {
            const int down = i / ACROSS, over = i % ACROSS;  // over: 4 groups on, which an exclusive or does
            code[i] = *reinterpret_cast<const uint4 *>(src + down * (DOWN * L::PITCH) + (src0 ^ (over * 64)));
            by[i] = gr_l + L::LW * over < chd
                        ? *reinterpret_cast<const uint16_t *>(src + sc0 + down * (DOWN * 2 * chd) + over * 2 * L::LW)
                        : 0u;
          }
          const int p0 = tile_of(u, t) * TP;
          if (p0 + TP > hi || (p0 < lo && p0 + TP > a.sinks)) {
            // a position no row sees counts as 0 whatever lies there
#pragma unroll
            for (int i = 0; i < L::ITEMS; ++i) {
              const int p = p0 + r0 + (i / ACROSS) * DOWN;
              if (!(p < hi && (p >= lo || p < a.sinks))) by[i] = 0;
            }
          }
#pragma unroll
          for (int i = 0; i < L::ITEMS; ++i) by[i] = __byte_perm(by[i], 0, 0x1010);
          __syncwarp();
          if (lane == 0) mbar_arrive(&cfree[at]);
          if (T >= 2) wait(&empty[side * 2 + buf], (T >> 1) - 1);
          uint8_t *dst = sm + (side * 2 + buf) * L::SIDE;
#pragma unroll
          for (int i = 0; i < L::ITEMS; ++i) {
            const uint32_t words[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t v[4];
              dequant_i4(words[k], v);
              *reinterpret_cast<uint4 *>(dst + (dst0 ^ (k << 4)) + (i / ACROSS) * (DOWN * 128) + (i % ACROSS) * 16384) =
                  make_uint4(mul2(v[0], by[i]), mul2(v[1], by[i]), mul2(v[2], by[i]), mul2(v[3], by[i]));
            }
          }
          fence_async_smem();  // written here, read by the tensor core (async proxy)
          mbar_arrive(&full[side * 2 + buf]);
        }
      } else {
        // ---- the softmax: warps 0-3 the even tiles, 4-7 the odd, a thread a row
        const int r = tid & 127, half = tid >> 7;  // half: also of the head's columns, in and out
        const int size = a.c.size, group = a.group;
        const bool live = r < u.live_rows, idle = (r & 96) >= u.live_rows;  // idle: no row of the warp is one
        const uint32_t lanes = (uint32_t)(r & 96) << 16;
        const int rr = u.rr0 + r, token = a.by_group.of(rr), hq = u.h * group + rr - token * group;
        // the queries' place also holds the results on their way out.  The
        // 16-byte piece j (of eight columns) of this half of row x:
        auto piece_of = [&](int x, int j) {
          const int k = half * (HDP / 16) + j;
          return reinterpret_cast<uint4 *>(sm + L::OFF_Q + (k >> 3) * 16384 + x * 128 + (((k & 7) ^ (x & 7)) << 4));
        };
        // memory is read and written a row's half by HDP / 16 neighbouring
        // lanes, the rows of the warp in turns
        constexpr int PIECES = HDP / 16, AT_ONCE = 32 / PIECES;
        auto row_at = [&](long at, int i) { return __shfl_sync(0xffffffffu, at, i * AT_ONCE + lane / PIECES); };
        const int my_piece = lane % PIECES, my_col = half * (HDP / 2) + 8 * my_piece;
        auto meet = [&](int i) {
          mbar_arrive(&both[i]);
          wait(&both[i], un);
        };
        float f = 0.0f;
        if (steps > 0) {
          const bool wide = wide_rows(a.q), bf = a.q.type == 3;
          auto value = [&](uint32_t x, int e) {
            if (bf) return __uint_as_float(e ? x & 0xffff0000u : x << 16);
            return __half2float(__ushort_as_half((uint16_t)(e ? x >> 16 : x)));
          };
          float big = 0.0f;
          if (!idle) {
            const long at = live ? (long)(u.q_first + token) * a.q.row_stride + (long)hq * a.q.head_stride : -1;
            const uint16_t *src = static_cast<const uint16_t *>(a.q.data);
            if (wide) {
#pragma unroll
              for (int i = 0; i < PIECES; ++i) {
                const long from = row_at(at, i);
                const bool have = from >= 0 && my_col < size;
                pk_copy16(piece_of((r & 96) + i * AT_ONCE + lane / PIECES, my_piece), src + (have ? from + my_col : 0),
                          have ? 16 : 0);
              }
              asm volatile("cp.async.wait_all;\n" ::: "memory");
            } else {
#pragma unroll 1
              for (int i = 0; i < PIECES; ++i) {
                const long from = row_at(at, i);
                const uint16_t *p = src + from + my_col;
                *piece_of((r & 96) + i * AT_ONCE + lane / PIECES, my_piece) =
                    from >= 0 && my_col < size ? make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16,
                                                            p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16)
                                               : make_uint4(0, 0, 0, 0);
              }
            }
            __syncwarp();
            if (bf) {
              uint32_t top = 0;  // the largest magnitude's bits, of even and odd columns
#pragma unroll 4
              for (int j = 0; j < PIECES; ++j) {
                const uint4 v = *piece_of(r, j);
                top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                             __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
              }
              big = __uint_as_float(max(top << 16, top & 0xffff0000u));
            }
          }
          half_big[half][r] = big;
          meet(0);
          big = __uint_as_float(max(__float_as_uint(big), __float_as_uint(half_big[half ^ 1][r])));
          // bf16: by the power of two that puts the largest in [2^13, 2^14); f16: as they are.  The
          // scale's sign goes along, so that the largest score is the largest weight's.
          const int e8 = (int)(__float_as_uint(big) >> 23);
          const int ex = bf && big > 0.0f && e8 < 255 ? min(140 - max(e8, 1), 126) : 0;
          const float up = a.scale < 0.0f ? -pow2i(ex) : pow2i(ex);
          f = fabsf(a.scale) * 1.4426950408889634f * pow2i(-ex);
          if (!idle) {
#pragma unroll 2
            for (int j = 0; j < PIECES; ++j) {
              const uint4 v = *piece_of(r, j);
              const uint32_t x[4] = {v.x, v.y, v.z, v.w};
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)  // columns e and e + 4 of the eight
                y[e] = half2_bits(value(x[e >> 1], e & 1) * up, value(x[2 + (e >> 1)], e & 1) * up);
              *piece_of(r, j) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
          fence_async_smem();
          mbar_arrive(qfull);
        } else {
          meet(0);  // the sums of the unit before are read
        }
        const int p_row = u.fill + token, pos = live && p_row < a.c.positions ? max(p_row, -1) : -1;
        const int p_first = u.fill + a.by_group.of(u.rr0), p_last = u.hi - 1, past = u.past;
        float m = -INFINITY;  // the maximum in use (of scores as the products leave them) when l was last added to
        uint64_t sum = 0;
        for (int t = (step0 ^ half) & 1; t < steps; t += 2) {
          const int T = step0 + t, sb = T % L::SB;
          const int tile0 = tile_of(u, t) * TP;
          const bool all = !past && tile0 + TP - 1 <= p_first &&
                           (a.window <= 0 || tile0 > p_last - a.window || tile0 + TP <= a.sinks);
          const uint32_t at = lanes + L::T_S + sb * 64;
          uint32_t x[32];
          auto scores = [&](int c) {  // 32 of the tile's columns, what the row does not see as -inf
            tc_ld32(at + c, x);
            tc_ld_wait();
            if (!all) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const int j = tile0 + c + i;
                if (!(j <= pos && (a.window <= 0 || j > pos - a.window || j < a.sinks))) x[i] = 0xff800000u;
              }
            }
          };
          wait(&sfull[sb], T / L::SB);
          tc_after();
          float top = -INFINITY;
          if (!idle) {
#pragma unroll
            for (int c = 32; c >= 0; c -= 32) {
              scores(c);
              float mx[2] = {top, top};
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                mx[0] = fmaxf(mx[0], fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
                mx[1] = fmaxf(mx[1], fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
              }
              top = fmaxf(mx[0], mx[1]);
            }
          }
          // the maximum in use goes from tile to tile, from half to half
          float now = -INFINITY;
          if (t > 0) {
            wait(&mtold[(T - 1) & 1], (T - 1) >> 1);
            now = shared_m[(T - 1) & 1][r];
          }
          const bool grown = top > now && (now == -INFINITY || (top - now) * f > (float)L::LAG);
          const float before = now;
          if (grown) now = top;
          shared_m[T & 1][r] = now;
          mbar_arrive(&mtold[T & 1]);
          if (!idle) {
            if (__any_sync(0xffffffffu, now != m)) {
              const float back = now == m ? 1.0f : m == -INFINITY ? 0.0f : exp2_fast((m - now) * f);
              sum = mulf2(sum, pair2(back, back));
              m = now;
            }
            if (t > 0 && __any_sync(0xffffffffu, grown)) {
              const float back = !grown ? 1.0f : before == -INFINITY ? 0.0f : exp2_fast((before - now) * f);
              const uint64_t back2 = pair2(back, back);
              wait(&vdone[(T - 1) % L::SB], (T - 1) / L::SB);
              tc_after();
#pragma unroll 1
              for (int c = 0; c < HDP; c += 16) {
                uint32_t o[16];
                tc_ld16(lanes + c, o);
                tc_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                  const uint64_t y = mulf2((uint64_t)o[i] | (uint64_t)o[i + 1] << 32, back2);
                  o[i] = (uint32_t)y;
                  o[i + 1] = (uint32_t)(y >> 32);
                }
                tc_st16(lanes + c, o);
              }
            }
            const float base = now == -INFINITY ? 0.0f : now;
            const uint64_t low = pair2(-base, -base), f2 = pair2(f, f), keep = pair2(L::KEEP, L::KEEP);
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
              if (c) scores(c);  // the first half is still there
              uint32_t p[16];
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                // KEEP at the largest, however large
                const uint64_t d = fma2(add2((uint64_t)x[i] | (uint64_t)x[i + 1] << 32, low), f2, keep);
                float y = exp2_fast(first2(d)), z = exp2_fast(second2(d));
                if (!all) {
                  y = x[i] == 0xff800000u ? 0.0f : y;
                  z = x[i + 1] == 0xff800000u ? 0.0f : z;
                }
                p[i / 2] = half2_bits(y, z);
                sum = add2(sum, pair2(y, z));
              }
              tc_st16(at + c / 2, p);
            }
            tc_st_wait();
            tc_before();
          }
          mbar_arrive(&pfull[sb]);
        }
        // ---- the rows out
        float l = first2(sum) + second2(sum);
        if (steps > 0) {
          const int T = step0 + steps - 1;
          wait(&mtold[T & 1], T >> 1);
          const float now = shared_m[T & 1][r];
          if (m != now && l != 0.0f) l *= exp2_fast((m - now) * f);
          m = now;
          wait(&vdone[T % L::SB], T / L::SB);
          tc_after();
        }
        half_sum[half][r] = l;
        meet(1);
        l += half_sum[half ^ 1][r];
        if (!idle) {
          const bool wide = wide_rows(a.out), whole = u.whole;
          const float inv = whole ? (l == 0.0f ? 0.0f : __fdividef(1.0f, l)) : 1.0f;
          const long at = !live  ? -1
                          : whole ? (long)(u.q_first + token) * a.out.row_stride + (long)hq * a.out.head_stride
                                  : (long)r * size;
          // 16 bits: the half's columns at once; partial sums, in 32: half of
          // them at a time (of a 64-wide head straight from the registers)
          constexpr int PART = HDP > 64 ? HDP / 4 : 32;
          for (int c0 = half * (HDP / 2); c0 < min(size, (half + 1) * (HDP / 2)); c0 += whole ? HDP / 2 : PART) {
#pragma unroll 1
            for (int k = 0; k < (whole ? HDP / 2 : PART) / 32; ++k) {
              uint32_t o[32];
              if (steps > 0) {
                tc_ld32(lanes + c0 + 32 * k, o);
                tc_ld_wait();
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0;
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float y[8] = {__uint_as_float(o[8 * e]) * inv,     __uint_as_float(o[8 * e + 2]) * inv,
                                    __uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 6]) * inv,
                                    __uint_as_float(o[8 * e + 1]) * inv, __uint_as_float(o[8 * e + 3]) * inv,
                                    __uint_as_float(o[8 * e + 5]) * inv, __uint_as_float(o[8 * e + 7]) * inv};
                if (whole) {
                  store8(piece_of(r, 4 * k + e), a.out.type, 0, true, y);
                } else if (HDP == 64) {
                  if (live) store8(u.piece, 1, at + c0 + 8 * e, true, y);
                } else {
                  *reinterpret_cast<float4 *>(piece_of(r, 8 * k + 2 * e)) = make_float4(y[0], y[1], y[2], y[3]);
                  *reinterpret_cast<float4 *>(piece_of(r, 8 * k + 2 * e + 1)) = make_float4(y[4], y[5], y[6], y[7]);
                }
              }
            }
            if (!whole && HDP == 64) continue;
            __syncwarp();
            const int col = c0 + (whole ? 8 : 4) * my_piece;
            const bool in = col < size;
            if (whole && !wide) {
#pragma unroll 1
              for (int i = 0; i < PIECES; ++i) {
                const long to = row_at(at, i);
                const uint4 v = *piece_of((r & 96) + i * AT_ONCE + lane / PIECES, my_piece);
                uint16_t *p = static_cast<uint16_t *>(a.out.data) + to + col;
                const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                if (to >= 0 && in) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) p[2 * e] = (uint16_t)x[e], p[2 * e + 1] = (uint16_t)(x[e] >> 16);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < PIECES; ++i) {
                const long to = row_at(at, i);
                const uint4 v = *piece_of((r & 96) + i * AT_ONCE + lane / PIECES, my_piece);
                uint4 *p = whole ? reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out.data) + to + col)
                                 : reinterpret_cast<uint4 *>(u.piece + to + col);
                if (to >= 0 && in) *p = v;
              }
            }
            __syncwarp();
          }
          if (!whole && live && !half) {
            u.piece[(size_t)RB * size + r] = m == -INFINITY ? -INFINITY : m * f;
            u.piece[(size_t)RB * size + RB + r] = l;
          }
        }
        tc_before();
      }
      step0 += steps;
      spent += steps > 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[un & 1]);
    }
    if (warp == 16) {  // nor is a product, or an arrival on a barrier
      if (elect_one()) tc_commit(over);
      wait(over, 0);
    }
  }
  if (failed) pack_trouble(a.c);
  __syncthreads();
  if (warp == 16) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(0), "r"(512) : "memory");
  }
}

template <int HDP>
static cudaError_t tc_ready(PackPlan *plan) {
  static std::atomic<int> known[PACK_DEVICES];
  plan->tile = PackTc<HDP>::TP;
  plan->over = PackTc<HDP>::OVER;
  plan->pitch = PackTc<HDP>::PITCH;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < PACK_DEVICES && known[dev].load())) return e;
  e = cudaFuncSetAttribute(pack_attend_tc_kernel<HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, PackTc<HDP>::SMEM);
  if (e == cudaSuccess && dev < PACK_DEVICES) known[dev].store(1);
  return e;
}

template <int HDP>
static cudaError_t tc_run(const PackAttend &a, const PackPlan &p, const CUtensorMap &tmk, const CUtensorMap &tmv,
                          cudaStream_t st) {
  return pack_launch(pack_attend_tc_kernel<HDP>, dim3(p.grid), TC_THREADS, PackTc<HDP>::SMEM, st, false, 0, a, tmk, tmv,
                     p.tall);
}

}  // namespace igc

using namespace igc;

cudaError_t igc_pack_tc_ready(PackPlan *p) {
  return p->wide == 64 ? tc_ready<64>(p) : p->wide == 128 ? tc_ready<128>(p) : tc_ready<256>(p);
}

cudaError_t igc_launch_pack_tc(const PackAttend *a, const PackPlan *p, const CUtensorMap *tmk, const CUtensorMap *tmv,
                               cudaStream_t st) {
  return p->wide == 64    ? tc_run<64>(*a, *p, *tmk, *tmv, st)
         : p->wide == 128 ? tc_run<128>(*a, *p, *tmk, *tmv, st)
                          : tc_run<256>(*a, *p, *tmk, *tmv, st);
}
