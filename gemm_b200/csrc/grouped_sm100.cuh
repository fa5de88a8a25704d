// Products of a ragged batch with one matrix per group, for sm_100a.  The rows of the batch are
// sorted by group; group e owns rows [offsets[e], offsets[e+1]), read from device memory, so a
// router's result never has to visit the host.  One kernel template serves
//
//   kGroupedNt   y[t,n]    = sum_k x[t,k] W[e][n,k]                 (bf16)
//   kGroupedDx   dx[t,k]   = sum_n dy[t,n] W[e][n,k]                (bf16, gradient of the rows)
//   kGroupedDw   dW[e][n,k] = sum_{t in e} dy[t,n] x[t,k]           (bf16, gradient of the matrices)
//   kMxNt        y[t,n]    = sum_k x[t,k] W[e][n,k]                 (both in MXFP4: E2M1 codes, one
//                                                                   E8M0 scale per 32 values of K)
//
// all with fp32 accumulation in tensor memory and one rounding to bf16.  The dense MXFP4 product is
// the last one with a single group.
//
// Roles of a tile.  The matrix operand always takes the 128 tensor-memory lanes of a CTA (256 of a
// pair) and the rows of the batch take the accumulator's COLUMNS.  Lanes come in steps of 128, but
// the column count N of an MMA is a run-time value in steps of 16 (32 for a pair): a group of 40
// rows costs an N = 48 product instead of a 128-row tile, which is what makes ragged groups and
// single tokens cheap, and a group's rows are cut into equal tiles rather than full ones and a
// remnant.  dW has no ragged output; there the group's rows are the contraction.
//
//   warp 0      TMA producer      warp 1      UMMA issuer (leader CTA of a pair)
//   next 4 (8)  epilogue: tcgen05.ld -> bf16 -> shared memory (rows of the batch transposed on the way, by
//               stmatrix) -> 16-byte stores, dW by TMA; overlapped with the next tile through a second
//               accumulator, which the MXFP4 pair has no room for.  Where CTAs share a tile's
//               contraction: partial sums to the CTA that adds them up, straight from the accumulator
//   next one    kGroupedDw only: clears the rows of a tile's last k-block that belong to the next
//               group (both operands: a zero times a neighbour's Inf would still be NaN)
//   last one    CTAs that share a contraction only: frees the buffers of partial sums
//
// Every CTA (pair, cluster) walks tiles worker, worker + workers, ... of the list (group, lane tile,
// column tile).  Its prefix sums are in registers of each warp (up to 32 groups) or, built at the start,
// in shared memory.
// Every wait is bounded; on expiry the role records a code, raises the CTA's abort flag and falls
// through to the tear-down.
#pragma once

#include "device_errors.cuh"
#include "ptx.cuh"

namespace neogemm {

enum GroupedOp : int { kGroupedNt = 0, kGroupedDx = 1, kGroupedDw = 2, kMxNt = 3 };

constexpr int kMaxGroups = 1024;

// A buffer of partial sums: 128 lanes x 16 columns in fp32 (from each CTA of the cluster its share of
// the lanes).
constexpr int kPartCols = 16;
constexpr int kPartBytes = 128 * kPartCols * 4;
constexpr int kMaxPartBufs = 8;

struct GroupedParams {
  const void* offsets;      // groups + 1 ascending row indices, or null: one group of all rows
  int offsets_are_64;
  int groups;
  int rows;                 // rows of the batch
  int lanes;                // extent of the axis on the tensor-memory lanes (N; K for dx)
  int cols;                 // kGroupedDw: extent of the column axis (K)
  int depth;                // contraction length (K; N for dx; for dW the rows of the batch)
  int lane_tiles;           // tiles along `lanes`
  int col_cap;              // widest accumulator of a tile (a multiple of the column granularity)
  int col_box;              // rows of the ragged operand's large boxes (a CTA's share of col_cap)
  int small_box;            // and of its small ones
  int slots, per_slot;      // streaming kernels: ring slots, and the k-blocks that each takes
  int part_bufs;            // buffers of partial sums (2, 4 or 8)
  int col_tiles;            // kGroupedDw: tiles along `cols`
  int zero_rest;            // write zeros to the rows of no group (0: leave them)
  int vector_out;           // 16-byte stores are possible (alignment of base and pitches); for dW the
                            // result leaves by TMA then
  __nv_bfloat16* out;
  long long out_pitch;      // elements between rows of the result
  long long out_stack;      // kGroupedDw: elements between the groups' matrices
  int sf_row_blocks;        // kMxNt: 128-row blocks of scales per matrix of the stack
  int sf_k_blocks;          // kMxNt: 128-value blocks of scales along K
  int* status;
};

// kCtaGroup == 2: tiles of 256 lanes x up to kCols columns on CTA pairs, for groups of many rows.
//
// kSplit > 1: the streaming kernels, for groups of few rows, where the time is that of reading the
// matrices once.  A cluster of kSplit CTAs shares a tile of 128 lanes: each takes an equal part of
// the contraction, and at the end each collects the partial sums of 128 / kSplit lanes from the
// others through distributed shared memory and adds them in rank order.  So the SMs' shares differ
// by a fraction of a tile however many tiles there are (6 groups of 3584 rows are 168 tiles: in
// whole tiles, two rounds on 148 SMs for 1.14 rounds of work).  Two ways of evening out the lanes
// instead were slower: tiles of fewer lanes take as many k-blocks, each with its fixed cost, and
// contiguous runs per SM scatter the addresses that are read at a time (32 groups of 3584 x 2048:
// 102 us against 86 when this was tried).
//
// dW with kSplit > 1: for few tiles of a long contraction (two groups of 840 x 408 with 9254 rows:
// 42.2 us on single CTAs, 23 on clusters of four).
template <int kOp_, int kCtaGroup_, int kSplit_, int kCols_, int kStages_>
struct GroupedConfig {
  static constexpr int kOp = kOp_;
  static constexpr int kCtaGroup = kCtaGroup_;
  static constexpr int kCols = kCols_;              // widest accumulator (UMMA N) of a tile
  static constexpr int kStages = kStages_;          // ring slots (streaming: at most)
  static constexpr int kSplit = kSplit_;            // CTAs that share a tile's contraction
  static constexpr bool kStream = kSplit > 1 && kOp != kGroupedDw;   // ring sized at run time
  static constexpr int kCluster = kCtaGroup * kSplit;
  static constexpr int kLaneRows = 128;             // lanes per CTA
  static constexpr int kLaneTile = kLaneRows * kCtaGroup;
  static constexpr int kHalfCols = kCols / kCtaGroup;   // column rows a CTA fetches at most
  static constexpr int kBlockK = (kOp == kMxNt) ? 256 : 64;   // values of K per 128-byte row
  static constexpr int kStepK = (kOp == kMxNt) ? 64 : 16;     // values of K per MMA
  static constexpr int kColStep = 16 * kCtaGroup;   // granularity of a tile's N
  // Shared memory of one ring slot.
  static constexpr int kLaneBytes = kLaneRows * 128;
  static constexpr int kColBytes = kHalfCols * 128;
  // MXFP4: the instruction takes the scales of 128 rows from four columns of tensor memory that
  // start at a multiple of four, so lanes and columns start at multiples of 128 rows, the blocks in
  // which the scales are stored.  A group's first tile may use a part of its columns only.
  static constexpr int kScaleCols = (kCols + 127) / 128;      // blocks of scales of the columns
  static constexpr int kScaleBytes = (kOp == kMxNt) ? 1024 * (1 + kScaleCols) : 0;
  static constexpr int kStageBytes = kLaneBytes + kColBytes + kScaleBytes;
  // Two accumulators, so that a tile's epilogue overlaps the next tile's products.  The MXFP4 pair
  // takes one of 256 columns instead (the scales need the rest of tensor memory): narrower tiles are
  // bound by shared memory - 256 x 128 reads and fills 192 bytes per cycle of the 128 there are - and
  // its eight epilogue warps pull the accumulator into registers, packed, before they store anything.
  static constexpr int kAccs = (kOp == kMxNt && kCtaGroup == 2) ? 1 : 2;
  // Eight warps also where short contractions are bound by writing their result; Y and dX on pairs
  // read their matrices for longer than four take (32 groups of 3584 x 2048, 1001 rows: 79.6 us, and
  // 82.7 with eight).
  static constexpr int kEpiWarps = (kAccs == 1 || (kOp == kGroupedDw && kCtaGroup == 2)) ? 8 : 4;
  static constexpr int kEpiCols = kCols * 4 / kEpiWarps;   // columns that a warp stores at most
  // And takes into registers at a time: all of them where the next tile waits for it, else half, so that
  // nothing spills (of 227 KB shared memory no cache is left: in the MXFP4 pair a spill of 100 words
  // cost 16 us of 77).
  static constexpr int kPull = kAccs == 1 ? 128 : 64;
  // Per warp 32 x 32 bf16; kSplit > 1: buffers of partial sums instead, part_bufs of them (streaming
  // kernels: those beyond two at the expense of the ring).
  // dW: one or two boxes of 32 x 64 bf16 per warp.
  static constexpr int kBoxBufs = (kOp == kGroupedDw && kCtaGroup == 1) ? 2 : 1;
  static constexpr int kEpiWarpBytes = kOp == kGroupedDw ? 4096 * kBoxBufs : 2048;
  static constexpr int kEpiBytes = kStream ? 2 * kPartBytes : kSplit > 1 ? kMaxPartBufs * kPartBytes
                                                                       : kEpiWarps * kEpiWarpBytes;
  static constexpr int kTableBytes = (3 * kMaxGroups + 1) * 4;
  static constexpr int kBarrierBytes = (3 * kStages + 4 + 3 * kMaxPartBufs) * 8 + 16;
  static constexpr int kRestBytes = kEpiBytes + kTableBytes + 12 + kBarrierBytes + 1024;
  static constexpr int kRingBytes = kStream ? (232448 - kRestBytes) / 1024 * 1024 : kStages * kStageBytes;
  static_assert(kEpiBytes % 1024 == 0, "the ring starts on the swizzle's alignment");
  static constexpr int kSmemBytes = kRingBytes + kRestBytes;
  // The accumulators, and behind them (MXFP4) the scales of every k-block in the ring: per 128
  // values of K four columns per 128 rows.
  static constexpr int kScaleTmemCols = (kOp == kMxNt) ? 8 * (1 + kScaleCols) : 0;
  static constexpr int kScaleSets = (kOp != kMxNt) ? 0 : kStream ? (512 - kAccs * kCols) / kScaleTmemCols : kStages;
  static constexpr int kTmemNeeded = kAccs * kCols + kScaleSets * kScaleTmemCols;
  static constexpr int kTmemCols = (kCtaGroup == 2) ? 512 : kTmemNeeded <= 128 ? 128
                                 : kTmemNeeded <= 256 ? 256 : 512;
  // Behind the epilogue: the warp that clears rows (dW), and the one that frees buffers of partial sums.
  static constexpr int kClearWarp = 2 + kEpiWarps;
  static constexpr int kFreeWarp = kClearWarp + (kOp == kGroupedDw ? 1 : 0);
  static constexpr int kThreads = 32 * (kFreeWarp + (kSplit > 1 ? 1 : 0));
  // Arrivals that complete a ring slot's phase besides its bytes: the slot's producer, and for
  // dW one per CTA (the last block of a tile is handed over by the warps that cleared its rows).
  static constexpr int kFullArrivals = (kOp == kGroupedDw) ? kCtaGroup : 1;
  static_assert(kStageBytes % 1024 == 0, "every slot must keep the swizzle's alignment");
  static_assert(kSmemBytes <= 232448, "exceeds 227 KB of shared memory per CTA");
  static_assert(kSmemBytes > 116224, "one CTA per SM: tensor memory is not shared");
  static_assert(kTmemNeeded <= 512, "tensor memory");
  static_assert(kCols % 32 == 0 && kCols <= 256 && kHalfCols % 32 == 0, "columns");
  static_assert(kRingBytes - (kStream ? kMaxPartBufs - 2 : 0) * kPartBytes >= 2 * kStageBytes,
                "two full blocks");
  static_assert(kOp != kMxNt || kScaleSets >= kStages * (kStream ? 2 : 1), "scales of every k-block in the ring");
};

// What a tile computes.  Every role derives it from the tile's number.
struct GroupedTile {
  int group;
  int lane0;      // index on lane 0 of the tile
  int col_row;    // row of the ragged operand (index of the column axis for dW) in column 0
  int lo, hi;     // columns that are this tile's to store
  int mma_n;      // columns computed: hi rounded up
  int k_row;      // kGroupedDw: first row of the contraction
  int k_len;      // contraction length
  int first_kb;   // this CTA's k-blocks
  int blocks;     // (0: its sum is zero)
};

__device__ __forceinline__ void report_error(int* status, volatile int* abort_flag, int code,
                                             int tile, int aux) {
  *abort_flag = 1;
  if (status != nullptr && atomicCAS(status, 0, code) == 0) {
    status[1] = static_cast<int>(blockIdx.x);
    status[2] = tile;
    status[3] = aux;
    __threadfence_system();
  }
}

// Tiles along the columns of a group.
template <class Cfg>
__device__ __forceinline__ int column_tiles(const GroupedParams& p, int begin, int end) {
  if (end <= begin) return 0;
  if (Cfg::kOp != kMxNt && end - begin <= p.col_cap) return 1;
  if (Cfg::kOp == kMxNt) return (end - begin / 128 * 128 + Cfg::kCols - 1) / Cfg::kCols;
  return (end - begin + p.col_cap - 1) / p.col_cap;
}

// The copy and matrix instructions take their operands from the warp's uniform registers.  A value
// that the compiler cannot prove uniform, or one in a branch or loop that it cannot, is moved there
// each time it is used: about 90 cycles a copy instead of 17.  So whatever came from shared memory or
// from the thread's index is made uniform once, the conditions of the roles' loops included.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

__device__ __forceinline__ void make_uniform(GroupedTile& t) {
  t.group = uniform(t.group);
  t.lane0 = uniform(t.lane0);
  t.col_row = uniform(t.col_row);
  t.lo = uniform(t.lo);
  t.hi = uniform(t.hi);
  t.mma_n = uniform(t.mma_n);
  t.k_row = uniform(t.k_row);
  t.k_len = uniform(t.k_len);
  t.first_kb = uniform(t.first_kb);
  t.blocks = uniform(t.blocks);
}

// A wait for a phase that another CTA completes: the polls stay cheap, and one test at cluster scope behind
// them orders what follows after what that CTA did.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, const volatile int* abort_flag) {
  return ptx::mbar_wait(bar, parity, abort_flag) && ptx::mbar_wait<true>(bar, parity, abort_flag);
}

// Rows [begin, end) of group e, clamped to the batch: indices that are out of order or out of range cost
// the result, never an access.  True if they were in order.  If any were not, the ranges still overlap
// and in_order() has to follow.
__device__ __forceinline__ bool group_range(const GroupedParams& p, int e, int* begin, int* end) {
  long long b = 0, f = p.rows;
  if (p.offsets != nullptr) {
    if (p.offsets_are_64) {
      b = static_cast<const long long*>(p.offsets)[e];
      f = static_cast<const long long*>(p.offsets)[e + 1];
    } else {
      b = static_cast<const int*>(p.offsets)[e];
      f = static_cast<const int*>(p.offsets)[e + 1];
    }
  }
  const bool good = b >= 0 && f >= b && f <= p.rows;
  b = b < 0 ? 0 : b > p.rows ? p.rows : b;
  f = f < b ? b : f > p.rows ? p.rows : f;
  *begin = static_cast<int>(b);
  *end = static_cast<int>(f);
  return good;
}

// Ranges of 32 consecutive groups, one per lane, of offsets that were not in order: an index that descends
// counts as the largest in front of it (`before`, for the first lane).  So no two groups share a row - two
// tiles would store it - and there are no more tiles than in order.  (begin, end, largest index so far.)
// A call, not inline: inlined, this path that hardly ever runs cost dW of 513 rows, 8 x 1024 x 2048, 11.0 us
// instead of 10.3.
__device__ __noinline__ int3 in_order(int before, int begin, int end) {
  const int lane = static_cast<int>(ptx::lane_id());
  int top = max(end, before);
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int other = __shfl_up_sync(0xffffffffu, top, d);
    if (lane >= d) top = max(top, other);
  }
  const int previous = __shfl_up_sync(0xffffffffu, top, 1);
  return make_int3(lane > 0 ? previous : max(begin, before), top, __shfl_sync(0xffffffffu, top, 31));
}

// Records offsets that were clamped: the launch is not aborted.
__device__ __forceinline__ void report_offsets(const GroupedParams& p, int e) {
  if (blockIdx.x == 0 && p.status != nullptr && atomicCAS(p.status, 0, kDevBounds) == 0) {
    p.status[1] = 0;
    p.status[2] = e;
    p.status[3] = 4;
    __threadfence_system();
  }
}

// In shared memory, for more than 32 groups.
struct GroupTable {
  int *begin, *end;   // [kMaxGroups]
  int* first;         // [kMaxGroups + 1]
};

// The tiles of one worker (a CTA, a pair, or a cluster that splits the contraction), in order.
// Every role walks its own copy.
template <class Cfg>
struct GroupedTiles {
  // Row ranges and first tiles of the groups: up to 32 of them are held by the lanes of each warp, which
  // then needs neither shared memory nor a barrier between reading the offsets and its first tile; more
  // are in shared memory.
  const GroupTable& table;
  int my_begin, my_end, my_first, total;
  bool good;   // this lane's group was in order
  int next, last, step;
  int split_rank;
  int group, g0, g1, tiles, share;  // the group of the last tile: its rows and its columns' tiles
  int group_first, group_last;      // its first tile and the next group's

  __device__ __forceinline__ GroupedTiles(const GroupedParams& p, const GroupTable& table_, int worker,
                                          int workers, int split_rank_)
      : table(table_), good(true), next(worker), step(workers), split_rank(split_rank_),
        group_last(0) {
    if (p.groups <= 32) {
      const int lane = static_cast<int>(ptx::lane_id());
      good = group_range(p, min(lane, p.groups - 1), &my_begin, &my_end);
      if (!__all_sync(0xffffffffu, good)) {
        const int3 range = in_order(0, my_begin, my_end);
        my_begin = range.x, my_end = range.y;
      }
      const int mine = Cfg::kOp == kGroupedDw || lane >= p.groups
                           ? 0 : column_tiles<Cfg>(p, my_begin, my_end) * p.lane_tiles;
      int scan = mine;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int other = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += other;
      }
      my_first = scan - mine;
      total = __shfl_sync(0xffffffffu, scan, 31);
    } else {
      total = table.first[p.groups];
    }
    total = uniform(total);
    last = Cfg::kOp == kGroupedDw ? p.groups * p.lane_tiles * p.col_tiles : total;
  }

  __device__ __forceinline__ int begin_of(const GroupedParams& p, int e) const {
    return p.groups <= 32 ? __shfl_sync(0xffffffffu, my_begin, e) : table.begin[e];
  }
  __device__ __forceinline__ int end_of(const GroupedParams& p, int e) const {
    return p.groups <= 32 ? __shfl_sync(0xffffffffu, my_end, e) : table.end[e];
  }
  // First tile of group e <= groups.
  __device__ __forceinline__ int first_of(const GroupedParams& p, int e) const {
    if (p.groups > 32) return table.first[e];
    const int first = __shfl_sync(0xffffffffu, my_first, e & 31);
    return e < p.groups ? first : total;
  }

  __device__ __forceinline__ bool take(const GroupedParams& p, GroupedTile& t) {
    if (next >= last) return false;
    if (Cfg::kOp == kGroupedDw) {
      const int per_group = p.lane_tiles * p.col_tiles;
      t.group = next / per_group;
      const int local = next - t.group * per_group;
      const int lane_tile = local / p.col_tiles;
      t.lane0 = lane_tile * Cfg::kLaneTile;
      t.col_row = (local - lane_tile * p.col_tiles) * Cfg::kCols;
      t.lo = 0;
      t.hi = min(Cfg::kCols, p.cols - t.col_row);
      t.k_row = begin_of(p, t.group);
      t.k_len = end_of(p, t.group) - t.k_row;
    } else {
      if (next >= group_last) {
        // Last group whose first tile is not behind this one: groups without tiles share their
        // first tile with the next group and lose the comparison.  The warp looks at every 32nd
        // group, then at the 32 from there (bisection cost 500 cycles a tile in each role).
        const int lane = static_cast<int>(ptx::lane_id());
        if (p.groups <= 32) {
          group = __popc(__ballot_sync(0xffffffffu, lane < p.groups && my_first <= next)) - 1;
        } else {
          int a = 32 * (__popc(__ballot_sync(0xffffffffu, lane * 32 < p.groups &&
                                             table.first[min(lane * 32, p.groups)] <= next)) - 1);
          a += __popc(__ballot_sync(0xffffffffu, a + lane < p.groups &&
                                                     table.first[min(a + lane, p.groups)] <= next)) - 1;
          group = a;
        }
        g0 = begin_of(p, group);
        g1 = end_of(p, group);
        group_first = first_of(p, group);
        group_last = first_of(p, group + 1);
        tiles = column_tiles<Cfg>(p, g0, g1);
        // Equal shares of the columns, in steps of the MMA's granularity.
        share = Cfg::kCols;
        if (Cfg::kOp != kMxNt)
          share = ((tiles == 1 ? g1 - g0 : (g1 - g0 + tiles - 1) / tiles) + Cfg::kColStep - 1) /
                  Cfg::kColStep * Cfg::kColStep;
      }
      t.group = group;
      const int local = next - group_first;
      // Streaming: tiles that are read at a time lie side by side.
      int c, lane_tile;
      if (Cfg::kStream) {
        c = local < p.lane_tiles ? 0 : local / p.lane_tiles;
        lane_tile = local - c * p.lane_tiles;
      } else {
        lane_tile = tiles == 1 ? local : local / tiles;
        c = local - lane_tile * tiles;
      }
      t.lane0 = lane_tile * Cfg::kLaneTile;
      t.col_row = (Cfg::kOp == kMxNt ? g0 / 128 * 128 : g0) + c * share;
      t.lo = max(g0 - t.col_row, 0);
      t.hi = max(min(g1 - t.col_row, share), 0);
      t.k_row = 0;
      t.k_len = p.depth;
    }
    next += step;
    t.mma_n = max((t.hi + Cfg::kColStep - 1) / Cfg::kColStep, 1) * Cfg::kColStep;
    const int blocks = (t.k_len + Cfg::kBlockK - 1) / Cfg::kBlockK;
    t.first_kb = blocks * split_rank / Cfg::kSplit;
    t.blocks = blocks * (split_rank + 1) / Cfg::kSplit - t.first_kb;
    return true;
  }
};

// What a k-block of a tile fetches of the ragged operand, and the block's size.
template <class Cfg>
struct BlockLayout {
  bool small;             // the columns in use lie in one small box; otherwise a large one from column 0
  int first_col;          // column of the box's first row
  uint32_t fetched;       // bytes of the whole block

  __device__ __forceinline__ BlockLayout(const GroupedParams& p, const GroupedTile& t, int rank) {
    small = false;
    first_col = 0;
    if (Cfg::kOp == kGroupedDw) {
      fetched = Cfg::kLaneBytes + (t.mma_n / Cfg::kCtaGroup + 63) / 64 * 8192;
    } else {
      const int half = t.mma_n / Cfg::kCtaGroup;
      const int lo = max(t.lo - rank * half, 0), hi = max(min(t.hi - rank * half, half), 1);
      first_col = lo & ~(p.small_box - 1);
      small = hi - first_col <= p.small_box;
      if (!small) first_col = 0;
      fetched = Cfg::kLaneBytes + (small ? p.small_box : p.col_box) * 128 + Cfg::kScaleBytes;
    }
  }
};

// Tensor maps of the operands, by box: lanes (128 rows, MN-major lanes 64 x 64), columns (col_box and
// small_box rows), scales (MXFP4) of the lanes and of the columns; the result of dW (boxes of 32 rows
// x 64 columns, clipped at the matrices' edges).
struct GroupedMaps {
  CUtensorMap lanes, cols, small_cols, lane_scales, col_scales, result;
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1)
grouped_kernel(const __grid_constant__ GroupedMaps maps, const GroupedParams p) {
  using namespace ptx;
  constexpr int kCtaGroup = Cfg::kCtaGroup;
  constexpr int kStages = Cfg::kStages;
  constexpr bool kDw = Cfg::kOp == kGroupedDw;
  constexpr bool kMx = Cfg::kOp == kMxNt;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t epi_base = smem_base;
  const uint32_t ring = epi_base + (Cfg::kStream ? p.part_bufs * kPartBytes : Cfg::kEpiBytes);
  const uint32_t bar_base = epi_base + Cfg::kEpiBytes + Cfg::kRingBytes;
  const uint32_t full_bar = bar_base;                        // [kStages]
  const uint32_t empty_bar = full_bar + 8 * kStages;         // [kStages]
  const uint32_t clear_bar = empty_bar + 8 * kStages;        // [kStages] dW: last block has landed
  const uint32_t tmem_full_bar = clear_bar + 8 * kStages;    // [2]
  const uint32_t tmem_empty_bar = tmem_full_bar + 16;        // [2]
  const uint32_t part_full_bar = tmem_empty_bar + 16;                // [kMaxPartBufs] have arrived
  const uint32_t part_read_bar = part_full_bar + 8 * kMaxPartBufs;   // and been read by this CTA's warps
  const uint32_t part_free_bar = part_read_bar + 8 * kMaxPartBufs;   // all CTAs' may be written again
  uint8_t* tail_gen = smem_gen + (part_free_bar + 8 * kMaxPartBufs - smem_base);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(tail_gen);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail_gen + 4);
  int* const words = reinterpret_cast<int*>(tail_gen + 16);
  const GroupTable table{words, words + kMaxGroups, words + 2 * kMaxGroups};

  const int warp = uniform(static_cast<int>(threadIdx.x >> 5));
  const uint32_t lane = lane_id();
  const int cluster_rank = (Cfg::kCluster > 1) ? uniform(static_cast<int>(cluster_ctarank())) : 0;
  const int rank = (kCtaGroup == 2) ? cluster_rank : 0;          // in a pair
  const int split_rank = (Cfg::kSplit > 1) ? cluster_rank : 0;   // along the contraction
  const bool is_leader = rank == 0;
  const int worker = static_cast<int>(blockIdx.x) / Cfg::kCluster;
  const int num_workers = static_cast<int>(gridDim.x) / Cfg::kCluster;

  // ---------------------------------------------------------------- set-up
  if (threadIdx.x == 0) {
    griddep_launch_dependents();
    *abort_flag = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar + 8 * s, Cfg::kFullArrivals);
      mbar_init(empty_bar + 8 * s, 1);
      mbar_init(clear_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tmem_full_bar + 8 * a, 1);
      mbar_init(tmem_empty_bar + 8 * a, Cfg::kEpiWarps * kCtaGroup);
    }
    fence_barrier_init();
  }
  if (Cfg::kSplit > 1 && threadIdx.x >= 32 * Cfg::kFreeWarp && static_cast<int>(lane) < p.part_bufs) {
    mbar_init(part_full_bar + 8 * lane, 1);
    mbar_init(part_read_bar + 8 * lane, 4);
    mbar_init(part_free_bar + 8 * lane, Cfg::kSplit);
    fence_barrier_init();
    mbar_arrive_expect_tx(part_full_bar + 8 * lane, kPartBytes);
  }
  if (warp == 0 && lane == 0 && p.depth > 0) {   // without a contraction there are no maps
    prefetch_tensormap(&maps.lanes);
    prefetch_tensormap(&maps.cols);
    if (!kDw) prefetch_tensormap(&maps.small_cols);
    if (kDw && p.vector_out) prefetch_tensormap(&maps.result);
    if (kMx) {
      prefetch_tensormap(&maps.lane_scales);
      prefetch_tensormap(&maps.col_scales);
    }
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::kTmemCols);
    tmem_relinquish<1>();
  }
  tcgen05_fence_before();
  if (Cfg::kCluster > 1) cluster_sync_all(); else __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = uniform(*tmem_slot);
  // The pair's MMA addresses both CTAs' tensor memory with the leader's address.
  const bool usable = kCtaGroup == 1 || tmem_base == 0;
  if (!usable && threadIdx.x == 0)
    report_error(p.status, abort_flag, kDevTmemAddress, 0, static_cast<int>(tmem_base));
  // Global memory from here on: wait for the previous kernel of the stream.
  griddep_wait();
  if (p.groups > 32) {
    int bad = 0;
    for (int e = threadIdx.x; e < p.groups; e += Cfg::kThreads)
      if (!group_range(p, e, table.begin + e, table.end + e)) {
        report_offsets(p, e);
        bad = 1;
      }
    bad = __syncthreads_or(bad);
    if (warp == 0) {
      int sum = 0, top = 0;
      for (int base = 0; base < p.groups; base += 32) {
        const int e = base + static_cast<int>(lane);
        if (bad) {
          const int3 range = in_order(top, e < p.groups ? table.begin[e] : 0, e < p.groups ? table.end[e] : 0);
          if (e < p.groups) table.begin[e] = range.x, table.end[e] = range.y;
          top = range.z;
        }
        const int mine =
            !kDw && e < p.groups ? column_tiles<Cfg>(p, table.begin[e], table.end[e]) * p.lane_tiles : 0;
        int scan = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const int other = __shfl_up_sync(0xffffffffu, scan, d);
          if (static_cast<int>(lane) >= d) scan += other;
        }
        if (e < p.groups) table.first[e] = sum + scan - mine;
        sum += __shfl_sync(0xffffffffu, scan, 31);
      }
      if (lane == 0) table.first[p.groups] = sum;
    }
    __syncthreads();
  }
  GroupedTiles<Cfg> tiles(p, table, worker, num_workers, split_rank);
  GroupedTile t;
  int tile = 0;   // of this worker, for error records
  // Ring slots.  Streaming: sized for the widest tile of the launch, of one or two k-blocks.
  const uint32_t col_bytes = Cfg::kStream ? p.col_box * 128 : Cfg::kColBytes;
  const uint32_t block_bytes = Cfg::kLaneBytes + col_bytes + Cfg::kScaleBytes;
  const int per_slot = Cfg::kStream ? p.per_slot : 1;
  const uint32_t slot_bytes = block_bytes * per_slot;
  const uint32_t slots = Cfg::kStream ? p.slots : kStages;

  // ---------------------------------------------------------------- roles
  if (!usable) {
    // Nothing is issued.
  } else if (warp == 0) {
    // ======================= TMA producer =======================
    uint32_t stage = 0, phase = 0;
    const uint32_t leader_full = (kCtaGroup == 2) ? mapa_u32(full_bar, 0) : full_bar;
    bool ok = true;
    for (; ok && tiles.take(p, t); ++tile) {
      make_uniform(t);
      const BlockLayout<Cfg> at(p, t, rank);
      const uint32_t fetched = uniform(at.fetched);
      uint32_t expected = at.fetched;   // by the leader of a pair: for both CTAs
      if (kCtaGroup == 2) expected += BlockLayout<Cfg>(p, t, 1 - rank).fetched;
      expected = uniform(expected);
      const bool small = uniform(at.small) != 0;
      const int first_col = uniform(at.first_col);
      const int half = t.mma_n / kCtaGroup;
      const int lane_row = t.lane0 + rank * Cfg::kLaneRows;
      const int col_row = t.col_row + rank * half + first_col;
      const CUtensorMap* map_c = small ? &maps.small_cols : &maps.cols;
      const uint32_t to_cols = Cfg::kLaneBytes + first_col * 128;
      const uint32_t to_scales = Cfg::kLaneBytes + col_bytes;
      int scale_row = 0, col_scale_row = 0;
      if (kMx) {
        scale_row = (t.group * p.sf_row_blocks + lane_row / 128) * p.sf_k_blocks;
        col_scale_row = t.col_row / 128;
      }
      for (int kb0 = 0; kb0 < t.blocks; kb0 += per_slot) {
        ok = __all_sync(0xffffffffu, mbar_wait(empty_bar + 8 * stage, phase ^ 1, abort_flag));
        if (!ok) {
          if (lane == 0)
            report_error(p.status, abort_flag, kDevTimeoutProducer, tile, static_cast<int>(stage));
          break;
        }
        const int blocks = Cfg::kStream ? min(per_slot, t.blocks - kb0) : 1;
        uint32_t sl = ring + stage * slot_bytes;
        // dW: the last block of a group's rows is handed over by the warp that clears its tail.
        const bool clear = kDw && t.k_len - (t.first_kb + kb0) * 64 < 64;
        const uint32_t own = (clear ? clear_bar : full_bar) + 8 * stage;
        const uint32_t bar = (kCtaGroup == 1 || clear) ? own : leader_full + 8 * stage;
        if (elect_one()) {
          if (kCtaGroup == 1 || clear) {
            mbar_arrive_expect_tx(own, fetched * blocks);
          } else if (is_leader) {
            mbar_arrive_expect_tx(own, expected);
            if (kDw) mbar_arrive(own);
          }
        }
        __syncwarp();
        // Everything a copy needs is worked out outside the elected lane's branch, where the warp's
        // uniform registers hold it: 17 cycles a copy, against about 95 inside.
        for (int j = 0; j < blocks; ++j, sl += block_bytes) {
          const int kb = t.first_kb + kb0 + j;
          const uint32_t sc = sl + to_cols, ss = sl + to_scales;
          const int k0 = kb * (kMx ? 128 : 64);   // first element (MXFP4: byte) of the block
          const int row = t.k_row + k0;
          const int scales_l = scale_row + 2 * kb;
          auto load = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2) {
            if (kCtaGroup == 1 || clear) tma_load_3d(dst, map, bar, c0, c1, c2);
            else tma_load_3d_pair(dst, map, bar, c0, c1, c2);
          };
          if (elect_one()) {
            if constexpr (kDw) {
              load(sl, &maps.lanes, lane_row, row, 0);
              load(sl + 8192, &maps.lanes, lane_row + 64, row, 0);
#pragma unroll
              for (int b = 0; b < Cfg::kHalfCols / 64; ++b)
                if (b * 64 < half) load(sc + b * 8192, &maps.cols, col_row + b * 64, row, 0);
            } else {
              if constexpr (Cfg::kOp == kGroupedDx) {
                load(sl, &maps.lanes, lane_row, k0, t.group);
                load(sl + 8192, &maps.lanes, lane_row + 64, k0, t.group);
              } else {
                load(sl, &maps.lanes, k0, lane_row, t.group);
              }
              load(sc, map_c, k0, col_row, 0);
              if constexpr (kMx) {
                // Two consecutive 512-byte tiles of scales (128 rows x 128 values of K each) per
                // block of rows; past the end of K they are other tiles or zero fill, and not used.
                load(ss, &maps.lane_scales, 0, scales_l, 0);
                load(ss + 1024, &maps.col_scales, 0, 2 * kb, col_scale_row);
              }
            }
          }
          __syncwarp();
        }
        if (++stage == slots) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ======================= UMMA issuer =======================
    if (is_leader) {
      uint32_t stage = 0, phase = 0;
      int count = 0;   // tiles with a contraction so far: their accumulators alternate
      const uint32_t sets_per_slot = Cfg::kScaleSets / slots;
      bool ok = true;
      for (; ok && tiles.take(p, t); ++tile) {
        if (t.blocks == 0) continue;
        make_uniform(t);
        const uint32_t acc = count % Cfg::kAccs, acc_phase = (count / Cfg::kAccs) & 1;
        ++count;
        if (!__all_sync(0xffffffffu, mbar_wait<kCtaGroup == 2, Cfg::kAccs == 1>(
                                             tmem_empty_bar + 8 * acc, acc_phase ^ 1, abort_flag))) {
          if (lane == 0)
            report_error(p.status, abort_flag, kDevTimeoutMmaTmem, tile, static_cast<int>(acc));
          break;
        }
        tcgen05_fence_after();
        const uint32_t tmem_d = tmem_base + acc * Cfg::kCols;
        const uint32_t idesc =
            kMx ? make_idesc_mxf4(Cfg::kLaneTile, static_cast<uint32_t>(t.mma_n))
                : make_idesc_bf16(Cfg::kLaneTile, static_cast<uint32_t>(t.mma_n)) |
                      (Cfg::kOp == kGroupedDx ? kIdescTransposeA : 0u) |
                      (kDw ? kIdescTransposeA | kIdescTransposeB : 0u);
        for (int kb0 = 0; kb0 < t.blocks; kb0 += per_slot) {
          if (!__all_sync(0xffffffffu,
                          mbar_wait<kDw && kCtaGroup == 2>(full_bar + 8 * stage, phase, abort_flag))) {
            if (lane == 0)
              report_error(p.status, abort_flag, kDevTimeoutMmaFull, tile, static_cast<int>(stage));
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const int blocks = Cfg::kStream ? min(per_slot, t.blocks - kb0) : 1;
          uint32_t sl = ring + stage * slot_bytes;
          for (int j = 0; j < blocks; ++j, sl += block_bytes) {
            const int kb = t.first_kb + kb0 + j;
            const uint32_t sc = sl + Cfg::kLaneBytes;
            // A K-major operand moves 32 bytes along its swizzled rows per step, an MN-major one two
            // groups of eight rows.
            constexpr uint64_t kLaneStep = (kDw || Cfg::kOp == kGroupedDx) ? 128 : 2;
            constexpr uint64_t kColStepDesc = kDw ? 128 : 2;
            const uint64_t dl = (kLaneStep == 128) ? make_smem_desc_mn_sw128(sl, 8192)
                                                   : make_smem_desc_sw128(sl);
            const uint64_t dc = kDw ? make_smem_desc_mn_sw128(sc, 8192) : make_smem_desc_sw128(sc);
            const int left = t.k_len - kb * Cfg::kBlockK;
            const uint32_t first = kb0 + j > 0 ? 1u : 0u;
            if constexpr (kMx) {
              // Scales of 128 values of K: four columns of tensor memory per block of 128 rows.
              const uint32_t set = Cfg::kStream ? stage * sets_per_slot + j : stage;
              const uint32_t tsl = tmem_base + Cfg::kAccs * Cfg::kCols + set * Cfg::kScaleTmemCols;
              const uint32_t tsc = tsl + 8;
              const uint64_t ds = make_smem_desc_scales(sc + col_bytes);
              if (elect_one()) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  tmem_copy_32x128b_x4<kCtaGroup>(tsl + h * 4, ds + h * 32);
#pragma unroll
                  for (int b = 0; b < Cfg::kScaleCols; ++b)
                    tmem_copy_32x128b_x4<kCtaGroup>(tsc + (h * Cfg::kScaleCols + b) * 4,
                                                    ds + 64 * (1 + b) + h * 32);
                }
                // (A test per step between the instructions doubles the time of issuing them.)
                auto step = [&](int k) {
                  umma_mxf4<kCtaGroup>(tmem_d, dl + 2 * k, dc + 2 * k,
                                       idesc | idesc_scale_bytes((k & 1) * 2), tsl + (k >> 1) * 4,
                                       tsc + (k >> 1) * Cfg::kScaleCols * 4, k > 0 ? 1u : first);
                };
                if (left >= Cfg::kBlockK) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) step(k);
                } else {
                  for (int k = 0; k * Cfg::kStepK < left; ++k) step(k);
                }
              }
            } else {
              if (elect_one()) {
                auto step = [&](int k) {
                  umma_bf16<kCtaGroup>(tmem_d, dl + kLaneStep * k, dc + kColStepDesc * k, idesc,
                                       k > 0 ? 1u : first);
                };
                if (left >= Cfg::kBlockK) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) step(k);
                } else {
                  for (int k = 0; k * Cfg::kStepK < left; ++k) step(k);
                }
              }
            }
            __syncwarp();
          }
          if (elect_one()) {
            if (kCtaGroup == 2) umma_commit_both_ctas(empty_bar + 8 * stage);
            else umma_commit<1>(empty_bar + 8 * stage);
          }
          __syncwarp();
          if (++stage == slots) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if (elect_one()) {
          if (kCtaGroup == 2) umma_commit_both_ctas(tmem_full_bar + 8 * acc);
          else umma_commit<1>(tmem_full_bar + 8 * acc);
        }
        __syncwarp();
      }
    }
  } else if (warp < 2 + Cfg::kEpiWarps) {
    // ======================= epilogue =======================
    constexpr int kPull = Cfg::kPull;
    const int quad = warp & 3;   // the warp's quarter of the tensor-memory lanes
    const int first_col = (warp - 2) / 4 * Cfg::kEpiCols;   // and its share of the columns
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t stage_buf = epi_base + (warp - 2) * Cfg::kEpiWarpBytes;
    uint32_t buf = 0;   // dW: the warp's next box
    int count = 0;
    int parts = 0;   // column groups of partial sums so far
    for (; tiles.take(p, t); ++tile) {
      const uint32_t acc = count % Cfg::kAccs, acc_phase = (count / Cfg::kAccs) & 1;
      if (t.blocks > 0) {
        ++count;
        if (!__all_sync(0xffffffffu, mbar_wait(tmem_full_bar + 8 * acc, acc_phase, abort_flag))) {
          if (lane == 0)
            report_error(p.status, abort_flag, kDevTimeoutEpilogue, tile, static_cast<int>(acc));
          break;
        }
        tcgen05_fence_after();
      }
      const int lane_first = t.lane0 + rank * Cfg::kLaneRows + quad * 32;   // of this warp
      const int lane_end = p.lanes;
      const int cols_end = min(t.hi, first_col + Cfg::kEpiCols);   // of this warp
      auto in_use = [&](int c) { return lane_first < lane_end && c < cols_end && c + 32 > t.lo; };
      auto hand_back = [&] {
        if (t.blocks == 0) return;
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kCtaGroup == 2) mbar_arrive_cluster(mapa_u32(tmem_empty_bar + 8 * acc, 0));
          else mbar_arrive(tmem_empty_bar + 8 * acc);
        }
      };
      // Up to kPull columns of this warp's lanes from `c`, rounded to bf16 and packed in pairs of
      // columns: lane by lane for dW, else as fragments of 8 x 8 matrices, which leave transposed.
      // The accumulator goes back after the last load.
      auto pull = [&](int c, uint32_t (&w)[kPull / 32][16]) {
        __syncwarp();   // the aligned loads need the warp converged after its predicated stores
        if (t.blocks == 0) {
#pragma unroll
          for (int i = 0; i < kPull / 32; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) w[i][j] = 0u;
          return;
        }
#pragma unroll
        for (int h = 0; h < kPull / 32; h += 2) {
          uint32_t r[2][32];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t at = tmem_base + acc * Cfg::kCols + lane_base + c + (h + i) * 32;
            if (in_use(c + (h + i) * 32)) {
              if constexpr (kDw) {
                tmem_ld_32x32b_x32(at, r[i]);
              } else {
                tmem_ld_16x256b_x4(at, reinterpret_cast<uint32_t(&)[16]>(r[i][0]));
                tmem_ld_16x256b_x4(at + (16u << 16), reinterpret_cast<uint32_t(&)[16]>(r[i][16]));
              }
            }
          }
          tmem_ld_wait();
          if ((h + 2) * 32 == kPull && c + kPull >= cols_end) hand_back();
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[h + i][j] = pack_bf16x2(__uint_as_float(r[i][2 * j]), __uint_as_float(r[i][2 * j + 1]));
        }
      };
      // A block of 32 rows x 32 values of the result through shared memory: 64 bytes a row, 16-byte units
      // swizzled against conflicts.
      auto store = [&](int c, const uint32_t (&w)[16]) {
        const uint32_t s = stage_buf;
        auto unit_at = [&](int row, int unit) { return s + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4); };
        __syncwarp();   // the previous block has been read
        if constexpr (kDw) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st_shared_v4(unit_at(lane, j), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        } else {
          // Eight rows of the batch at a time: w[2 u + s + 8 h] holds columns 8 u .. of lanes 16 h + 8 s ..
#pragma unroll
          for (int u = 0; u < 4; ++u)
            st_matrix_x4_trans(unit_at(u * 8 + (lane & 7), lane >> 3), w[2 * u], w[2 * u + 1],
                               w[8 + 2 * u], w[8 + 2 * u + 1]);
        }
        __syncwarp();
        // Rows [from, to) of the block exist, and `width` values of each.
        const int from = kDw ? 0 : max(t.lo - c, 0);
        const int to = kDw ? min(lane_end - lane_first, 32) : min(t.hi - c, 32);
        const int width = kDw ? t.hi - c : lane_end - lane_first;
        __nv_bfloat16* first =
            kDw ? p.out + t.group * p.out_stack + lane_first * p.out_pitch + t.col_row + c
                : p.out + static_cast<long long>(t.col_row + c) * p.out_pitch + lane_first;
        if (p.vector_out) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + static_cast<int>(lane >> 2), unit = static_cast<int>(lane & 3);
            const int left = width - unit * 8;
            if (row < from || row >= to || left <= 0) continue;
            uint32_t v[4];
            ld_shared_v4(unit_at(row, unit), v);
            __nv_bfloat16* dst = first + row * p.out_pitch + unit * 8;
            if (left >= 8) {
              *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (j < left)
                  reinterpret_cast<unsigned short*>(dst)[j] =
                      static_cast<unsigned short>(v[j >> 1] >> ((j & 1) * 16));
            }
          }
        } else {
          // Rows that do not start on 16 bytes: a row per instruction, 64 bytes side by side.
          // (Eight values per lane, as above, took three times as long for 310 x 127: 20.3 and 7.9 us.)
#pragma unroll 1
          for (int row0 = 0; row0 < 32; row0 += 4) {
            unsigned short v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = ld_shared_b16(unit_at(row0 + i, lane >> 3) + (lane & 7) * 2);
            unsigned short* dst =
                reinterpret_cast<unsigned short*>(first + row0 * p.out_pitch) + lane;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (row0 + i >= from && row0 + i < to && static_cast<int>(lane) < width)
                dst[i * p.out_pitch] = v[i];
          }
        }
      };
      if constexpr (Cfg::kSplit > 1) {
        // Partial sums, kPartCols columns at a time: this warp's lanes go to the CTA that collects
        // them, [source][four columns][lane][4]; then this warp adds up four columns of the lanes
        // that its own CTA collects.  The next columns are on their way meanwhile.
        constexpr int kSplit = Cfg::kSplit, kOwn = 128 / kSplit;   // lanes that a CTA collects
        constexpr uint32_t kSource = kOwn * kPartCols * 4;
        const uint32_t dest = quad * kSplit / 4;
        const uint32_t dest_lane = (quad * 32) % kOwn + lane;
        const uint32_t dest_base = mapa_u32(epi_base, dest) + split_rank * kSource + dest_lane * 16;
        const uint32_t dest_full = mapa_u32(part_full_bar, dest);
        const int part_mask = p.part_bufs - 1, part_shift = __popc(part_mask);
        const int c_first = t.lo & ~(kPartCols - 1);
        bool ok = true;
        auto send = [&](int c, int n) {
          uint32_t r[16];
          __syncwarp();   // the aligned load needs the warp converged after its predicated stores
          if (t.blocks > 0) {
            tmem_ld_32x32b_x16(tmem_base + acc * Cfg::kCols + lane_base + c, r);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) r[j] = 0u;
          }
          const uint32_t b = n & part_mask;
          ok = ok && __all_sync(0xffffffffu, wait_cluster(part_free_bar + 8 * b,
                                                          ((n >> part_shift) & 1) ^ 1, abort_flag));
          if (!ok) return;
          // (Ordinary stores and a release at cluster scope took 1500 cycles: the release waits for
          // every store in flight, those of the result included.)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            st_async_v4(dest_base + b * kPartBytes + j * (kOwn * 16), dest_full + 8 * b, r[4 * j],
                        r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        };
        auto collect = [&](int c, int n) {
          const uint32_t b = n & part_mask;
          ok = ok && __all_sync(0xffffffffu, wait_cluster(part_full_bar + 8 * b, (n >> part_shift) & 1,
                                                          abort_flag));
          if (!ok) return;
          // Arm the buffer for its next use: nothing can arrive before this warp has read it, below.
          if (quad == 0 && lane == 0) mbar_arrive_expect_tx(part_full_bar + 8 * b, kPartBytes);
          float sum[kOwn / 32][4];
#pragma unroll
          for (int h = 0; h < kOwn / 32; ++h) {
            const uint32_t at = epi_base + b * kPartBytes + (quad * kOwn + h * 32 + lane) * 16;
#pragma unroll
            for (int q = 0; q < kSplit; ++q) {
              uint32_t v[4];
              ld_shared_v4(at + q * kSource, v);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                sum[h][j] = q == 0 ? __uint_as_float(v[j]) : sum[h][j] + __uint_as_float(v[j]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(part_read_bar + 8 * b);
#pragma unroll
          for (int h = 0; h < kOwn / 32; ++h) {
            const int n_out = t.lane0 + split_rank * kOwn + h * 32 + static_cast<int>(lane);
            const int row = c + quad * 4;
            if constexpr (kDw) {   // four neighbours of a row
              __nv_bfloat16* dst = p.out + t.group * p.out_stack + n_out * p.out_pitch + t.col_row + row;
              if (n_out >= p.lanes || row >= t.hi) continue;
              if (p.vector_out) {
                *reinterpret_cast<uint2*>(dst) =
                    make_uint2(pack_bf16x2(sum[h][0], sum[h][1]), pack_bf16x2(sum[h][2], sum[h][3]));
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (row + j < t.hi) dst[j] = __float2bfloat16_rn(sum[h][j]);
              }
              continue;
            }
            __nv_bfloat16* dst = p.out + static_cast<long long>(t.col_row + row) * p.out_pitch + n_out;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (row + j >= t.lo && row + j < t.hi && n_out < p.lanes)
                dst[j * p.out_pitch] = __float2bfloat16_rn(sum[h][j]);
          }
        };
        send(c_first, parts);
        for (int c = c_first; c < t.hi; c += kPartCols) {
          const int n = parts++;
          if (c + kPartCols < t.hi) send(c + kPartCols, n + 1);
          else hand_back();   // all of the accumulator has been read
          collect(c, n);
        }
        if (!ok) {
          if (lane == 0) report_error(p.status, abort_flag, kDevTimeoutEpilogue, tile, 2);
          break;
        }
      } else {
        const int c_first = max(first_col, t.lo & ~31);
        if (!in_use(c_first)) hand_back();
        for (int c = c_first; in_use(c); c += kPull) {
          uint32_t w[kPull / 32][16];
          pull(c, w);
          if (kDw && p.vector_out) {
            // 32 rows x 64 columns through the warp's 4 KB as one swizzled box (dW of short groups is
            // bound by its stores).
#pragma unroll
            for (int i = 0; i < kPull / 32; i += 2) {
              if (!in_use(c + i * 32)) continue;
              if (lane == 0) tma_store_wait_read<Cfg::kBoxBufs - 1>();
              __syncwarp();
              const uint32_t box = stage_buf + buf * 4096;
              buf = (buf + 1) % Cfg::kBoxBufs;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint32_t* v = &w[i + j / 4][4 * (j & 3)];
                st_shared_v4(box + lane * 128 + ((j ^ (lane & 7)) << 4), v[0], v[1], v[2], v[3]);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_3d(&maps.result, box, t.col_row + c + i * 32, lane_first, t.group);
                tma_store_commit();
              }
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < kPull / 32; ++i)
            if (in_use(c + i * 32)) store(c + i * 32, w[i]);
        }
      }
    }
    // Shared memory outlives the stores' reads of it.
    if (kDw && lane == 0) tma_store_wait_read<0>();
    __syncwarp();
    if (!kDw && p.zero_rest) {
      // Rows of no group: in front of the first and behind the last.
      const int head = tiles.begin_of(p, 0), tail = tiles.end_of(p, p.groups - 1);
      const int rest = head + p.rows - tail;
      for (int i = static_cast<int>(blockIdx.x) * Cfg::kEpiWarps + warp - 2; i < rest;
           i += static_cast<int>(gridDim.x) * Cfg::kEpiWarps) {
        const int row = i < head ? i : tail + i - head;
        __nv_bfloat16* dst = p.out + static_cast<long long>(row) * p.out_pitch;
        int c = static_cast<int>(lane) * 8;
        if (p.vector_out)
          for (; c + 8 <= p.lanes; c += 256)
            *reinterpret_cast<uint4*>(dst + c) = make_uint4(0, 0, 0, 0);
        for (; c < p.lanes; c += 256)
          for (int j = c; j < min(c + 8, p.lanes); ++j) dst[j] = __float2bfloat16_rn(0.f);
      }
    }
  } else if (kDw && warp == Cfg::kClearWarp) {
    // ======================= rows of the next group =======================
    uint32_t stage = 0, parities = 0;
    bool ok = true;
    for (; ok && tiles.take(p, t); ++tile) {
      if (t.blocks == 0) continue;
      const int valid = t.k_len - (t.first_kb + t.blocks - 1) * 64;   // rows of the last block
      stage = (stage + t.blocks - 1) % kStages;
      if (valid < 64) {
        if (!__all_sync(0xffffffffu, mbar_wait(clear_bar + 8 * stage, (parities >> stage) & 1,
                                               abort_flag))) {
          if (lane == 0)
            report_error(p.status, abort_flag, kDevTimeoutProducer, tile, static_cast<int>(stage));
          ok = false;
          break;
        }
        parities ^= 1u << stage;
        // A box is 64 rows of 128 bytes; the swizzle moves bytes inside a row only.  The products
        // stop at the next multiple of 16 rows.
        const uint32_t last_byte = static_cast<uint32_t>((valid + 15) / 16 * 16) * 128;
        const uint32_t sl = ring + stage * Cfg::kStageBytes;
        const int boxes = 2 + (t.mma_n / kCtaGroup + 63) / 64;   // the lane operand's two in front
        for (int b = 0; b < boxes; ++b)
          for (uint32_t o = static_cast<uint32_t>(valid) * 128 + lane * 16; o < last_byte; o += 512)
            st_shared_v4(sl + b * 8192 + o, 0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (kCtaGroup == 2) mbar_arrive_release_cluster(mapa_u32(full_bar + 8 * stage, 0));
          else mbar_arrive(full_bar + 8 * stage);
        }
      }
      stage = (stage + 1) % kStages;
    }
  } else if (Cfg::kSplit > 1) {
    // ======================= buffers of partial sums: back to the senders =======================
    // The senders overwrite what this CTA's four warps have read, so the loads have to be ordered in front
    // of their next stores by a release at cluster scope.  That takes 1200 to 4200 cycles while the SM
    // streams, whichever warp does it (in the epilogue's own, 16 x 28672 x 8192 in MXFP4: 30.7 us with its
    // quantisation, 27.7 here; 32 groups of 3584 x 2048 with two rows each: 35.6 and 27).  So a warp of its own
    // does it, once for all that has been read meanwhile, and not at all for buffers that no later step
    // fills.
    const int bufs = p.part_bufs, mask = bufs - 1, shift = __popc(mask);
    int known = 0;   // column groups of the tiles looked at: these are to come
    bool ok = true, more = true;
    for (int n = 0; ok;) {
      while (more && known <= n + 2 * bufs) {
        more = tiles.take(p, t);
        if (more) known += (t.hi + kPartCols - 1) / kPartCols - t.lo / kPartCols;
      }
      if (known <= n + bufs) break;
      ok = __all_sync(0xffffffffu, mbar_wait(part_read_bar + 8 * (n & mask), (n >> shift) & 1, abort_flag));
      if (!ok) {
        if (lane == 0) report_error(p.status, abort_flag, kDevTimeoutEpilogue, n, 3);
        break;
      }
      int end = n + 1;
      while (end < n + bufs && known > end + bufs &&
             __all_sync(0xffffffffu, mbar_test_wait(part_read_bar + 8 * (end & mask), (end >> shift) & 1)))
        ++end;
      if (lane < Cfg::kSplit) {
        fence_cluster();
        for (; n < end; ++n) mbar_arrive_relaxed_cluster(mapa_u32(part_free_bar + 8 * (n & mask), lane));
      }
      __syncwarp();
      n = end;
    }
  }
  __syncwarp();

  if (warp == 0 && !tiles.good) report_offsets(p, min(static_cast<int>(lane), p.groups - 1));
  __syncwarp();

  // ---------------------------------------------------------------- tear-down
  tcgen05_fence_before();
  if (Cfg::kCluster > 1) cluster_sync_all(); else __syncthreads();
  if (*abort_flag != 0) {
    // Let boxes still in flight land in this CTA's shared memory before it is released.
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
    if (Cfg::kCluster > 1) cluster_sync_all(); else __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc<1>(tmem_base, Cfg::kTmemCols);
  }
}

}  // namespace neogemm
