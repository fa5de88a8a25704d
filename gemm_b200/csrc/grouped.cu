// Host side of the grouped and MXFP4 products (contracts: include/neogemm.h; kernel:
// grouped_sm100.cuh).
#include "../../include/neogemm.h"

#include <algorithm>
#include <cstring>
#include <mutex>

#include "grouped_sm100.cuh"
#include "host.cuh"

namespace neogemm {
namespace {

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxExtent = 0x7fffffffll - 4096;   // room for tile coordinates past the end
constexpr int64_t kMaxPitch = 1ll << 38;              // elements; keeps every product below in 64 bits

struct KernelEntry {
  int op, cta_group, split, columns, stages;
  int lane_step;   // lanes of a tile
  int col_step;    // granularity of a tile's columns
  int lane_box;    // rows of the lane operand's boxes
  int ring_bytes, scale_bytes;   // shared memory: the ring, and the scales of a k-block
  const void* fn;
  int smem_bytes, threads;
};

template <class Cfg>
KernelEntry make_entry() {
  constexpr bool kMnMajor = Cfg::kOp == kGroupedDw || Cfg::kOp == kGroupedDx;   // boxes of 64 x 64
  return KernelEntry{Cfg::kOp, Cfg::kCtaGroup, Cfg::kSplit, Cfg::kCols, Cfg::kStages, Cfg::kLaneTile,
                     Cfg::kColStep, kMnMajor ? 64 : 128, Cfg::kRingBytes, Cfg::kScaleBytes,
                     reinterpret_cast<const void*>(&grouped_kernel<Cfg>),
                     Cfg::kSmemBytes, Cfg::kThreads};
}

// [operation][variant]; the middle one of dW splits its contraction, the narrow one does not
enum Variant : int { kNarrow = 0, kWide = 1, kMiddle = 2, kVariants = 3 };
const KernelEntry kKernels[4][kVariants] = {
    {make_entry<GroupedConfig<kGroupedNt, 1, 4, 128, 8>>(), make_entry<GroupedConfig<kGroupedNt, 2, 1, 256, 6>>(),
     make_entry<GroupedConfig<kGroupedNt, 1, 2, 128, 8>>()},
    {make_entry<GroupedConfig<kGroupedDx, 1, 4, 128, 8>>(), make_entry<GroupedConfig<kGroupedDx, 2, 1, 256, 6>>(),
     make_entry<GroupedConfig<kGroupedDx, 1, 2, 128, 8>>()},
    {make_entry<GroupedConfig<kGroupedDw, 1, 1, 128, 5>>(), make_entry<GroupedConfig<kGroupedDw, 2, 1, 256, 5>>(),
     make_entry<GroupedConfig<kGroupedDw, 1, 4, 128, 4>>()},
    {make_entry<GroupedConfig<kMxNt, 1, 4, 128, 8>>(), make_entry<GroupedConfig<kMxNt, 2, 1, 256, 5>>(),
     make_entry<GroupedConfig<kMxNt, 1, 2, 128, 8>>()},
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tensor map of a stack of matrices, innermost dimension first; pitches in bytes.  Every operand has
// three dimensions, so that one copy instruction serves all of them.
int encode(const DeviceView& dev, CUtensorMap* map, CUtensorMapDataType type, const void* base,
           int64_t inner, int64_t rows, int64_t stack, int64_t pitch, int64_t stack_pitch,
           uint32_t box_inner, uint32_t box_rows, bool swizzle, uint32_t box_stack = 1) {
  if (pitch % 16 != 0 || stack_pitch % 16 != 0 || pitch >= (1ll << 40) || stack_pitch >= (1ll << 40))
    return NEOGEMM_ERR_UNSUPPORTED;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(stack)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch), static_cast<cuuint64_t>(stack_pitch)};
  const cuuint32_t box[3] = {box_inner, box_rows, box_stack}, ones[3] = {1, 1, 1};
  auto try_encode = [&] {
    return dev.encode(
        map, type, 3, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
        swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (try_encode()) return NEOGEMM_OK;
  // A host thread that has made no runtime call yet (autograd runs a backward pass in one of its own) has
  // no context for the driver call: bind the device's and try again.
  if (cudaSetDevice(dev.index) == cudaSuccess && try_encode()) return NEOGEMM_OK;
  cudaGetLastError();
  return NEOGEMM_ERR_DESCRIPTOR;
}

// bf16 matrices, boxes of 64 elements (a 128-byte swizzle row); pitches in elements.  A single
// matrix's distance to the next is nobody's to use.
int encode_bf16(const DeviceView& dev, CUtensorMap* map, const void* base, int64_t inner,
                int64_t rows, int64_t stack, int64_t pitch, int64_t stack_pitch, int64_t box_rows) {
  return encode(dev, map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, inner, rows, stack, pitch * 2,
                (stack == 1 ? pitch : stack_pitch) * 2, 64, static_cast<uint32_t>(box_rows), true);
}

int launch(const DeviceView& dev, const KernelEntry& k, int64_t tiles_at_most,
           const GroupedMaps& maps, const GroupedParams& params, cudaStream_t stream) {
  const int cluster = k.cta_group * k.split;
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.blockDim = dim3(static_cast<unsigned>(k.threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(k.smem_bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int nattr = 0;
  if (cluster > 1) {
    attr[nattr].id = cudaLaunchAttributeClusterDimension;
    attr[nattr].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[nattr].val.clusterDim.y = 1;
    attr[nattr].val.clusterDim.z = 1;
    ++nattr;
  }
  cfg.attrs = attr;
  cfg.numAttrs = nattr;

  // Clusters that the device holds at a time: the launch is one such wave, with a fixed list of
  // tiles for each.
  static std::mutex mu;
  static int resident[kMaxDevices][4][kVariants] = {};
  const int variant = static_cast<int>(&k - kKernels[k.op]);
  int workers;
  {
    std::lock_guard<std::mutex> lock(mu);
    int& known = resident[dev.index][k.op][variant];
    if (known == 0) {
      RelaxedCapture relaxed;
      if (cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem_bytes) !=
          cudaSuccess) {
        cudaGetLastError();
        return NEOGEMM_ERR_LAUNCH;
      }
      int most = dev.sm_count / cluster;
      if (cluster > 1) {
        cfg.gridDim = dim3(static_cast<unsigned>(most * cluster), 1, 1);
        int fit = 0;
        if (cudaOccupancyMaxActiveClusters(&fit, k.fn, &cfg) != cudaSuccess || fit < 1) {
          cudaGetLastError();
          return NEOGEMM_ERR_LAUNCH;
        }
        most = std::min(most, fit);
      }
      known = most;
    }
    workers = known;
  }
  workers = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(workers, tiles_at_most)));
  cfg.gridDim = dim3(static_cast<unsigned>(workers * cluster), 1, 1);
  if (tuning_value(10) != 0) {
    // The kernel's set-up overlaps the tail of the stream's previous kernel (see launcher.cu).
    attr[nattr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[nattr].val.programmaticStreamSerializationAllowed = 1;
    ++nattr;
  }
  cfg.numAttrs = nattr;
  void* args[2] = {const_cast<GroupedMaps*>(&maps), const_cast<GroupedParams*>(&params)};
  if (cudaLaunchKernelExC(&cfg, k.fn, args) != cudaSuccess) {
    cudaGetLastError();
    return NEOGEMM_ERR_LAUNCH;
  }
  record_config(k.cta_group, k.columns, k.stages, 1, static_cast<int>(cfg.gridDim.x), 0);
  return NEOGEMM_OK;
}

// Checks that every entry point shares.
int check_extents(const void* offsets, int64_t groups, int64_t T, int64_t N, int64_t K,
                  int offsets_are_64) {
  if (groups < 0 || T < 0 || N < 0 || K < 0) return NEOGEMM_ERR_BAD_ARG;
  if (groups > kMaxGroups || T > kMaxExtent || N > kMaxExtent || K > kMaxExtent)
    return NEOGEMM_ERR_UNSUPPORTED;
  if (groups > 0 && offsets == nullptr) return NEOGEMM_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(offsets) & (offsets_are_64 ? 7 : 3)) != 0)
    return NEOGEMM_ERR_UNSUPPORTED;
  return NEOGEMM_OK;
}

int zero_rows(void* out, int64_t pitch, int64_t rows, int64_t width, cudaStream_t stream) {
  DeviceView dev;
  const int rc = acquire_device(&dev);
  if (rc != NEOGEMM_OK) return rc;
  if (cudaMemset2DAsync(out, static_cast<size_t>(pitch) * 2, 0, static_cast<size_t>(width) * 2,
                        static_cast<size_t>(rows), stream) != cudaSuccess) {
    cudaGetLastError();
    return NEOGEMM_ERR_CUDA;
  }
  return NEOGEMM_OK;
}

// Sizes that the rows' products share.  Streaming kernels keep as many columns per tile as a group
// is likely to need (four times the average and some); a group of more rows reads its matrix once per
// tile.
int fill_rows(const KernelEntry& k, int64_t groups, int64_t T, int64_t lanes, GroupedParams* p,
              int64_t* tiles_at_most) {
  int64_t cap = k.columns;
  if (k.split > 1) {
    // MXFP4 tiles take their rows from a frame of the whole batch.
    const int64_t likely = k.op == kMxNt ? T : std::min(T, 4 * (T / groups) + 16);
    cap = std::min(cap, ceil_div(likely, k.col_step) * k.col_step);
  }
  const int64_t lane_tiles = ceil_div(lanes, k.lane_step);
  // MXFP4 tiles that start in front of their group may touch one more than its length says.
  const int64_t tiles = lane_tiles * (2 * std::min(groups, T) + T / (k.op == kMxNt ? k.columns : cap));
  if (tiles > kMaxExtent) return NEOGEMM_ERR_UNSUPPORTED;
  *tiles_at_most = tiles;
  p->lane_tiles = static_cast<int>(lane_tiles);
  p->col_cap = static_cast<int>(cap);
  // A CTA fetches its columns as one box: a small one where that covers them (tails of groups).
  p->col_box = static_cast<int>(ceil_div(cap / k.cta_group, 16) * 16);
  p->small_box = std::min(p->col_box, 32);
  if (p->col_box > 32) p->col_box = static_cast<int>(ceil_div(p->col_box, 32) * 32);
  if (k.split > 1) {
    // Slots of two k-blocks where four of them fit: half the waits.
    const int block = 128 * 128 + p->col_box * 128 + k.scale_bytes;
    // Buffers of partial sums for two tiles of the average or more, up to eight: a buffer is free again some
    // 1200 to 4200 cycles after it was read.  The ring gets the rest of shared memory (32 groups of 3584 x
    // 2048, bf16, four-way: 24 rows each 90 us with eight buffers, 83 with four; 64 x 28672 x 8192 in MXFP4
    // 27 with eight, 43 with two).
    p->part_bufs = cap <= kPartCols ? 2 : T / groups <= 2 * kPartCols ? 4 : kMaxPartBufs;
    const int ring_bytes = k.ring_bytes - (p->part_bufs - 2) * kPartBytes;
    p->per_slot = ring_bytes / (2 * block) >= 4 ? 2 : 1;
    p->slots = std::min(k.stages, ring_bytes / (p->per_slot * block));
  }
  return NEOGEMM_OK;
}

// Which kernel serves a product, from the average rows of a group (the groups themselves are known to
// the GPU only).  Measured, us, four-way / two-way split / pairs, groups of equal length:
//   bf16, 32 groups of 3584 x 2048:  2 rows a group 71.5 73.2 77.1   16: 78.7 81.3 79.3
//                                    24: 83.3 84.9 80.0              128: 153 105 90
//   dX, the same groups:             2: 71.8 70.5 71.6   8: 79 72.6 72.9   15: 77 73.0 72.9   64: 93 85 76.8
//   MXFP4, the same groups:          0.25: 11.2 8.2 8.1  4: 34.5 25.0 24.9   16: 37.1 25.6 25.1
//   MXFP4, one matrix 28672 x 8192:  16: 22.8 25.5 25.5  64: 27.0 31.6 26.8  96: 33.6 34.8 27.7
// MXFP4 tiles of several groups reach over the batch's frame of 128 rows, so the pairs pay off from
// 8 rows a group on; a single matrix has no such waste.  Where a few long tiles would leave most pairs
// idle their contraction is split after all: estimated in k-blocks, eight of which stand for a tile's
// start and end (512 x 1024 x 8192 in MXFP4: 10.7 13.8 14.0; dX of 946 rows, 8 groups of 3704 x 424:
// 14.5 20.5 26.2); a ratio of 1.4 allows for the exchange of partial sums.  Below, the four-way split is
// taken where each CTA still has several k-blocks of a tile, or where there is at most about one tile per
// cluster (8 groups of 1024 x 1024, 2 rows: 4.9 5.7 6.2); many tiles of a short contraction have nothing
// to split (dX of 373 rows, 52 groups of 112 x 1344: 25.0 14.4 8.1).
int variant_of(int op, int64_t groups, int64_t T, int64_t lanes, int64_t depth, int sm_count) {
  const int forced = tuning_value(13);
  if (forced >= 0) return forced;
  const bool mx = op == kMxNt;
  const int64_t blocks = ceil_div(depth, mx ? 256 : 64), rows = T / groups;
  const int64_t wide_from = mx ? (groups == 1 ? 96 : 8) : op == kGroupedDx ? 8 : 24;
  if (rows >= wide_from) {
    const int64_t tiles = ceil_div(lanes, 256) * groups * ceil_div(rows, 256);
    const int64_t split_tiles = ceil_div(lanes, 128) * groups * ceil_div(rows, 128);
    const int64_t pairs = std::max(sm_count / 2, 1), fours = std::max(sm_count * 2 / 9, 1);
    const int64_t wide = ceil_div(tiles, pairs) * (blocks + 8);
    const int64_t two = ceil_div(split_tiles, pairs) * (ceil_div(blocks, 2) + 8);
    const int64_t four = ceil_div(split_tiles, fours) * (ceil_div(blocks, 4) + 8);
    if (5 * wide <= 7 * std::min(two, four)) return kWide;
    return four < two ? kNarrow : kMiddle;
  }
  const int64_t tiles = ceil_div(lanes, 128) * std::min(groups, T);
  if (tiles > sm_count && blocks < 8) return kWide;
  return blocks >= (mx ? 16 : 24) || tiles <= 40 ? kNarrow : kMiddle;
}

// Y or dX: rows of the batch in, rows out.
int grouped_rows(int op, const void* R, const void* W, void* out, const void* offsets,
                 int offsets_are_64, int64_t groups, int64_t T, int64_t N, int64_t K, int64_t ldr,
                 int64_t ldw, int64_t stack_w, int64_t ldo, int zero_rest, cudaStream_t stream) {
  int rc = check_extents(offsets, groups, T, N, K, offsets_are_64);
  if (rc != NEOGEMM_OK) return rc;
  const int64_t depth = op == kGroupedDx ? N : K;    // contraction
  const int64_t lanes = op == kGroupedDx ? K : N;    // width of the result
  if (T == 0 || lanes == 0) return NEOGEMM_OK;
  if (out == nullptr || ldo < lanes) return NEOGEMM_ERR_BAD_ARG;
  if (ldo > kMaxPitch || ldr > kMaxPitch || ldw > kMaxPitch || stack_w > kMaxPitch)
    return NEOGEMM_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(out) & 1) != 0) return NEOGEMM_ERR_UNSUPPORTED;
  if (groups == 0) return zero_rest ? zero_rows(out, ldo, T, lanes, stream) : NEOGEMM_OK;
  if (depth > 0) {
    if (R == nullptr || W == nullptr || ldr < depth || ldw < K) return NEOGEMM_ERR_BAD_ARG;
    if (groups > 1 && stack_w <= 0) return NEOGEMM_ERR_BAD_ARG;
    if (ldr % 8 != 0 || ldw % 8 != 0 || (groups > 1 && stack_w % 8 != 0) || !aligned16(R) ||
        !aligned16(W))
      return NEOGEMM_ERR_UNSUPPORTED;
  }
  DeviceView dev;
  rc = acquire_device(&dev);
  if (rc != NEOGEMM_OK) return rc;

  const KernelEntry& k = kKernels[op][variant_of(op, groups, T, lanes, depth, dev.sm_count)];
  GroupedParams p;
  std::memset(&p, 0, sizeof(p));
  p.offsets = offsets;
  p.offsets_are_64 = offsets_are_64;
  p.groups = static_cast<int>(groups);
  p.rows = static_cast<int>(T);
  p.lanes = static_cast<int>(lanes);
  p.depth = static_cast<int>(depth);
  int64_t tiles;
  rc = fill_rows(k, groups, T, lanes, &p, &tiles);
  if (rc != NEOGEMM_OK) return rc;
  GroupedMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (depth > 0) {
    rc = encode_bf16(dev, &maps.lanes, W, K, N, groups, ldw, stack_w, k.lane_box);
    if (rc == NEOGEMM_OK) rc = encode_bf16(dev, &maps.cols, R, depth, T, 1, ldr, 0, p.col_box);
    if (rc == NEOGEMM_OK) rc = encode_bf16(dev, &maps.small_cols, R, depth, T, 1, ldr, 0, p.small_box);
    if (rc != NEOGEMM_OK) return rc;
  }
  p.zero_rest = zero_rest;
  p.vector_out = ldo % 8 == 0 && aligned16(out);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_pitch = ldo;
  p.status = dev.status;
  return launch(dev, k, tiles, maps, p, stream);
}

// Scale tiles as a matrix of 512-byte rows, read two at a time, of one or more blocks of rows.
int encode_scales(const DeviceView& dev, CUtensorMap* map, const void* base, int64_t tiles,
                  int64_t row_blocks, int box_blocks) {
  return encode(dev, map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 128, tiles, row_blocks, 512,
                512 * tiles, 128, 2, false, static_cast<uint32_t>(box_blocks));
}

int encode_codes(const DeviceView& dev, CUtensorMap* map, const void* base, int64_t K, int64_t rows,
                 int64_t stack, int64_t box_rows) {
  return encode(dev, map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, K / 2, rows, stack, K / 2,
                stack == 1 ? K / 2 : K / 2 * rows, 128, static_cast<uint32_t>(box_rows), true);
}

int mx_rows(const void* Xc, const void* Xs, const void* Wc, const void* Ws, void* Y,
            const void* offsets, int offsets_are_64, int64_t groups, int64_t T, int64_t N, int64_t K,
            int64_t ldy, int zero_rest, cudaStream_t stream) {
  if (T == 0 || N == 0) return NEOGEMM_OK;
  if (Y == nullptr || ldy < N) return NEOGEMM_ERR_BAD_ARG;
  if (ldy > kMaxPitch) return NEOGEMM_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(Y) & 1) != 0 || K % 64 != 0) return NEOGEMM_ERR_UNSUPPORTED;
  if (groups == 0) return zero_rest ? zero_rows(Y, ldy, T, N, stream) : NEOGEMM_OK;
  if (K > 0) {
    if (Xc == nullptr || Xs == nullptr || Wc == nullptr || Ws == nullptr) return NEOGEMM_ERR_BAD_ARG;
    if (!aligned16(Xc) || !aligned16(Xs) || !aligned16(Wc) || !aligned16(Ws))
      return NEOGEMM_ERR_UNSUPPORTED;
  }
  DeviceView dev;
  int rc = acquire_device(&dev);
  if (rc != NEOGEMM_OK) return rc;

  const KernelEntry& k = kKernels[kMxNt][variant_of(kMxNt, groups, T, N, K, dev.sm_count)];
  const int64_t k_tiles = ceil_div(K, 128), w_tiles = ceil_div(N, 128), x_tiles = ceil_div(T, 128);
  if (groups * w_tiles * k_tiles > kMaxExtent) return NEOGEMM_ERR_UNSUPPORTED;
  GroupedParams p;
  std::memset(&p, 0, sizeof(p));
  p.offsets = offsets;
  p.offsets_are_64 = offsets_are_64;
  p.groups = static_cast<int>(groups);
  p.rows = static_cast<int>(T);
  p.lanes = static_cast<int>(N);
  p.depth = static_cast<int>(K);
  int64_t tiles;
  rc = fill_rows(k, groups, T, N, &p, &tiles);
  if (rc != NEOGEMM_OK) return rc;
  GroupedMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (K > 0) {
    rc = encode_codes(dev, &maps.lanes, Wc, K, N, groups, k.lane_box);
    if (rc == NEOGEMM_OK) rc = encode_codes(dev, &maps.cols, Xc, K, T, 1, p.col_box);
    if (rc == NEOGEMM_OK) rc = encode_codes(dev, &maps.small_cols, Xc, K, T, 1, p.small_box);
    if (rc == NEOGEMM_OK) rc = encode_scales(dev, &maps.lane_scales, Ws, groups * w_tiles * k_tiles, 1, 1);
    if (rc == NEOGEMM_OK)
      rc = encode_scales(dev, &maps.col_scales, Xs, k_tiles, x_tiles, (k.columns + 127) / 128);
    if (rc != NEOGEMM_OK) return rc;
  }
  p.zero_rest = zero_rest;
  p.vector_out = ldy % 8 == 0 && aligned16(Y);
  p.out = static_cast<__nv_bfloat16*>(Y);
  p.out_pitch = ldy;
  p.sf_row_blocks = static_cast<int>(w_tiles);
  p.sf_k_blocks = static_cast<int>(k_tiles);
  p.status = dev.status;
  return launch(dev, k, tiles, maps, p, stream);
}

}  // namespace
}  // namespace neogemm

using namespace neogemm;

extern "C" {

int neogemm_grouped_nt(const void* X, const void* W, void* Y, const void* offsets,
                       int offsets_are_64, int64_t groups, int64_t T, int64_t N, int64_t K,
                       int64_t ldx, int64_t ldw, int64_t stack_w, int64_t ldy, int zero_rest,
                       void* stream) {
  return grouped_rows(kGroupedNt, X, W, Y, offsets, offsets_are_64, groups, T, N, K, ldx, ldw,
                      stack_w, ldy, zero_rest, static_cast<cudaStream_t>(stream));
}

int neogemm_grouped_dx(const void* dY, const void* W, void* dX, const void* offsets,
                       int offsets_are_64, int64_t groups, int64_t T, int64_t N, int64_t K,
                       int64_t lddy, int64_t ldw, int64_t stack_w, int64_t lddx, int zero_rest,
                       void* stream) {
  return grouped_rows(kGroupedDx, dY, W, dX, offsets, offsets_are_64, groups, T, N, K, lddy, ldw,
                      stack_w, lddx, zero_rest, static_cast<cudaStream_t>(stream));
}

int neogemm_grouped_dw(const void* dY, const void* X, void* dW, const void* offsets,
                       int offsets_are_64, int64_t groups, int64_t T, int64_t N, int64_t K,
                       int64_t lddy, int64_t ldx, void* stream) {
  int rc = check_extents(offsets, groups, T, N, K, offsets_are_64);
  if (rc != NEOGEMM_OK) return rc;
  if (groups == 0 || N == 0 || K == 0) return NEOGEMM_OK;
  if (dW == nullptr) return NEOGEMM_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(dW) & 1) != 0) return NEOGEMM_ERR_UNSUPPORTED;
  if (T > 0) {
    if (dY == nullptr || X == nullptr || lddy < N || ldx < K) return NEOGEMM_ERR_BAD_ARG;
    if (lddy > kMaxPitch || ldx > kMaxPitch) return NEOGEMM_ERR_UNSUPPORTED;
    if (lddy % 8 != 0 || ldx % 8 != 0 || !aligned16(dY) || !aligned16(X))
      return NEOGEMM_ERR_UNSUPPORTED;
  }
  DeviceView dev;
  rc = acquire_device(&dev);
  if (rc != NEOGEMM_OK) return rc;

  // Tiles of 128 x 128 on single CTAs, or 256 x 256 on pairs where those have a tile each and a
  // contraction that is longer than writing its result.  Measured, us, single / pairs: 32 groups of
  // 2048 x 1024 with 32 rows 31.5 33.0, 128 rows 40.7 42.3, 512 rows 89.3 77.0; of 27 groups of
  // 2608 x 1032 with 12 rows 37.5 40.8, 128 rows 56.2 54.1; 8 groups of 1024 x 2048 with 64 rows
  // 10.4 11.9; 4 groups of 256 x 512 with 2048 rows 11.4 18.4.
  // Few tiles of a long contraction share it in clusters of four, at the cost of 14 blocks of 64 rows a
  // tile.  Single / four: one group of 128 x 128 with 1024 rows 6.4 7.1, 2048 rows 9.5 7.9; 4 groups of
  // 256 x 512 with 1024 rows 6.8 8.3, 2048 rows 9.9 9.3; 8 of them with 2048 rows 10.2 13.6, 4096 rows
  // 16.6 16.8; 2 of 840 x 408 with 4627 rows 32.1 23.8.
  const int forced = tuning_value(13);
  const int64_t pair_tiles = groups * ceil_div(N, 256) * ceil_div(K, 256);
  const int64_t single_tiles = groups * ceil_div(N, 128) * ceil_div(K, 128);
  const int64_t blocks = ceil_div(T, 64 * groups), fours = std::max(dev.sm_count * 2 / 9, 1);
  int variant = kNarrow;
  if (pair_tiles >= dev.sm_count && T / groups >= 128) variant = kWide;
  else if (single_tiles <= dev.sm_count && ceil_div(single_tiles, fours) * (blocks + 56) < 4 * blocks)
    variant = kMiddle;
  if (forced >= 0) variant = forced;
  const KernelEntry& k = kKernels[kGroupedDw][variant];
  GroupedMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (T > 0) {
    rc = encode_bf16(dev, &maps.lanes, dY, N, T, 1, lddy, 0, 64);
    if (rc == NEOGEMM_OK) rc = encode_bf16(dev, &maps.cols, X, K, T, 1, ldx, 0, 64);
    if (rc != NEOGEMM_OK) return rc;
  }
  GroupedParams p;
  std::memset(&p, 0, sizeof(p));
  p.offsets = offsets;
  p.offsets_are_64 = offsets_are_64;
  p.groups = static_cast<int>(groups);
  p.rows = static_cast<int>(T);
  p.lanes = static_cast<int>(N);
  p.cols = static_cast<int>(K);
  p.depth = static_cast<int>(T);
  const int64_t lane_tiles = ceil_div(N, k.lane_step), col_tiles = ceil_div(K, k.columns);
  const int64_t tiles = groups * lane_tiles * col_tiles;
  if (tiles > kMaxExtent) return NEOGEMM_ERR_UNSUPPORTED;
  p.lane_tiles = static_cast<int>(lane_tiles);
  p.col_tiles = static_cast<int>(col_tiles);
  p.part_bufs = kMaxPartBufs;
  p.vector_out = K % 8 == 0 && aligned16(dW);
  if (p.vector_out) {
    rc = encode_bf16(dev, &maps.result, dW, K, N, groups, K, N * K, 32);
    if (rc != NEOGEMM_OK) return rc;
  }
  p.out = static_cast<__nv_bfloat16*>(dW);
  p.out_pitch = K;
  p.out_stack = N * K;
  p.status = dev.status;
  return launch(dev, k, tiles, maps, p, static_cast<cudaStream_t>(stream));
}

int neogemm_mxfp4_nt(const void* A_codes, const void* A_scales, const void* B_codes,
                     const void* B_scales, void* C, int64_t M, int64_t N, int64_t K, int64_t ldc,
                     void* stream) {
  if (M < 0 || N < 0 || K < 0) return NEOGEMM_ERR_BAD_ARG;
  if (M > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return NEOGEMM_ERR_UNSUPPORTED;
  return mx_rows(A_codes, A_scales, B_codes, B_scales, C, nullptr, 0, 1, M, N, K, ldc, 0,
                 static_cast<cudaStream_t>(stream));
}

int neogemm_grouped_mxfp4_nt(const void* X_codes, const void* X_scales, const void* W_codes,
                             const void* W_scales, void* Y, const void* offsets,
                             int offsets_are_64, int64_t groups, int64_t T, int64_t N, int64_t K,
                             int64_t ldy, int zero_rest, void* stream) {
  const int rc = check_extents(offsets, groups, T, N, K, offsets_are_64);
  if (rc != NEOGEMM_OK) return rc;
  return mx_rows(X_codes, X_scales, W_codes, W_scales, Y, offsets, offsets_are_64, groups, T, N, K,
                 ldy, zero_rest, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
