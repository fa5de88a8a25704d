// Conversion between bf16 / fp32 and MXFP4 (format and contracts: include/neogemm.h).
//
// Both directions move each value once and are bound by HBM.  A lane owns 8 consecutive values (16
// bytes of bf16), four lanes a block of 32; a warp covers 256 values of K in four rows that are 32
// apart, because those are the rows whose scales are neighbours in the format: lane 0 of the first
// and of the second 128 values each write their 16 bytes of scales as one word vector.
#include "../../include/neogemm.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <cstring>

#include "host.cuh"
#include "ptx.cuh"

namespace neogemm {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsPerItem = 4;     // rows r, r + 32, r + 64, r + 96 of a block of 128

struct ConvertParams {
  const void* x;
  unsigned char* codes;
  unsigned char* scales;
  __nv_bfloat16* y;
  long long stack, rows, K, ldx, stack_x;
  long long row_blocks, k_tiles, k_items;   // 128-row blocks, 128-value tiles, 256-value items
  long long items;
};

struct Item {
  long long matrix, row_block, k0, row;     // row: r % 32 of the item's rows
};

__device__ __forceinline__ Item item_of(const ConvertParams& p, long long i) {
  Item it;
  it.k0 = (i % p.k_items) * 256;
  i /= p.k_items;
  it.row = i % 32;
  i /= 32;
  it.row_block = i % p.row_blocks;
  it.matrix = i / p.row_blocks;
  return it;
}

__device__ __forceinline__ long long scale_tile(const ConvertParams& p, const Item& it) {
  return ((it.matrix * p.row_blocks + it.row_block) * p.k_tiles + it.k0 / 128) * 512 + it.row * 16;
}

// Two fp32 to E2M1, nearest even, saturating: `lo` in the low four bits of the byte.
__device__ __forceinline__ uint32_t e2m1_pair(float lo, float hi) {
  uint32_t out;
  asm("{\n"
      ".reg .b8 b;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n"
      "cvt.u32.u8 %0, b;\n"
      "}\n" : "=r"(out) : "f"(hi), "f"(lo));
  return out;
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads) mxfp4_quantize_kernel(const ConvertParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kThreads / 32);
  for (long long i = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
       i < p.items; i += warps) {
    const Item it = item_of(p, i);
    const long long k = it.k0 + lane * 8;
    const bool in_k = k < p.K;       // K is a multiple of 32: a block is inside or outside
    float v[kRowsPerItem][8];
#pragma unroll
    for (int q = 0; q < kRowsPerItem; ++q) {
      const long long row = it.row_block * 128 + q * 32 + it.row;
      const bool in = in_k && row < p.rows;
      const long long at = it.matrix * p.stack_x + row * p.ldx + k;
      if (kF32) {
        float4 a = make_float4(0, 0, 0, 0), b = a;
        if (in) {
          const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + at);
          a = src[0];
          b = src[1];
        }
        v[q][0] = a.x; v[q][1] = a.y; v[q][2] = a.z; v[q][3] = a.w;
        v[q][4] = b.x; v[q][5] = b.y; v[q][6] = b.z; v[q][7] = b.w;
      } else {
        uint4 a = make_uint4(0, 0, 0, 0);
        if (in) a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.x) + at);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[q][2 * j] = __uint_as_float(w[j] << 16);
          v[q][2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
    uint32_t words[kRowsPerItem];   // the four scales of this lane's 128 values, row by row
#pragma unroll
    for (int q = 0; q < kRowsPerItem; ++q) {
      const long long row = it.row_block * 128 + q * 32 + it.row;
      const bool in = in_k && row < p.rows;
      // Largest magnitude as bits: ordered like the values, with Inf and NaN on top.
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[q][j]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const uint32_t e = top >> 23;
      const bool bad = e == 255;
      const uint32_t s = e > 2 ? e - 2 : 0;            // biased exponent of the block's scale
      const float up = __uint_as_float((254 - s) << 23);   // 2^(127 - s): a normal number
      uint32_t code = 0;
      if (!bad) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          code |= e2m1_pair(v[q][2 * j] * up, v[q][2 * j + 1] * up) << (8 * j);
      }
      if (in)
        reinterpret_cast<uint32_t*>(p.codes)[((it.matrix * p.rows + row) * p.K + k) >> 3] = code;
      // The block's four lanes agree; gather four blocks' bytes into a word.
      uint32_t byte = in ? (bad ? 255u : s) : 0u;
      uint32_t word = byte << (8 * ((lane >> 2) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      words[q] = word;
    }
    if ((lane & 15) == 0 && (it.k0 + lane * 8) / 128 < p.k_tiles)
      *reinterpret_cast<uint4*>(p.scales + scale_tile(p, it) + (lane >> 4) * 512) =
          make_uint4(words[0], words[1], words[2], words[3]);
  }
}

// An E2M1 code as fp32: exponent and mantissa sit three bits wide; code 1 is the subnormal 0.5.
__device__ __forceinline__ float e2m1_value(uint32_t code) {
  const uint32_t m = code & 7;
  const uint32_t bits = m == 0 ? 0u : m == 1 ? 0x3f000000u : (m << 22) + 0x3f000000u;
  return __uint_as_float(bits | ((code & 8) << 28));
}

__global__ void __launch_bounds__(kThreads) mxfp4_dequantize_kernel(const ConvertParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kThreads / 32);
  for (long long i = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
       i < p.items; i += warps) {
    const Item it = item_of(p, i);
    const long long k = it.k0 + lane * 8;
    if (k >= p.K) continue;
    const uint4 sw = *reinterpret_cast<const uint4*>(p.scales + scale_tile(p, it) + (lane >> 4) * 512);
    const uint32_t words[kRowsPerItem] = {sw.x, sw.y, sw.z, sw.w};
    uint32_t code[kRowsPerItem];
#pragma unroll
    for (int q = 0; q < kRowsPerItem; ++q) {
      const long long row = it.row_block * 128 + q * 32 + it.row;
      code[q] = row < p.rows
          ? reinterpret_cast<const uint32_t*>(p.codes)[((it.matrix * p.rows + row) * p.K + k) >> 3]
          : 0u;
    }
#pragma unroll
    for (int q = 0; q < kRowsPerItem; ++q) {
      const long long row = it.row_block * 128 + q * 32 + it.row;
      if (row >= p.rows) continue;
      const uint32_t s = (words[q] >> (8 * ((lane >> 2) & 3))) & 255u;
      // 2^(s - 127); the smallest is half of the smallest normal number.
      const float scale = __uint_as_float(s == 255 ? 0x7fc00000u : s == 0 ? 0x00400000u : s << 23);
      uint32_t out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        out[j] = ptx::pack_bf16x2(e2m1_value(code[q] >> (8 * j)) * scale,
                                  e2m1_value(code[q] >> (8 * j + 4)) * scale);
      *reinterpret_cast<uint4*>(p.y + (it.matrix * p.rows + row) * p.K + k) =
          make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void fill(ConvertParams& p, int64_t stack, int64_t rows, int64_t K) {
  p.stack = stack;
  p.rows = rows;
  p.K = K;
  p.row_blocks = (rows + 127) / 128;
  p.k_tiles = (K + 127) / 128;
  p.k_items = (K + 255) / 256;
  p.items = stack * p.row_blocks * 32 * p.k_items;
}

int launch(const DeviceView& dev, const void* fn, ConvertParams& p, cudaStream_t stream) {
  // Eight blocks of 256 threads fill an SM.
  const long long blocks = std::min<long long>((p.items + kThreads / 32 - 1) / (kThreads / 32),
                                               8ll * dev.sm_count);
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tuning_value(10) != 0 ? 1 : 0;
  void* args[1] = {&p};
  if (cudaLaunchKernelExC(&cfg, fn, args) != cudaSuccess) {
    cudaGetLastError();
    return NEOGEMM_ERR_LAUNCH;
  }
  return NEOGEMM_OK;
}

int check(int64_t stack, int64_t rows, int64_t K, const void* codes, const void* scales) {
  if (stack < 0 || rows < 0 || K < 0) return NEOGEMM_ERR_BAD_ARG;
  if (K % 32 != 0) return NEOGEMM_ERR_UNSUPPORTED;
  // Extents far past any memory would overflow the products below.
  if (stack > (1ll << 31) || rows > (1ll << 31) || K > (1ll << 31)) return NEOGEMM_ERR_UNSUPPORTED;
  if (stack == 0 || rows == 0 || K == 0) return NEOGEMM_OK;
  if (stack * rows > (1ll << 45) / K) return NEOGEMM_ERR_UNSUPPORTED;
  if (codes == nullptr || scales == nullptr) return NEOGEMM_ERR_BAD_ARG;
  if (!aligned16(codes) || !aligned16(scales)) return NEOGEMM_ERR_UNSUPPORTED;
  return NEOGEMM_OK;
}

}  // namespace
}  // namespace neogemm

using namespace neogemm;

extern "C" {

int neogemm_mxfp4_quantize(const void* X, int x_is_f32, void* codes, void* scales, int64_t stack,
                           int64_t rows, int64_t K, int64_t ldx, int64_t stack_x, void* stream) {
  int rc = check(stack, rows, K, codes, scales);
  if (rc != NEOGEMM_OK) return rc;
  if (stack == 0 || rows == 0 || K == 0) return NEOGEMM_OK;
  if (X == nullptr || ldx < K || stack_x < 0) return NEOGEMM_ERR_BAD_ARG;
  if (!aligned16(X) || ldx % 8 != 0 || (stack > 1 && stack_x % 8 != 0)) return NEOGEMM_ERR_UNSUPPORTED;
  DeviceView dev;
  rc = acquire_device(&dev);
  if (rc != NEOGEMM_OK) return rc;
  ConvertParams p;
  std::memset(&p, 0, sizeof(p));
  fill(p, stack, rows, K);
  p.x = X;
  p.codes = static_cast<unsigned char*>(codes);
  p.scales = static_cast<unsigned char*>(scales);
  p.ldx = ldx;
  p.stack_x = stack_x;
  const void* fn = x_is_f32 ? reinterpret_cast<const void*>(&mxfp4_quantize_kernel<true>)
                            : reinterpret_cast<const void*>(&mxfp4_quantize_kernel<false>);
  return launch(dev, fn, p, static_cast<cudaStream_t>(stream));
}

int neogemm_mxfp4_dequantize(const void* codes, const void* scales, void* Y, int64_t stack,
                             int64_t rows, int64_t K, void* stream) {
  int rc = check(stack, rows, K, codes, scales);
  if (rc != NEOGEMM_OK) return rc;
  if (stack == 0 || rows == 0 || K == 0) return NEOGEMM_OK;
  if (Y == nullptr) return NEOGEMM_ERR_BAD_ARG;
  if (!aligned16(Y)) return NEOGEMM_ERR_UNSUPPORTED;
  DeviceView dev;
  rc = acquire_device(&dev);
  if (rc != NEOGEMM_OK) return rc;
  ConvertParams p;
  std::memset(&p, 0, sizeof(p));
  fill(p, stack, rows, K);
  p.codes = static_cast<unsigned char*>(const_cast<void*>(codes));
  p.scales = static_cast<unsigned char*>(const_cast<void*>(scales));
  p.y = static_cast<__nv_bfloat16*>(Y);
  return launch(dev, reinterpret_cast<const void*>(&mxfp4_dequantize_kernel), p,
                static_cast<cudaStream_t>(stream));
}

}  // extern "C"
