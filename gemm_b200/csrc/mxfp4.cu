// Conversion between bf16 / fp32 and MXFP4 (format and contracts: include/neogemm.h).
//
// Both directions move each value once, which HBM bounds as long as the instructions per value are few
// (straightforward code, about 15 per value, was bound by issue slots at 60 % of the bandwidth): bf16
// stays packed in pairs through maximum and scaling, codes become bf16 by byte permutes of two
// eight-entry tables.  A lane owns 8 consecutive values (16 bytes of bf16) and four lanes a block of
// 32; a warp covers up to 1024 consecutive values of a row.
#include "../../include/neogemm.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <cstring>

#include "host.cuh"
#include "ptx.cuh"

namespace neogemm {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kParts = 4;             // 256 values each
constexpr int kSpan = 256 * kParts;   // values of a row that a warp covers

struct ConvertParams {
  const void* x;
  unsigned char* codes;
  unsigned char* scales;
  __nv_bfloat16* y;
  long long stack, rows, K, ldx, stack_x;
  long long row_blocks, k_tiles;   // 128-row blocks, 128-value tiles
  unsigned spans;                  // warps per row
};

// A warp's place: (row of the padded matrix, span of K); false past the end.
__device__ __forceinline__ bool place(const ConvertParams& p, long long* row, long long* k) {
  const unsigned warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const unsigned r = warp / p.spans;
  *row = r;
  *k = static_cast<long long>(warp - r * p.spans) * kSpan + (threadIdx.x & 31) * 8;
  return r < p.row_blocks * 128;
}

// Byte of this lane's scale in the first 256 values of its span; 1024 bytes further per 256 values.
__device__ __forceinline__ long long scale_at(const ConvertParams& p, long long matrix, long long row,
                                              long long k0) {
  return ((matrix * p.row_blocks + row / 128) * p.k_tiles + k0 / 128) * 512 + (row & 31) * 16 +
         ((row >> 5) & 3) * 4 + ((threadIdx.x >> 2) & 3);
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

// Exponent of the largest magnitude (biased) to the block's biased scale exponent.
__device__ __forceinline__ uint32_t scale_of(uint32_t e) { return e == 255 ? 255u : e > 2 ? e - 2 : 0u; }

template <bool kF32>
__global__ void __launch_bounds__(kThreads) mxfp4_quantize_kernel(const ConvertParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  long long row, k0;
  if (!place(p, &row, &k0)) return;
  const bool in_rows = row < p.rows;
  // Padding: the scales of rows past the last, and of blocks between K and the next 128.
  const long long k_scales = p.k_tiles * 128;
  for (long long m = blockIdx.y; m < p.stack; m += gridDim.y) {
    const long long src = m * p.stack_x + row * p.ldx + k0;
    uint32_t* codes = reinterpret_cast<uint32_t*>(p.codes + ((m * p.rows + row) * p.K + k0) / 2);
    unsigned char* scales = p.scales + scale_at(p, m, row, k0);
    const uint4* x = kF32 ? reinterpret_cast<const uint4*>(static_cast<const float*>(p.x) + src)
                          : reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.x) + src);
    uint4 a[kParts], b[kParts];   // raw bits; b only for fp32
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      a[q] = b[q] = make_uint4(0, 0, 0, 0);
      if (in_rows && k0 + q * 256 < p.K) {   // K is a multiple of 32: blocks are whole
        a[q] = __ldcs(x + q * (kF32 ? 64 : 32));
        if (kF32) b[q] = __ldcs(x + q * 64 + 1);
      }
    }
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      const long long k = k0 + q * 256;
      const bool in = in_rows && k < p.K;
      float v[8];
      uint32_t s;
      // Magnitudes as bits are ordered like the values, with Inf and NaN on top.
      if (kF32) {
        const uint32_t w[8] = {a[q].x, a[q].y, a[q].z, a[q].w, b[q].x, b[q].y, b[q].z, b[q].w};
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, w[j] & 0x7fffffffu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        s = scale_of(top >> 23);
        const float up = __uint_as_float((254 - min(s, 252u)) << 23);   // 2^(127 - s), a normal number
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]) * up;
      } else {
        uint32_t w[4] = {a[q].x, a[q].y, a[q].z, a[q].w};
        uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = max(top >> 16, top & 0xffffu);
        s = scale_of(top >> 7);
        // A power of two: exact, but for values far below the smallest code's half.
        const uint32_t up = (254 - min(s, 252u)) * 0x00800080u;
        __nv_bfloat162 up2;
        memcpy(&up2, &up, 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          __nv_bfloat162 t;
          memcpy(&t, &w[j], 4);
          t = __hmul2(t, up2);
          memcpy(&w[j], &t, 4);
          v[2 * j] = __uint_as_float(w[j] << 16);
          v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
      }
      uint32_t code = e2m1_pair(v[0], v[1]) | e2m1_pair(v[2], v[3]) << 8 | e2m1_pair(v[4], v[5]) << 16 |
                      e2m1_pair(v[6], v[7]) << 24;
      if (s == 255) code = 0;
      if (in) codes[q * 32] = code;
      if ((threadIdx.x & 3) == 0 && k < k_scales)
        scales[q * 1024] = static_cast<unsigned char>(in ? s : 0u);
    }
  }
}

// Four codes in the low 16 bits of `m` (magnitudes, sign bits clear) to the bytes of their bf16.
__device__ __forceinline__ uint32_t high_bytes(uint32_t m) { return __byte_perm(0x3f3f3f00u, 0x40404040u, m); }
__device__ __forceinline__ uint32_t low_bytes(uint32_t m) { return __byte_perm(0xc0800000u, 0xc0804000u, m); }

__global__ void __launch_bounds__(kThreads) mxfp4_dequantize_kernel(const ConvertParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  long long row, k0;
  if (!place(p, &row, &k0) || row >= p.rows) return;
  for (long long m = blockIdx.y; m < p.stack; m += gridDim.y) {
    const long long first = (m * p.rows + row) * p.K + k0;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.codes + first / 2);
    const unsigned char* scales = p.scales + scale_at(p, m, row, k0);
    uint4* out = reinterpret_cast<uint4*>(p.y + first);
    uint32_t code[kParts], scale[kParts];
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      code[q] = scale[q] = 0;
      if (k0 + q * 256 < p.K) {
        code[q] = __ldcs(codes + q * 32);
        scale[q] = scales[q * 1024];
      }
    }
#pragma unroll
    for (int q = 0; q < kParts; ++q) {
      // 2^(s - 127) in bf16, twice; the smallest is half of the smallest normal number.
      const uint32_t s = scale[q];
      const uint32_t bits = s == 255 ? 0x7fc07fc0u : s == 0 ? 0x00400040u : s * 0x00800080u;
      __nv_bfloat162 factor;
      memcpy(&factor, &bits, 4);
      const uint32_t mag = code[q] & 0x77777777u, even = code[q] << 4;
      uint32_t w[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // Sign bits of four codes to the top bits of four bytes: codes 0 and 2 from `even`.
        const uint32_t sign = __byte_perm(even, code[q], h ? 0x7362 : 0x5140) & 0x80808080u;
        const uint32_t hi = high_bytes(mag >> (16 * h)) | sign, lo = low_bytes(mag >> (16 * h));
        w[2 * h] = __byte_perm(lo, hi, 0x5140);
        w[2 * h + 1] = __byte_perm(lo, hi, 0x7362);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __nv_bfloat162 t;
        memcpy(&t, &w[j], 4);
        t = __hmul2(t, factor);
        memcpy(&w[j], &t, 4);
      }
      if (k0 + q * 256 < p.K) out[q * 32] = make_uint4(w[0], w[1], w[2], w[3]);
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
  p.spans = static_cast<unsigned>((K + kSpan - 1) / kSpan);
}

int launch(const void* fn, ConvertParams& p, cudaStream_t stream) {
  const long long warps = p.row_blocks * 128 * p.spans;
  if (warps > 0xffffffffll - kWarps) return NEOGEMM_ERR_UNSUPPORTED;
  const long long x = (warps + kWarps - 1) / kWarps, y = std::min<long long>(p.stack, 65535);
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(x), static_cast<unsigned>(y), 1);
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
  // Extents far past any memory would overflow the products above.
  if (stack > (1ll << 31) || rows > (1ll << 31) || K > (1ll << 31)) return NEOGEMM_ERR_UNSUPPORTED;
  if (stack == 0 || rows == 0 || K == 0) return NEOGEMM_OK;
  if (stack > (1ll << 45) / rows || stack * rows > (1ll << 45) / K) return NEOGEMM_ERR_UNSUPPORTED;
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
  const int64_t step = x_is_f32 ? 4 : 8;   // elements in 16 bytes
  if (ldx > 1ll << 45 || stack_x > 1ll << 45) return NEOGEMM_ERR_UNSUPPORTED;
  if (!aligned16(X) || (rows > 1 && ldx % step != 0) || (stack > 1 && stack_x % step != 0))
    return NEOGEMM_ERR_UNSUPPORTED;
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
  return launch(fn, p, static_cast<cudaStream_t>(stream));
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
  return launch(reinterpret_cast<const void*>(&mxfp4_dequantize_kernel), p,
                static_cast<cudaStream_t>(stream));
}

}  // extern "C"
