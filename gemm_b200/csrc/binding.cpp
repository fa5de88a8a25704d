// PyTorch binding: module `neoGEMM`, function `neoGemmV1(A, B, C)` - the reference's operator
// surface (nemgemmV03.cu:343-398; legacy `neogemm`, neogemmV02.cu:262-306) - on top of the C ABI
// of libneogemm.so.  Only this file sees torch headers; it is compiled by the host compiler.
//
// Differences from the reference binding, all on the safe side:
//   * dtype, device, rank, contiguity and shape agreement are checked (the reference reads raw
//     data_ptr<at::BFloat16>() unchecked, nemgemmV03.cu:349-351);
//   * the launch goes to torch's current stream on A's device (the reference uses the legacy
//     default stream of whatever device is current, nemgemmV03.cu:383);
//   * failures raise RuntimeError (the reference prints to stderr, nemgemmV03.cu:387-390).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <string>
#include <utility>

#include "neogemm.h"

namespace {

void check_matrix(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (there is no CPU path)");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16");
  TORCH_CHECK(t.dim() == 2, name, " must be 2-D");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have contiguous rows");
}

int64_t row_pitch(const torch::Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1);
}

void run(const torch::Tensor& A, const torch::Tensor& B, void* C, int64_t ldc, bool col_major) {
  const int64_t M = A.size(0), K = A.size(1), N = B.size(0);
  c10::cuda::CUDAGuard guard(A.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(A.device().index()).stream();
  const int rc = neogemm_bf16_nt(A.data_ptr(), B.data_ptr(), C, M, N, K, row_pitch(A),
                                 row_pitch(B), ldc, col_major ? 1 : 0, nullptr, 0,
                                 static_cast<void*>(stream));
  TORCH_CHECK(rc == NEOGEMM_OK, "neoGEMM: ", neogemm_status_str(rc));
}

void check_pair(const torch::Tensor& A, const torch::Tensor& B) {
  check_matrix(A, "A");
  check_matrix(B, "B");
  TORCH_CHECK(A.device() == B.device(), "A and B must be on the same device");
  TORCH_CHECK(A.size(1) == B.size(1), "A is [M,K] and B is [N,K]: their K differ");
}

// C <- A * B^T stored column-major in C (element (i,j) at j*M + i), as the reference does.
void neoGemmV1(torch::Tensor A, torch::Tensor B, torch::Tensor C) {
  check_pair(A, B);
  TORCH_CHECK(C.is_cuda() && C.scalar_type() == at::kBFloat16, "C must be a CUDA bfloat16 tensor");
  TORCH_CHECK(C.device() == A.device(), "C must be on the same device as A and B");
  TORCH_CHECK(C.is_contiguous() && C.numel() == A.size(0) * B.size(0),
              "C must be contiguous with M*N elements");
  run(A, B, C.data_ptr(), std::max<int64_t>(A.size(0), 1), true);
}

// Row-major convenience: returns C[M,N].
torch::Tensor matmul(torch::Tensor A, torch::Tensor B) {
  check_pair(A, B);
  auto C = torch::empty({A.size(0), B.size(0)}, A.options());
  run(A, B, C.data_ptr(), std::max<int64_t>(B.size(0), 1), false);
  return C;
}

// ----------------------------------------------------------------------------------------------
// Products grouped by expert, and MXFP4 (gemm_b200.ops documents them).  Here rather than over
// ctypes because they serve single decoding steps: checks, allocation and launch cost the host
// about half.
// ----------------------------------------------------------------------------------------------
// Numbers in messages.  Not through a stream: where the compiler links its C++ library statically, the
// streams' number formatting looks for facets of another copy of the library and crashes.
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}

void check_status(int rc) {
  // Raises gemm_b200._lib.NeoGemmError with the code.
  if (rc != NEOGEMM_OK) pybind11::module_::import("gemm_b200._lib").attr("check")(rc);
}

// A new tensor beside `like`, past the dispatcher (a quantisation, of two: 5.3 -> 4.7 us on the host).
torch::Tensor empty_beside(const torch::Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::detail::empty_cuda(shape, type, like.device(), c10::nullopt);
}

struct Rows {
  int64_t count, width, pitch;
};

// A bf16 matrix with contiguous rows that is read.  A single row's pitch is nobody's to use: it gets
// a legal one.
Rows rows_operand(const torch::Tensor& t, const char* name, const torch::Tensor& first) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must live on a CUDA device (there is no CPU path)");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 2, name, " must be 2-D, got shape ", text(t.sizes()));
  TORCH_CHECK_VALUE(t.get_device() == first.get_device(), name, " must be on ", first.device());
  TORCH_CHECK_VALUE(t.size(1) <= 1 || t.stride(1) == 1, name,
                    " must have unit stride along its last dimension");
  return Rows{t.size(0), t.size(1), t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 8 * 8};
}

// The bytes of a tensor as `count` runs of `width` bytes, `pitch` apart; false if they are not such.
struct Runs {
  intptr_t begin, end;   // first byte, and the one behind the last
  int64_t count, width, pitch;
};

bool runs_of(const torch::Tensor& t, Runs* r) {
  c10::SmallVector<std::pair<int64_t, int64_t>, 4> dims;   // (stride in bytes, size)
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1 && t.stride(d) != 0)
      dims.emplace_back(t.stride(d) * static_cast<int64_t>(t.element_size()), t.size(d));
  std::sort(dims.begin(), dims.end());
  r->begin = r->end = reinterpret_cast<intptr_t>(t.data_ptr());
  r->count = 1;
  r->width = r->pitch = t.element_size();
  r->end += r->width;
  bool simple = true;
  for (const auto& [stride, size] : dims) {
    r->end += stride * (size - 1);
    if (r->count == 1 && stride <= r->width) {
      r->width = stride * (size - 1) + r->width;
    } else if (r->count == 1) {
      r->pitch = stride;
      r->count = size;
    } else if (stride == r->pitch * r->count) {
      r->count *= size;
    } else {
      simple = false;
    }
  }
  return simple;
}

// Whether two tensors have a byte in common: exactly, if the runs of both are equally far apart or one has
// a single run; other views count as sharing when their address ranges do.
bool share_memory(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  Runs x, y;
  const bool simple = runs_of(a, &x) & runs_of(b, &y);
  if (x.end <= y.begin || y.end <= x.begin) return false;
  if (!simple || (x.count > 1 && y.count > 1 && x.pitch != y.pitch)) return true;
  if (x.count == 1 && y.count == 1) return true;
  const int64_t pitch = x.count > 1 ? x.pitch : y.pitch;
  const int64_t apart = ((y.begin - x.begin) % pitch + pitch) % pitch;   // y's run behind x's, in a period
  return apart < x.width || apart + y.width > pitch;
}

// A result is written while the operands are read.
void check_apart(const torch::Tensor& out, const torch::Tensor& operand, const char* name) {
  TORCH_CHECK_VALUE(!share_memory(out, operand), "out must not share memory with ", name);
}

// A caller's tensor has other values now: a graph that saved the earlier ones must not use them.
void note_written(const c10::optional<torch::Tensor>& out) {
  if (out.has_value() && !out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
}

struct Result {
  torch::Tensor tensor;
  int64_t pitch;
  int zero_rest;   // a fresh result is zero in the rows of no group
};

Result rows_result(const c10::optional<torch::Tensor>& out, const torch::Tensor& like, int64_t rows,
                   int64_t width) {
  if (!out.has_value())
    return Result{empty_beside(like, {rows, width}, at::kBFloat16),
                  std::max<int64_t>(width, 1), 1};
  const torch::Tensor& t = *out;
  TORCH_CHECK_VALUE(t.is_cuda(), "out must live on a CUDA device (there is no CPU path)");
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "out must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) == width &&
                        t.get_device() == like.get_device(),
                    "out must be [", text(rows), ",", text(width), "] on ", like.device());
  TORCH_CHECK_VALUE(width <= 1 || t.stride(1) == 1, "out must have unit stride along its last dimension");
  return Result{t, row_pitch(t), 0};
}

int64_t group_count(const torch::Tensor& offsets, const torch::Tensor& like) {
  TORCH_CHECK_TYPE(offsets.scalar_type() == at::kInt || offsets.scalar_type() == at::kLong,
                   "offsets must be int32 or int64, got ", offsets.scalar_type());
  TORCH_CHECK_VALUE(offsets.is_cuda() && offsets.get_device() == like.get_device(),
                    "offsets must be on ", like.device());
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.size(0) >= 1 && offsets.is_contiguous(),
                    "offsets must be a contiguous vector of groups + 1 row indices");
  return offsets.size(0) - 1;
}

void* stream_of(const torch::Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

using RowsFunction = int (*)(const void*, const void*, void*, const void*, int, int64_t, int64_t, int64_t,
                             int64_t, int64_t, int64_t, int64_t, int64_t, int, void*);

torch::Tensor grouped_rows(RowsFunction fn, const char* name, bool transposed, const torch::Tensor& rows,
                           const torch::Tensor& w, const torch::Tensor& offsets,
                           const c10::optional<torch::Tensor>& out) {
  const Rows r = rows_operand(rows, name, rows);
  TORCH_CHECK_TYPE(w.scalar_type() == at::kBFloat16, "w must be bfloat16, got ", w.scalar_type());
  TORCH_CHECK_VALUE(w.dim() == 3, "w must be [groups, N, K], got shape ", text(w.sizes()));
  TORCH_CHECK_VALUE(w.is_cuda() && w.get_device() == rows.get_device(), "w must be on ", rows.device());
  const int64_t N = w.size(1), K = w.size(2);
  TORCH_CHECK_VALUE(K <= 1 || w.stride(2) == 1, "w must have unit stride along its last dimension");
  const int64_t groups = group_count(offsets, rows);
  TORCH_CHECK_VALUE(w.size(0) == groups, "w has ", text(w.size(0)), " matrices but offsets delimit ", text(groups),
                    " groups");
  TORCH_CHECK_VALUE(r.width == (transposed ? N : K), name, " is [", text(r.count), ",", text(r.width),
                    "] but w is [groups,", text(N), ",", text(K), "]: expected rows of ",
                    text(transposed ? N : K));
  TORCH_CHECK_VALUE(groups <= 1 || w.stride(0) > 0 || w.numel() == 0,
                    "w must hold a matrix per group, not one expanded over them");
  c10::cuda::CUDAGuard guard(rows.device());
  Result y = rows_result(out, rows, r.count, transposed ? K : N);
  if (out.has_value()) {
    check_apart(*out, rows, name);
    check_apart(*out, w, "w");
    check_apart(*out, offsets, "offsets");
  }
  check_status(fn(rows.data_ptr(), w.data_ptr(), y.tensor.data_ptr(), offsets.data_ptr(),
                  offsets.scalar_type() == at::kLong, groups, r.count, N, K, r.pitch,
                  N > 1 ? w.stride(1) : (K + 15) / 8 * 8, groups > 1 ? w.stride(0) : 0, y.pitch,
                  y.zero_rest, stream_of(rows)));
  note_written(out);
  return y.tensor;
}

torch::Tensor grouped_matmul(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& offsets,
                             const c10::optional<torch::Tensor>& out) {
  return grouped_rows(&neogemm_grouped_nt, "x", false, x, w, offsets, out);
}

torch::Tensor grouped_matmul_dx(const torch::Tensor& dy, const torch::Tensor& w,
                                const torch::Tensor& offsets, const c10::optional<torch::Tensor>& out) {
  return grouped_rows(&neogemm_grouped_dx, "dy", true, dy, w, offsets, out);
}

torch::Tensor grouped_matmul_dw(const torch::Tensor& dy, const torch::Tensor& x,
                                const torch::Tensor& offsets, const c10::optional<torch::Tensor>& out) {
  const Rows d = rows_operand(dy, "dy", dy), r = rows_operand(x, "x", dy);
  const int64_t groups = group_count(offsets, dy);
  TORCH_CHECK_VALUE(r.count == d.count, "dy has ", text(d.count), " rows but x has ", text(r.count));
  c10::cuda::CUDAGuard guard(dy.device());
  torch::Tensor dw;
  if (out.has_value()) {
    dw = *out;
    TORCH_CHECK_VALUE(dw.scalar_type() == at::kBFloat16 && dw.is_cuda() &&
                          dw.get_device() == dy.get_device() && dw.dim() == 3 && dw.size(0) == groups &&
                          dw.size(1) == d.width && dw.size(2) == r.width && dw.is_contiguous(),
                      "out must be a contiguous bfloat16 [", text(groups), ",", text(d.width), ",",
                      text(r.width), "] on ",
                      dy.device());
    check_apart(dw, dy, "dy");
    check_apart(dw, x, "x");
    check_apart(dw, offsets, "offsets");
  } else {
    dw = empty_beside(dy, {groups, d.width, r.width}, at::kBFloat16);
  }
  check_status(neogemm_grouped_dw(dy.data_ptr(), x.data_ptr(), dw.data_ptr(), offsets.data_ptr(),
                                  offsets.scalar_type() == at::kLong, groups, d.count, d.width, r.width,
                                  d.pitch, r.pitch, stream_of(dy)));
  note_written(out);
  return dw;
}

// [.., ceil(rows/128), ceil(K/128), 32, 4, 4]
c10::SmallVector<int64_t, 6> scales_shape(at::IntArrayRef shape, int64_t K) {
  c10::SmallVector<int64_t, 6> s;
  if (shape.size() == 3) s.push_back(shape[0]);
  s.append({(shape[shape.size() - 2] + 127) / 128, (K + 127) / 128, 32, 4, 4});
  return s;
}

void check_mxfp4(const torch::Tensor& codes, const torch::Tensor& scales, const char* name, int64_t min_dim,
                 int64_t max_dim, const torch::Tensor& first) {
  TORCH_CHECK_VALUE(codes.is_cuda() && scales.is_cuda(), name,
                    " must live on a CUDA device (there is no CPU path)");
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, name,
                   ": codes and scales must be uint8");
  TORCH_CHECK_VALUE(codes.dim() >= min_dim && codes.dim() <= max_dim, name, ": codes of shape ",
                    text(codes.sizes()), " must have ", text(max_dim), min_dim < max_dim ? " dimensions at most" : " dimensions");
  TORCH_CHECK_VALUE(codes.get_device() == first.get_device() && scales.get_device() == first.get_device(),
                    name, ": all operands must be on the same device");
  const auto want = scales_shape(codes.sizes(), 2 * codes.size(-1));
  TORCH_CHECK_VALUE(scales.sizes() == at::IntArrayRef(want), name, ": scales of codes ",
                    text(codes.sizes()), " must be ", text(want), ", got ", text(scales.sizes()));
  TORCH_CHECK_VALUE(codes.is_contiguous() && scales.is_contiguous(), name,
                    ": codes and scales must be contiguous");
}

std::pair<torch::Tensor, torch::Tensor> quantize_mxfp4(const torch::Tensor& x) {
  TORCH_CHECK_VALUE(x.is_cuda(), "x must live on a CUDA device (there is no CPU path)");
  const bool f32 = x.scalar_type() == at::kFloat;
  TORCH_CHECK_TYPE(f32 || x.scalar_type() == at::kBFloat16, "x must be bfloat16 or float32, got ",
                   x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() == 2 || x.dim() == 3, "x must be [rows, K] or [stack, rows, K], got shape ",
                    text(x.sizes()));
  const int64_t rows = x.size(-2), K = x.size(-1), stack = x.dim() == 3 ? x.size(0) : 1;
  TORCH_CHECK_VALUE(K % 32 == 0, "K must be a multiple of 32, got ", text(K));
  TORCH_CHECK_VALUE(K <= 1 || x.stride(-1) == 1, "x must have unit stride along its last dimension");
  c10::cuda::CUDAGuard guard(x.device());
  c10::SmallVector<int64_t, 3> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = K / 2;
  torch::Tensor codes = empty_beside(x, shape, at::kByte);
  torch::Tensor scales = empty_beside(x, scales_shape(x.sizes(), K), at::kByte);
  check_status(neogemm_mxfp4_quantize(x.data_ptr(), f32, codes.data_ptr(), scales.data_ptr(), stack, rows,
                                      K, rows > 1 ? x.stride(-2) : K, stack > 1 ? x.stride(0) : 0,
                                      stream_of(x)));
  return {codes, scales};
}

torch::Tensor dequantize_mxfp4(const torch::Tensor& codes, const torch::Tensor& scales) {
  check_mxfp4(codes, scales, "q", 2, 3, codes);
  c10::cuda::CUDAGuard guard(codes.device());
  c10::SmallVector<int64_t, 3> shape(codes.sizes().begin(), codes.sizes().end());
  shape.back() *= 2;
  torch::Tensor out = empty_beside(codes, shape, at::kBFloat16);
  check_status(neogemm_mxfp4_dequantize(codes.data_ptr(), scales.data_ptr(), out.data_ptr(),
                                        shape.size() == 3 ? shape[0] : 1, shape[shape.size() - 2],
                                        shape.back(), stream_of(codes)));
  return out;
}

torch::Tensor matmul_mxfp4(const torch::Tensor& a, const torch::Tensor& a_scales, const torch::Tensor& b,
                           const torch::Tensor& b_scales, const c10::optional<torch::Tensor>& out) {
  check_mxfp4(a, a_scales, "a", 2, 2, a);
  check_mxfp4(b, b_scales, "b", 2, 2, a);
  const int64_t M = a.size(0), N = b.size(0), K = 2 * a.size(1);
  TORCH_CHECK_VALUE(2 * b.size(1) == K, "a is [M,K]=[", text(M), ",", text(K), "] but b is [N,K]=[",
                    text(N), ",", text(2 * b.size(1)), "]: K differs");
  c10::cuda::CUDAGuard guard(a.device());
  Result c = rows_result(out, a, M, N);
  if (out.has_value())
    for (const torch::Tensor* t : {&a, &a_scales, &b, &b_scales}) check_apart(*out, *t, "an operand");
  check_status(neogemm_mxfp4_nt(a.data_ptr(), a_scales.data_ptr(), b.data_ptr(), b_scales.data_ptr(),
                                c.tensor.data_ptr(), M, N, K, c.pitch, stream_of(a)));
  note_written(out);
  return c.tensor;
}

torch::Tensor grouped_matmul_mxfp4(const torch::Tensor& x, const torch::Tensor& x_scales,
                                   const torch::Tensor& w, const torch::Tensor& w_scales,
                                   const torch::Tensor& offsets, const c10::optional<torch::Tensor>& out) {
  check_mxfp4(x, x_scales, "x", 2, 2, x);
  check_mxfp4(w, w_scales, "w", 3, 3, x);
  const int64_t groups = group_count(offsets, x), T = x.size(0), N = w.size(1), K = 2 * x.size(1);
  TORCH_CHECK_VALUE(w.size(0) == groups, "w has ", text(w.size(0)), " matrices but offsets delimit ", text(groups),
                    " groups");
  TORCH_CHECK_VALUE(2 * w.size(2) == K, "x is [T,K]=[", text(T), ",", text(K), "] but w is [groups,N,K]=[",
                    text(groups), ",", text(N), ",", text(2 * w.size(2)), "]: K differs");
  c10::cuda::CUDAGuard guard(x.device());
  Result y = rows_result(out, x, T, N);
  if (out.has_value())
    for (const torch::Tensor* t : {&x, &x_scales, &w, &w_scales, &offsets}) check_apart(*out, *t, "an operand");
  check_status(neogemm_grouped_mxfp4_nt(x.data_ptr(), x_scales.data_ptr(), w.data_ptr(),
                                        w_scales.data_ptr(), y.tensor.data_ptr(), offsets.data_ptr(),
                                        offsets.scalar_type() == at::kLong, groups, T, N, K, y.pitch,
                                        y.zero_rest, stream_of(x)));
  note_written(out);
  return y.tensor;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "BF16 GEMM C = A * B^T for B200 (sm_100a): TMA + tcgen05 + TMEM";
  m.def("neoGemmV1", &neoGemmV1, "C <- A * B^T, column-major in C (reference-compatible)",
        pybind11::arg("A"), pybind11::arg("B"), pybind11::arg("C"));
  m.def("neogemm", &neoGemmV1, "legacy name of neoGemmV1", pybind11::arg("A"),
        pybind11::arg("B"), pybind11::arg("C"));
  m.def("matmul", &matmul, "returns row-major C[M,N] = A * B^T", pybind11::arg("A"),
        pybind11::arg("B"));
  m.def("_share_memory", &share_memory, "whether two tensors have a byte in common (the check of out=)",
        pybind11::arg("a"), pybind11::arg("b"));
  m.def("grouped_matmul", &grouped_matmul, "gemm_b200.ops.grouped_matmul", pybind11::arg("x"),
        pybind11::arg("w"), pybind11::arg("offsets"), pybind11::arg("out") = pybind11::none());
  m.def("grouped_matmul_dx", &grouped_matmul_dx, "gemm_b200.ops.grouped_matmul_dx", pybind11::arg("dy"),
        pybind11::arg("w"), pybind11::arg("offsets"), pybind11::arg("out") = pybind11::none());
  m.def("grouped_matmul_dw", &grouped_matmul_dw, "gemm_b200.ops.grouped_matmul_dw", pybind11::arg("dy"),
        pybind11::arg("x"), pybind11::arg("offsets"), pybind11::arg("out") = pybind11::none());
  m.def("quantize_mxfp4", &quantize_mxfp4, "gemm_b200.ops.quantize_mxfp4 as (codes, scales)",
        pybind11::arg("x"));
  m.def("dequantize_mxfp4", &dequantize_mxfp4, "gemm_b200.ops.dequantize_mxfp4", pybind11::arg("codes"),
        pybind11::arg("scales"));
  m.def("matmul_mxfp4", &matmul_mxfp4, "gemm_b200.ops.matmul_mxfp4", pybind11::arg("a_codes"),
        pybind11::arg("a_scales"), pybind11::arg("b_codes"), pybind11::arg("b_scales"),
        pybind11::arg("out") = pybind11::none());
  m.def("grouped_matmul_mxfp4", &grouped_matmul_mxfp4, "gemm_b200.ops.grouped_matmul_mxfp4",
        pybind11::arg("x_codes"), pybind11::arg("x_scales"), pybind11::arg("w_codes"),
        pybind11::arg("w_scales"), pybind11::arg("offsets"), pybind11::arg("out") = pybind11::none());
}
