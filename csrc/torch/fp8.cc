// 8-bit products of the torch binding: quantisation by blocks of 128 and the block-scaled product.
#include "common.h"

namespace mccl_torch {
namespace {

constexpr int64_t kBlock = 128;

int64_t blocksOf(int64_t n) { return (n + kBlock - 1) / kBlock; }

// Scales as bytes, a row's blocks adjacent and rows a multiple of four bytes apart.
Tensor scaleStore(at::IntArrayRef sizes, const Tensor& like) {
  std::vector<int64_t> padded(sizes.begin(), sizes.end());
  padded.back() = (padded.back() + 3) / 4 * 4;
  return at::empty(padded, like.options().dtype(at::kByte)).narrow(-1, 0, sizes.back());
}
Tensor scaleRows(const Tensor& s) {
  Tensor b = s.view(at::kByte);
  const int64_t d = b.dim(), pitch = b.stride(d - 2);
  const bool fits = b.stride(d - 1) == 1 && pitch >= b.size(d - 1) && pitch % 4 == 0 && (reinterpret_cast<uintptr_t>(b.data_ptr()) & 3u) == 0 &&
                    (d < 3 || b.stride(0) == pitch * b.size(1));
  if (fits) return b;
  return scaleStore(b.sizes(), b).copy_(b);
}

// Weights as the kernels take them: rows at 16-byte boundaries, those of all experts one pitch apart.
Tensor weightRows(const Tensor& w) {
  const int64_t d = w.dim(), pitch = w.stride(d - 2);
  if (w.stride(d - 1) == 1 && pitch >= w.size(d - 1) && pitch % 16 == 0 && aligned16(w) && (d < 3 || w.size(0) == 1 || w.stride(0) == pitch * w.size(1))) return w;
  return whole(w);
}

struct Quantized { Tensor data, scale; };       // scale: bytes

Quantized quantizedLike(const Tensor& x) {
  const int64_t M = x.size(0), K = x.size(1);
  return {at::empty({M, K}, x.options().dtype(at::kFloat8_e4m3fn)), scaleStore({M, blocksOf(K)}, x)};
}

// e4m3 values and e8m0 scales of bf16 x: [M, K] by blocks of 128 of a row, or (tiles) [.., N, K] by 128 x 128.
std::pair<Tensor, Tensor> fp8Quantize(const Tensor& xIn, bool tiles) {
  TORCH_CHECK(!recorded() && ordinary(xIn), "fp8_quantize: not under tracing, a dispatch mode or torch.func");
  Below below;
  c10::cuda::CUDAGuard guard(xIn.device());
  if (!tiles) {
    Tensor x = alignedRows(xIn);
    Quantized r = quantizedLike(x);
    check(mcclFp8QuantizeRows(x.data_ptr(), pitchOf(x), r.data.data_ptr(), x.size(1), r.scale.data_ptr(), r.scale.stride(0), x.size(0),
                              (int)x.size(1), streamOf(x)),
          "mcclFp8QuantizeRows");
    counters().gemm += x.size(0) > 0;
    return {r.data, r.scale.view(at::kFloat8_e8m0fnu)};
  }
  Tensor x = whole(xIn);
  const int64_t K = x.size(-1), N = x.size(-2), outer = x.dim() == 3 ? x.size(0) : 1;
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes[sizes.size() - 2] = blocksOf(N);
  sizes.back() = blocksOf(K);
  // Weights are laid out once: rows begin at whole lines, as in fp8Gemm below.
  std::vector<int64_t> store = x.sizes().vec();
  store.back() = blocksOf(K) * kBlock;
  Tensor q = at::empty(store, x.options().dtype(at::kFloat8_e4m3fn)).narrow(-1, 0, K), s = scaleStore(sizes, x);
  check(mcclFp8QuantizeTiles(x.data_ptr(), q.data_ptr(), q.stride(-2), s.data_ptr(), s.stride(-2), outer, (int)N, (int)K, streamOf(x)), "mcclFp8QuantizeTiles");
  counters().gemm++;
  return {q, s.view(at::kFloat8_e8m0fnu)};
}

// x: bf16, quantised here, or e4m3 with its scales.  None where an argument is not what the kernels take (the caller says which).
py::object fp8Gemm(const Tensor& x, const std::optional<Tensor>& xScale, const Tensor& wIn, const Tensor& wScale, const std::optional<Tensor>& ends) {
  constexpr int64_t kMost = INT32_MAX - 256;
  const int64_t wd = ends ? 3 : 2;
  if (recorded() || !ordinary(x) || !ordinary(wIn) || !ordinary(wScale) || !x.is_cuda() || x.dim() != 2 || wIn.dim() != wd || wScale.dim() != wd ||
      wIn.size(wd - 1) != x.size(1)) return py::none();
  const int64_t n = wIn.size(wd - 2), k = x.size(1);
  if (n < 1 || n % 8 || k < 1 || k % 16 || x.size(0) >= kMost || n >= kMost || k >= kMost || wIn.scalar_type() != at::kFloat8_e4m3fn ||
      wScale.scalar_type() != at::kFloat8_e8m0fnu || wScale.size(wd - 2) != blocksOf(n) || wScale.size(wd - 1) != blocksOf(k) || wIn.device() != x.device() ||
      wScale.device() != x.device()) return py::none();
  if (ends && (!ordinary(*ends) || (ends->scalar_type() != at::kInt && ends->scalar_type() != at::kLong) || ends->dim() != 1 || !ends->is_contiguous() ||
               ends->size(0) != wIn.size(0) || wScale.size(0) != wIn.size(0) || wIn.size(0) < 1 || wIn.size(0) > mcclGroupedGemmMaxGroups() ||
               ends->device() != x.device())) return py::none();
  if (xScale ? !ordinary(*xScale) || x.scalar_type() != at::kFloat8_e4m3fn || xScale->scalar_type() != at::kFloat8_e8m0fnu || xScale->dim() != 2 ||
                   xScale->size(0) != x.size(0) || xScale->size(1) != blocksOf(k) || xScale->device() != x.device()
             : x.scalar_type() != at::kBFloat16) return py::none();
  if (at::GradMode::is_enabled() && x.requires_grad()) return py::none();
  Below below;
  c10::cuda::CUDAGuard guard(x.device());
  Tensor rows = alignedRows(x), w = weightRows(wIn), ws = scaleRows(wScale);
  const int64_t M = x.size(0), K = x.size(1), N = w.size(-2), E = w.dim() == 3 ? w.size(0) : 1;
  Tensor y = at::empty({M, N}, x.options().dtype(at::kBFloat16));
  const void* e = ends ? ends->data_ptr() : nullptr;
  const int wide = ends && ends->scalar_type() == at::kLong;
  if (xScale) {
    Tensor xs = scaleRows(*xScale);
    checkProduct(mcclFp8Gemm(rows.data_ptr(), pitchOf(rows), xs.data_ptr(), xs.stride(0), w.data_ptr(), w.stride(-2), ws.data_ptr(), ws.stride(-2), y.data_ptr(), e, wide, (int)E, M,
                      (int)N, (int)K, streamOf(x)), "mcclFp8Gemm");
  } else {
    // One buffer for the quantised rows and, behind them, their scales.  Rows begin at whole lines: a tile's rows of 128 bytes that lie
    // across two lines take about twice as long to load (5003 rows of 2064 through 16 experts of 5504: 104 -> 93 us;
    // with the weights laid out so, too, 82 us).
    const int64_t pitch = blocksOf(K) * kBlock, ld = (blocksOf(K) + 3) / 4 * 4;
    Tensor work = at::empty({M * (pitch + ld)}, x.options().dtype(at::kByte));
    char* q = static_cast<char*>(work.data_ptr());
    checkProduct(mcclFp8GemmBf16Rows(rows.data_ptr(), pitchOf(rows), q, pitch, q + M * pitch, ld, w.data_ptr(), w.stride(-2), ws.data_ptr(), ws.stride(-2), y.data_ptr(), e, wide, (int)E, M,
                              (int)N, (int)K, streamOf(x)), "mcclFp8GemmBf16Rows");
    counters().gemm += M > 0;
  }
  counters().gemm += M > 0;
  return py::cast(y);
}

}  // namespace

void bindFp8(py::module_& m) {
  m.def("fp8_quantize", &fp8Quantize);
  m.def("fp8_gemm", &fp8Gemm);
}

}  // namespace mccl_torch
