// Tensor checks, output allocation and error translation of the router and the block-128 operators (mx8/router.py, mx8/block128.py):
// part of the `_C` module, on top of the C ABI like the rest of it.  A bad tensor raises ValueError, a status of the C ABI Mx8Error.
// It is C++ because the smallest calls are bound by the host: one decoding step of the router allocates seven outputs; it takes
// 7.2 us here (5 us of them on the GPU), 26 us as a Python function over ctypes.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <climits>
#include <optional>
#include <string>

#include "../../include/mx8.h"

namespace py = pybind11;
using OptTensor = std::optional<at::Tensor>;

namespace {

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

void check(int rc, const char* where) {
    if (rc == MX8_OK) return;
    const py::object cls = py::module_::import("mx8._lib").attr("Mx8Error");
    PyErr_SetObject(cls.ptr(), cls(rc, where).ptr());
    throw py::error_already_set();
}

void* stream() { return static_cast<void*>(c10::cuda::getCurrentCUDAStream().stream()); }

std::string shape_of(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

at::Device cuda_device(const at::Tensor& t, const char* name) {
    if (!t.defined() || !t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
    return t.device();
}

bool one_of(at::ScalarType t, at::ScalarType a, at::ScalarType b) { return t == a || t == b; }
constexpr auto FP8 = at::kFloat8_e4m3fn, U8 = at::kByte, F32 = at::kFloat, BF16 = at::kBFloat16, I32 = at::kInt;

int dim(int64_t n, const char* name) {
    if (n <= 0 || n > INT_MAX) refuse(std::string(name) + " must be between 1 and 2^31 - 1, got " + std::to_string(n));
    return static_cast<int>(n);
}

// past the dispatcher: half the time of at::empty
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device dev) { return at::detail::empty_cuda(shape, type, dev, std::nullopt); }

// a tensor inside an allocation, from its `first`-th element on (past the dispatcher too)
at::Tensor part_of(const at::Tensor& whole, int64_t first, at::IntArrayRef shape, at::IntArrayRef strides, at::ScalarType type) {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_and_strides(shape, strides, first);
    return t;
}

int64_t cdiv(int64_t n) { return (n + 127) / 128; }
int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }

// a tensor [.., rows, cols] whose columns are contiguous and whose matrices lie back to back: pointer and row pitch
struct Matrix {
    void* p = nullptr;
    long long pitch = 0;
};
Matrix matrix(const at::Tensor& t, const char* name, at::ScalarType a, at::ScalarType b, at::IntArrayRef shape, at::Device dev) {
    if (!t.defined() || t.device() != dev) refuse(std::string(name) + " must be a tensor on " + dev.str());
    if (!one_of(t.scalar_type(), a, b)) refuse(std::string(name) + " has dtype " + toString(t.scalar_type()) + ", expected " + toString(a) + " or " + toString(b));
    if (t.sizes() != shape) refuse(std::string(name) + " has shape " + shape_of(t.sizes()) + ", expected " + shape_of(shape));
    const int64_t n = t.dim(), rows = shape[n - 2], cols = shape[n - 1];
    if (cols > 1 && t.stride(n - 1) != 1) refuse(std::string(name) + " must have contiguous rows");
    // the stride of a dimension of size one says nothing: a single row may be taken to have any pitch
    int64_t pitch = rows > 1 ? t.stride(n - 2) : n == 3 && shape[0] > 1 ? t.stride(0) : pad16(cols);
    if (n == 3 && shape[0] > 1 && t.stride(0) != rows * pitch) refuse(std::string(name) + ": the matrices must lie back to back");
    return {t.data_ptr(), pitch};
}

void* vec(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, at::Device dev) {
    if (!t.defined() || t.device() != dev) refuse(std::string(name) + " must be a tensor on " + dev.str());
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous())
        refuse(std::string(name) + " must be contiguous " + toString(type) + " " + shape_of(shape) + ", got " + toString(t.scalar_type()) + " " + shape_of(t.sizes()));
    return t.data_ptr();
}
void* vec(const OptTensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, at::Device dev) {
    return t ? vec(*t, name, type, shape, dev) : nullptr;
}

// ------------------------------------------------------------------ router
struct Logits {
    int T, E, type;
    long long ld;
    at::Device dev;
};
Logits logits_of(const at::Tensor& l) {
    const at::Device dev = cuda_device(l, "logits");
    if (!one_of(l.scalar_type(), BF16, F32)) refuse(std::string("logits have dtype ") + toString(l.scalar_type()) + ", expected bfloat16 or float32");
    if (l.dim() != 2 || l.numel() == 0) refuse("logits must be [tokens, experts] and not empty");
    const int T = dim(l.size(0), "tokens"), E = dim(l.size(1), "experts");
    if (E > 1 && l.stride(1) != 1) refuse("logits must have contiguous rows");
    return {T, E, l.scalar_type() == F32 ? MX8_T_F32 : MX8_T_BF16, T > 1 ? l.stride(0) : static_cast<long long>(E), dev};
}

py::tuple router_topk(const at::Tensor& logits, int64_t topk, bool normalize, const OptTensor& token_mask) {
    const Logits l = logits_of(logits);
    c10::cuda::CUDAGuard guard(l.dev);
    const void* mask = vec(token_mask, "token_mask", at::kBool, {l.T}, l.dev);
    const int k = topk < INT_MIN ? INT_MIN : topk > INT_MAX ? INT_MAX : static_cast<int>(topk);
    const int64_t width = k < 1 || k > l.E || k > 32 ? 1 : k;                  // refused below
    // the few words for the experts, and in small calls all outputs, come from one allocation of each type (an allocation is 0.6 us of the
    // host's), each starting where an allocation of its own could.  Not from one for both types: torch.save refuses tensors of different
    // types on one storage.
    const auto up = [](int64_t n) { return (n + 127) / 128 * 128; };
    const int64_t pairs = l.T * width;
    const bool small = 2 * up(pairs) + up(l.T) <= 16384;
    struct Words {
        at::Tensor all;
        at::ScalarType type;
        int64_t next = 0;
    };
    Words ints{empty({up(l.E) + 128 + (small ? up(pairs) : 0)}, I32, l.dev), I32}, floats{empty({up(l.E) + 128 + (small ? up(pairs) + up(l.T) : 0)}, F32, l.dev), F32};
    const auto vector = [&](Words& w, int64_t n) {
        w.next += up(n);
        return part_of(w.all, w.next - up(n), {n}, {1}, w.type);
    };
    const auto matrix = [&](Words& w) {                                        // [T, width]
        w.next += up(pairs);
        return part_of(w.all, w.next - up(pairs), {l.T, width}, {width, 1}, w.type);
    };
    at::Tensor counts = vector(ints, l.E), prob_sum = vector(floats, l.E), num_valid = vector(ints, 1), loss = vector(floats, 1);
    at::Tensor idx = small ? matrix(ints) : empty({l.T, width}, I32, l.dev), weights = small ? matrix(floats) : empty({l.T, width}, F32, l.dev),
               lse = small ? vector(floats, l.T) : empty({l.T}, F32, l.dev), ws;
    const size_t need = mx8_router_topk_workspace_bytes(l.T, l.E);
    if (need) ws = empty({static_cast<int64_t>(need)}, U8, l.dev);
    check(mx8_router_topk(logits.data_ptr(), l.type, l.ld, l.T, l.E, k, normalize, mask, idx.data_ptr(), weights.data_ptr(), lse.data_ptr(),
                          counts.data_ptr(), prob_sum.data_ptr(), num_valid.data_ptr(), loss.data_ptr(), need ? ws.data_ptr() : nullptr, need, stream()),
          "router_topk");
    return py::make_tuple(idx, weights, lse, counts, prob_sum, num_valid, loss);
}

at::Tensor router_topk_bwd(const at::Tensor& logits, const at::Tensor& topk_idx, const at::Tensor& topk_weights, const at::Tensor& lse,
                           const at::Tensor& counts, const at::Tensor& num_valid, const OptTensor& d_topk_weights, const OptTensor& d_balance_loss,
                           bool normalize) {
    const Logits l = logits_of(logits);
    if (topk_idx.dim() != 2) refuse("topk_idx must be [tokens, topk]");
    if (!d_topk_weights && !d_balance_loss) refuse("one of d_topk_weights and d_balance_loss must be given");
    c10::cuda::CUDAGuard guard(l.dev);
    const int k = dim(topk_idx.size(1), "topk");
    const void *ip = vec(topk_idx, "topk_idx", I32, {l.T, k}, l.dev), *wp = vec(topk_weights, "topk_weights", F32, {l.T, k}, l.dev),
               *lp = vec(lse, "lse", F32, {l.T}, l.dev), *cp = vec(counts, "counts", I32, {l.E}, l.dev), *np = vec(num_valid, "num_valid", I32, {1}, l.dev),
               *dw = vec(d_topk_weights, "d_topk_weights", F32, {l.T, k}, l.dev), *dl = vec(d_balance_loss, "d_balance_loss", F32, {1}, l.dev);
    at::Tensor d = empty({l.T, l.E}, logits.scalar_type(), l.dev);
    check(mx8_router_topk_bwd(logits.data_ptr(), l.type, l.ld, l.T, l.E, k, normalize, ip, wp, lp, cp, np, dw, dl, d.data_ptr(), stream()), "router_topk_bwd");
    return d;
}

at::Tensor bwd_topk_weights(const at::Tensor& d_output, const at::Tensor& combine_buffer, const OptTensor& topk_idx) {
    const at::Device dev = cuda_device(d_output, "d_output");
    if (d_output.dim() != 2 || combine_buffer.dim() != 2 || d_output.numel() == 0 || combine_buffer.numel() == 0 ||
        combine_buffer.size(0) % d_output.size(0))
        refuse("d_output is [T, H], combine_buffer [T * topk, H], neither empty");
    c10::cuda::CUDAGuard guard(dev);
    const int T = dim(d_output.size(0), "tokens"), H = dim(d_output.size(1), "hidden"), k = dim(combine_buffer.size(0) / T, "topk");
    const void *gp = vec(d_output, "d_output", BF16, {T, H}, dev), *cp = vec(combine_buffer, "combine_buffer", BF16, {static_cast<int64_t>(T) * k, H}, dev),
               *ip = vec(topk_idx, "topk_idx", I32, {T, k}, dev);
    at::Tensor out = empty({T, k}, F32, dev);
    check(mx8_moe_bwd_topk_weights(gp, cp, ip, out.data_ptr(), T, H, k, stream()), "bwd_topk_weights");
    return out;
}

// ------------------------------------------------------------------ block-128 format
// [.., rows, cols] E4M3 whose rows start on 16-byte boundaries
at::Tensor bytes_out(at::Device dev, bool batched, int64_t E, int64_t rows, int64_t cols) {
    const int64_t pitch = pad16(cols);
    at::Tensor t = batched ? empty({E, rows, pitch}, FP8, dev) : empty({rows, pitch}, FP8, dev);
    if (pitch == cols) return t;
    return batched ? part_of(t, 0, {E, rows, cols}, {rows * pitch, pitch, 1}, FP8) : part_of(t, 0, {rows, cols}, {pitch, 1}, FP8);
}

py::tuple quantize_block128(const at::Tensor& x, bool normal, bool transposed, bool square, const OptTensor& row_index) {
    const at::Device dev = cuda_device(x, "x");
    if ((x.dim() != 2 && x.dim() != 3) || x.numel() == 0) refuse("x must be [M, N] or [E, M, N] and not empty");
    if (!normal && !transposed) refuse("at least one of return_normal / return_transposed must be set");
    const bool batched = x.dim() == 3;
    const Matrix xm = matrix(x, "x", BF16, F32, x.sizes(), dev);
    const int E = batched ? dim(x.size(0), "E") : 1, N = dim(x.size(-1), "N"), src = dim(x.size(-2), "M");
    int M = src;
    const void* ip = nullptr;
    if (row_index) {
        if (batched || square) refuse("row_index takes a 2-D x and row blocks");
        if (row_index->dim() != 1) refuse("row_index must be a vector");
        M = dim(row_index->size(0), "rows of row_index");
        ip = vec(*row_index, "row_index", I32, {M}, dev);
    }
    c10::cuda::CUDAGuard guard(dev);
    auto scales = [&](int64_t a, int64_t b) { return batched ? empty({E, a, b}, F32, dev) : empty({a, b}, F32, dev); };
    py::object none = py::none(), o[4] = {none, none, none, none};
    void *q = nullptr, *sc = nullptr, *qt = nullptr, *sct = nullptr;
    if (normal) {
        const at::Tensor t = bytes_out(dev, batched, E, M, N), s = square ? scales(cdiv(M), cdiv(N)) : scales(cdiv(N), M);
        q = t.data_ptr();
        sc = s.data_ptr();
        o[0] = py::cast(t);
        o[1] = py::cast(s);
    }
    if (transposed) {
        const at::Tensor t = bytes_out(dev, batched, E, N, M), s = square ? scales(cdiv(N), cdiv(M)) : scales(cdiv(M), N);
        qt = t.data_ptr();
        sct = s.data_ptr();
        o[2] = py::cast(t);
        o[3] = py::cast(s);
    }
    check(mx8_quantize_block128(xm.p, x.scalar_type() == F32 ? MX8_T_F32 : MX8_T_BF16, E, M, N, xm.pitch, ip, src, q, pad16(N), sc, qt, pad16(M), sct, square, stream()),
          "quantize_block128");
    return py::make_tuple(o[0], o[1], o[2], o[3]);
}

Matrix row_scales(const at::Tensor& t, const char* name, int64_t blocks, int64_t rows, at::Device dev) {
    Matrix m = matrix(t, name, F32, F32, {blocks, rows}, dev);
    if (m.pitch < rows) m.pitch = rows;
    return m;
}

void* groups_of(const at::Tensor& g, int& n, at::Device dev) {
    if (g.dim() != 1) refuse("group_rows must be a vector");
    n = dim(g.size(0), "groups");
    return vec(g, "group_rows", I32, {n}, dev);
}

at::Tensor gemm_block128(const at::Tensor& A, const at::Tensor& A_sc, const at::Tensor& B, const at::Tensor& B_sc, const at::Tensor& C,
                         const std::string& b_blocks, const OptTensor& group_rows) {
    const at::Device dev = cuda_device(A, "A");
    const bool square = b_blocks == "square";
    if (!square && b_blocks != "rows") refuse("b_blocks is \"square\" or \"rows\"");
    if (A.dim() != 2 || B.dim() != (group_rows ? 3 : 2)) refuse("A is [M, K]; B is [N, K], or [G, N, K] with group_rows");
    if (group_rows && !square) refuse("grouped weights have square blocks");
    const int M = dim(A.size(0), "M"), K = dim(A.size(1), "K"), N = dim(B.size(-2), "N");
    int G = 0;
    const void* gp = group_rows ? groups_of(*group_rows, G, dev) : nullptr;
    const Matrix a = matrix(A, "A", FP8, U8, {M, K}, dev), as = row_scales(A_sc, "A_sc", cdiv(K), M, dev), c = matrix(C, "C", BF16, F32, {M, N}, dev);
    const Matrix b = G ? matrix(B, "B", FP8, U8, {G, N, K}, dev) : matrix(B, "B", FP8, U8, {N, K}, dev);
    Matrix bs;
    if (square) {
        bs.p = G ? vec(B_sc, "B_sc", F32, {G, cdiv(N), cdiv(K)}, dev) : vec(B_sc, "B_sc", F32, {cdiv(N), cdiv(K)}, dev);
    } else {
        bs = row_scales(B_sc, "B_sc", cdiv(K), N, dev);
    }
    c10::cuda::CUDAGuard guard(dev);
    check(mx8_gemm_block128(a.p, a.pitch, as.p, as.pitch, b.p, b.pitch, bs.p, bs.pitch, square, c.p, c.pitch, M, N, K,
                            C.scalar_type() == F32 ? MX8_C_F32 : MX8_C_BF16, gp, G, stream()),
          "gemm_block128");
    return C;
}

at::Tensor gemm_block128_wgrad(const at::Tensor& A, const at::Tensor& A_sc, const at::Tensor& B, const at::Tensor& B_sc, const at::Tensor& C,
                               const at::Tensor& group_rows) {
    const at::Device dev = cuda_device(A, "A_t");
    if (A.dim() != 2 || B.dim() != 2) refuse("A_t is [M, R], B_t is [N, R]");
    const int M = dim(A.size(0), "M"), R = dim(A.size(1), "rows"), N = dim(B.size(0), "N");
    int G = 0;
    const void* gp = groups_of(group_rows, G, dev);
    const Matrix a = matrix(A, "A_t", FP8, U8, {M, R}, dev), b = matrix(B, "B_t", FP8, U8, {N, R}, dev), c = matrix(C, "C", BF16, F32, {G, M, N}, dev);
    const Matrix as = row_scales(A_sc, "A_t_sc", cdiv(R), M, dev), bs = row_scales(B_sc, "B_t_sc", cdiv(R), N, dev);
    c10::cuda::CUDAGuard guard(dev);
    check(mx8_gemm_block128_wgrad(a.p, a.pitch, as.p, as.pitch, b.p, b.pitch, bs.p, bs.pitch, c.p, c.pitch, M, N, R,
                                  C.scalar_type() == F32 ? MX8_C_F32 : MX8_C_BF16, gp, G, stream()),
          "gemm_block128_wgrad");
    return C;
}

}  // namespace

void bind_block128_router(py::module_& m) {
    m.def("router_topk", &router_topk, "", py::arg("logits"), py::arg("topk"), py::arg("normalize") = true, py::arg("token_mask") = std::nullopt);
    m.def("router_topk_bwd", &router_topk_bwd, "", py::arg("logits"), py::arg("topk_idx"), py::arg("topk_weights"), py::arg("lse"), py::arg("counts"),
          py::arg("num_valid"), py::arg("d_topk_weights") = std::nullopt, py::arg("d_balance_loss") = std::nullopt, py::arg("normalize") = true);
    m.def("bwd_topk_weights", &bwd_topk_weights, "", py::arg("d_output"), py::arg("combine_buffer"), py::arg("topk_idx") = std::nullopt);
    m.def("quantize_block128", &quantize_block128, "", py::arg("x"), py::arg("return_normal") = true, py::arg("return_transposed") = false,
          py::arg("square") = false, py::arg("row_index") = std::nullopt);
    m.def("gemm_block128", &gemm_block128, "", py::arg("A"), py::arg("A_sc"), py::arg("B"), py::arg("B_sc"), py::arg("C"), py::arg("b_blocks") = "square",
          py::arg("group_rows") = std::nullopt);
    m.def("gemm_block128_wgrad", &gemm_block128_wgrad, "", py::arg("A_t"), py::arg("A_t_sc"), py::arg("B_t"), py::arg("B_t_sc"), py::arg("C"),
          py::arg("group_rows"));
}
