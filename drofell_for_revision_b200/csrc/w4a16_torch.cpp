// Torch-facing fast path of the quantized linear's forward: one C++ call that takes the
// activation tensor, allocates the output from torch's caching allocator and calls
// w4a16_gemm on torch's current stream. The same call through ctypes costs several
// microseconds of Python argument checking and conversion per projection, which at
// decode sizes is as long as the kernel itself (the reference binds its extension with
// pybind11 for the same reason, After-Revision-DROFELL/cuda_extends/exllama/entry.cpp:
// 221-251,601-623).
//
// Workspaces (act-order X gather, split-K partials) are per handle, grown on demand and
// never freed before w4a16_torch_release: a CUDA graph captured with one still writes
// into it on replay.
#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/drofell_w4a16.h"

namespace {

struct Workspaces {
    at::Tensor current;
    std::vector<at::Tensor> retired;  // outgrown, kept alive for graphs that captured them
};

std::mutex g_mu;
std::unordered_map<uintptr_t, Workspaces> g_ws;

void check(int rc) {
    if (rc != W4A16_OK) TORCH_CHECK(false, "[w4a16 error ", rc, "] ", w4a16_last_error());
}

int dtype_of(const at::Tensor& x) {
    const int dtype = x.scalar_type() == at::kHalf       ? W4A16_DTYPE_FP16
                      : x.scalar_type() == at::kBFloat16 ? W4A16_DTYPE_BF16
                                                         : -1;
    TORCH_CHECK(dtype >= 0, "x must be float16 or bfloat16");
    return dtype;
}

// The handle's workspace of at least `need` bytes on x's device (nullptr for 0), grown
// by doubling; an outgrown one stays alive for the graphs that captured it.
void* workspace(uintptr_t handle, size_t need, const at::Tensor& x, size_t* bytes) {
    *bytes = 0;
    if (need == 0) return nullptr;
    std::lock_guard<std::mutex> lock(g_mu);
    Workspaces& w = g_ws[handle];
    if (!w.current.defined() || static_cast<size_t>(w.current.numel()) < need) {
        const int64_t size = w.current.defined() ? std::max<int64_t>(need, 2 * w.current.numel()) : need;
        if (w.current.defined()) w.retired.push_back(w.current);
        w.current = at::empty({size}, x.options().dtype(at::kByte));
    }
    *bytes = static_cast<size_t>(w.current.numel());
    return w.current.data_ptr();
}

// Y[..., N] = X[..., K] W (+ bias): the forward of QuantLinear for any M on PATH_AUTO.
at::Tensor linear(uintptr_t handle, const at::Tensor& x, const c10::optional<at::Tensor>& bias) {
    auto* h = reinterpret_cast<w4a16_matrix*>(handle);
    TORCH_CHECK(h != nullptr, "released q4 handle");
    int info[4];
    check(w4a16_info(h, info));
    const int64_t K = info[0], N = info[1];
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor (no CPU path exists)");
    TORCH_CHECK(x.size(-1) == K, "x and w have incompatible shapes");
    const int dtype = dtype_of(x);
    const at::Tensor x2 = x.reshape({-1, K}).contiguous();
    const int64_t M = x2.size(0);
    std::vector<int64_t> out_shape(x.sizes().begin(), x.sizes().end());
    out_shape.back() = N;
    at::Tensor out = at::empty(out_shape, x.options());
    if (M == 0) return out;
    const c10::cuda::CUDAGuard guard(x.device());
    size_t ws_bytes = 0;
    void* ws_ptr = workspace(handle, w4a16_workspace_size(h, static_cast<int>(M), dtype, W4A16_PATH_AUTO), x,
                             &ws_bytes);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    check(w4a16_gemm(h, x2.data_ptr(), static_cast<int>(M), out.data_ptr(), dtype, ws_ptr, ws_bytes,
                     W4A16_PATH_AUTO, stream));
    if (bias.has_value() && bias->defined()) out.add_(*bias);
    return out;
}

// The fused all-gather forward of a column-sharded linear: this rank's columns of
// X[M, K] W into columns [col0, col0 + N) of every rank's full Y[M, ld]
// (w4a16_gemm_gather). y_all is the address of a host array of the world's Y pointers
// that the caller keeps alive (built once per output buffer), so a call converts no
// Python objects besides x.
void gemm_gather(uintptr_t handle, uintptr_t comm, const at::Tensor& x, uintptr_t y_all, int64_t ld, int64_t col0) {
    auto* h = reinterpret_cast<w4a16_matrix*>(handle);
    TORCH_CHECK(h != nullptr, "released q4 handle");
    TORCH_CHECK(comm != 0 && y_all != 0, "the gather needs a comm and the ranks' Y pointers");
    int info[4];
    check(w4a16_info(h, info));
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) == info[0] && x.is_contiguous(),
                "x must be a contiguous CUDA [M, K] tensor");
    const int dtype = dtype_of(x);
    const int M = static_cast<int>(x.size(0));
    if (M == 0) return;
    const c10::cuda::CUDAGuard guard(x.device());
    size_t ws_bytes = 0;
    void* ws_ptr = workspace(handle, w4a16_workspace_size(h, M, dtype, W4A16_PATH_AUTO), x, &ws_bytes);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    check(w4a16_gemm_gather(h, reinterpret_cast<w4a16_comm*>(comm), x.data_ptr(), M,
                            reinterpret_cast<void* const*>(y_all), static_cast<int>(ld), static_cast<int>(col0),
                            dtype, ws_ptr, ws_bytes, stream));
}

// Drop a handle's workspaces (call before w4a16_destroy; graphs that used them must be
// released first).
void release(uintptr_t handle) {
    std::lock_guard<std::mutex> lock(g_mu);
    g_ws.erase(handle);
}

// ---------------------------------------------------------------- paged key-value cache
// Tensor checks common to append_kv and attention; shapes and types come before devices, so
// that they can be told apart without a GPU.
struct Paged {
    w4a16_pages pages;
    w4a16_seqs seqs;
};

void no_grad(const at::Tensor& t, const char* name) {
    TORCH_CHECK(!(c10::GradMode::is_enabled() && t.requires_grad()), name,
                " requires a gradient: the paged cache is for serving and has none (use torch.no_grad())");
}

void on_device(const at::Tensor& t, const at::Tensor& pages, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (no CPU path exists)");
    TORCH_CHECK(t.device() == pages.device(), name, " is on ", t.device(), ", the pages on ", pages.device());
}

void check_ints(const at::Tensor& t, int64_t dim, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim, name, " must be an int32 tensor of ", dim, " dimension(s)");
    TORCH_CHECK(t.size(dim - 1) <= 1 || t.stride(dim - 1) == 1, name, "'s last dimension must be contiguous");
}

w4a16_rows rows_of(const at::Tensor& t, const at::Tensor& pages, int64_t tokens, int64_t heads, const char* name) {
    TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == pages.size(3), name,
                " must be [", tokens, ", ", heads, ", ", pages.size(3), "], got ", t.sizes());
    TORCH_CHECK(t.scalar_type() == pages.scalar_type(), name, " must have the pages' type");
    TORCH_CHECK(t.stride(2) == 1, name, "'s last dimension must be contiguous");
    // the stride of a dimension of one is free: 0 is as good as any
    return w4a16_rows{t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
}

Paged paged_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& tables, const at::Tensor& lens,
               const c10::optional<at::Tensor>& cu_q, int64_t tokens, int64_t max_q) {
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides(),
                "k_pages and v_pages must be [pages, heads, page size, head dim] of the same strides");
    TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k_pages and v_pages must have the same type");
    TORCH_CHECK(k.stride(3) == 1, "the pages' last dimension must be contiguous");
    check_ints(tables, 2, "tables");
    check_ints(lens, 1, "lens");
    TORCH_CHECK(tables.size(0) == lens.size(0), "tables has ", tables.size(0), " sequences, lens ", lens.size(0));
    const int64_t most = 0x7fffffff;
    TORCH_CHECK(max_q >= 0 && max_q <= most && tokens <= most && k.size(0) <= most && tables.size(1) <= most &&
                    tables.size(0) <= most,
                "sizes must fit 32 bits");
    if (cu_q.has_value()) {
        check_ints(*cu_q, 1, "cu_q");
        TORCH_CHECK(cu_q->size(0) == lens.size(0) + 1, "cu_q must hold ", lens.size(0) + 1, " offsets, got ", cu_q->size(0));
    } else {
        TORCH_CHECK(tokens == lens.size(0), tokens, " rows for ", lens.size(0),
                    " sequences: without cu_q each has one new token");
    }
    TORCH_CHECK(k.is_cuda(), "k_pages must be a CUDA tensor (no CPU path exists)");
    on_device(v, k, "v_pages");
    on_device(tables, k, "tables");
    on_device(lens, k, "lens");
    if (cu_q.has_value()) on_device(*cu_q, k, "cu_q");
    Paged p = {};
    auto stride = [&](int64_t d) { return k.size(d) > 1 ? k.stride(d) : 0; };
    p.pages.k_dev = k.data_ptr();
    p.pages.v_dev = v.data_ptr();
    p.pages.stride_page = stride(0);
    p.pages.stride_head = stride(1);
    p.pages.stride_token = stride(2);
    p.pages.num_pages = static_cast<int>(k.size(0));
    p.pages.heads_kv = static_cast<int>(k.size(1));
    p.pages.page_size = static_cast<int>(k.size(2));
    p.pages.head_dim = static_cast<int>(k.size(3));
    p.pages.dtype = dtype_of(k);
    p.pages.device = k.device().index();
    p.seqs.tables_dev = tables.data_ptr<int32_t>();
    p.seqs.lens_dev = lens.data_ptr<int32_t>();
    p.seqs.cu_q_dev = cu_q.has_value() ? cu_q->data_ptr<int32_t>() : nullptr;
    p.seqs.table_stride = tables.size(0) > 1 ? tables.stride(0) : 0;
    p.seqs.table_width = static_cast<int>(tables.size(1));
    p.seqs.batch = static_cast<int>(lens.size(0));
    p.seqs.tokens = static_cast<int>(tokens);
    p.seqs.max_q = static_cast<int>(max_q);
    return p;
}

// q and out with the pages' sizes; out is made when none is given.
at::Tensor append_kv(const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& k, const at::Tensor& v,
                     const at::Tensor& tables, const at::Tensor& lens, const c10::optional<at::Tensor>& cu_q,
                     const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& rope, bool interleaved,
                     const c10::optional<at::Tensor>& q_out) {
    TORCH_CHECK(k.dim() == 3 && k_pages.dim() == 4, "k must be [tokens, heads, head dim] and k_pages 4-dimensional");
    const int64_t tokens = k.size(0);
    no_grad(k, "k");
    no_grad(v, "v");
    no_grad(k_pages, "k_pages");
    no_grad(v_pages, "v_pages");
    const w4a16_rows kr = rows_of(k, k_pages, tokens, k_pages.size(1), "k");
    const w4a16_rows vr = rows_of(v, k_pages, tokens, k_pages.size(1), "v");
    TORCH_CHECK(q.has_value() || !q_out.has_value(), "q_out without q");
    w4a16_rows qr = {}, qor = {};
    int64_t heads = 0;
    at::Tensor out;
    if (q.has_value()) {
        no_grad(*q, "q");
        TORCH_CHECK(q->dim() == 3, "q must be [tokens, heads, head dim]");
        heads = q->size(1);
        qr = rows_of(*q, k_pages, tokens, heads, "q");
        if (q_out.has_value()) {
            qor = rows_of(*q_out, k_pages, tokens, heads, "q_out");
            no_grad(*q_out, "q_out");
            out = *q_out;
        }
    }
    if (rope.has_value())
        TORCH_CHECK(rope->dim() == 2 && rope->scalar_type() == at::kFloat && rope->is_contiguous(),
                    "rope must be a contiguous float32 [positions, rope dim] table");
    const Paged p = paged_of(k_pages, v_pages, tables, lens, cu_q, tokens, tokens);
    on_device(k, k_pages, "k");
    on_device(v, k_pages, "v");
    if (q.has_value()) on_device(*q, k_pages, "q");
    if (rope.has_value()) on_device(*rope, k_pages, "rope");
    if (q_out.has_value()) on_device(*q_out, k_pages, "q_out");
    if (q.has_value() && !q_out.has_value()) {
        out = at::empty(q->sizes(), q->options());
        qor = w4a16_rows{out.data_ptr(), out.stride(0), out.stride(1)};
    }
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k_pages.device().index()).stream();
    if (tokens > 0)  // a q without heads is no q: k and v are stored all the same
        check(w4a16_append_kv(&p.pages, &p.seqs, &kr, &vr, heads > 0 ? &qr : nullptr, &qor, static_cast<int>(heads),
                              rope.has_value() ? rope->data_ptr<float>() : nullptr,
                              rope.has_value() ? static_cast<int>(std::min<int64_t>(rope->size(0), 0x7fffffff)) : 0,
                              rope.has_value() ? static_cast<int>(rope->size(1)) : 0, interleaved ? 1 : 0, stream));
    return out;
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
                           const at::Tensor& tables, const at::Tensor& lens, const c10::optional<at::Tensor>& cu_q,
                           int64_t max_q, double scale, int64_t window, int64_t sinks,
                           const c10::optional<at::Tensor>& out_arg) {
    TORCH_CHECK(q.dim() == 3 && k_pages.dim() == 4, "q must be [tokens, heads, head dim] and k_pages 4-dimensional");
    no_grad(q, "q");
    no_grad(k_pages, "k_pages");
    no_grad(v_pages, "v_pages");
    const int64_t tokens = q.size(0), heads = q.size(1);
    TORCH_CHECK(window >= 0 && window <= 0x7fffffff && sinks >= 0 && sinks <= 0x7fffffff,
                "window and sinks must be non-negative 32-bit numbers");
    const w4a16_rows qr = rows_of(q, k_pages, tokens, heads, "q");
    w4a16_rows outr = {};
    if (out_arg.has_value()) {
        no_grad(*out_arg, "out");
        outr = rows_of(*out_arg, k_pages, tokens, heads, "out");
    }
    const Paged p = paged_of(k_pages, v_pages, tables, lens, cu_q, tokens, max_q);
    on_device(q, k_pages, "q");
    if (out_arg.has_value()) on_device(*out_arg, k_pages, "out");
    const c10::cuda::CUDAGuard guard(k_pages.device());
    at::Tensor out = out_arg.has_value() ? *out_arg : at::empty(q.sizes(), q.options());
    if (!out_arg.has_value()) outr = w4a16_rows{out.data_ptr(), out.stride(0), out.stride(1)};
    if (tokens == 0) return out;
    // one workspace a call, from torch's allocator on the current stream: calls that overlap
    // on other streams, and graphs, have their own (bare memory: a tensor costs a microsecond)
    const size_t need = w4a16_paged_attention_workspace_size(&p.pages, &p.seqs, static_cast<int>(heads),
                                                             static_cast<int>(window), static_cast<int>(sinks));
    c10::DataPtr ws;
    if (need > 0) ws = c10::cuda::CUDACachingAllocator::get()->allocate(need);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k_pages.device().index()).stream();
    check(w4a16_paged_attention(&p.pages, &p.seqs, &qr, &outr, static_cast<int>(heads), static_cast<float>(scale),
                                static_cast<int>(window), static_cast<int>(sinks), ws.get(), need, stream));
    return out;
}

void copy_ids(const at::Tensor& k, const at::Tensor& v, const int32_t* src, const int32_t* dst, int64_t pairs) {
    TORCH_CHECK((k.dim() == 4 || k.dim() == 5) && k.sizes() == v.sizes() && k.strides() == v.strides() &&
                    k.scalar_type() == v.scalar_type(),
                "k_pages and v_pages must be [(layers,) pages, heads, page size, head dim] of the same type and strides");
    no_grad(k, "k_pages");
    no_grad(v, "v_pages");
    const int64_t at_page = k.dim() - 4;
    // a page's three dimensions, in whatever order, must fill one block of memory
    int64_t elems = 1, left = 3;
    bool used[3] = {};
    while (left > 0) {
        bool found = false;
        for (int i = 0; i < 3 && !found; ++i) {
            const int64_t n = k.size(at_page + 1 + i);
            if (!used[i] && (n == 1 || k.stride(at_page + 1 + i) == elems)) {
                used[i] = found = true;
                elems *= n;
            }
        }
        TORCH_CHECK(found, "a page must be one block of memory");
        --left;
    }
    TORCH_CHECK(k.is_cuda(), "k_pages must be a CUDA tensor (no CPU path exists)");
    on_device(v, k, "v_pages");
    if (k.numel() == 0) {
        TORCH_CHECK(pairs == 0, "no pages to copy");
        return;
    }
    const int64_t size = k.element_size(), pages = k.size(at_page), layers = k.dim() == 5 ? k.size(0) : 1;
    TORCH_CHECK(pages <= 0x7fffffff && layers <= 32767 && pairs <= 0x7fffffff, "sizes must fit 32 bits");
    const int64_t stride_page = pages > 1 ? k.stride(at_page) * size : elems * size;
    const int64_t stride_layer = layers > 1 ? k.stride(0) * size : 0;
    TORCH_CHECK(layers == 1 || stride_layer >= (pages - 1) * stride_page + elems * size ||
                    stride_page >= (layers - 1) * stride_layer + elems * size,
                "the layers' pages overlap");
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(k.device().index()).stream();
    check(w4a16_copy_pages(k.data_ptr(), v.data_ptr(), stride_layer, stride_page, static_cast<int>(layers),
                           static_cast<int>(pages), elems * size, src, dst, static_cast<int>(pairs), k.device().index(),
                           stream));
}

void copy_pages(const at::Tensor& k, const at::Tensor& v, const at::Tensor& src, const at::Tensor& dst) {
    for (const at::Tensor* t : {&src, &dst})
        TORCH_CHECK(t->dim() == 1 && t->scalar_type() == at::kInt && t->is_cpu() && t->is_contiguous(),
                    "src and dst must be lists of page ids on the host");
    TORCH_CHECK(src.size(0) == dst.size(0), src.size(0), " source pages for ", dst.size(0));
    copy_ids(k, v, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), src.size(0));
}

// The ids as Python lists: without the microseconds that two tensors cost.
void copy_page_lists(const at::Tensor& k, const at::Tensor& v, const std::vector<int64_t>& src,
                     const std::vector<int64_t>& dst) {
    TORCH_CHECK(src.size() == dst.size(), src.size(), " source pages for ", dst.size());
    std::vector<int32_t> ids[2];
    for (int i = 0; i < 2; ++i) {
        const std::vector<int64_t>& from = i ? dst : src;
        ids[i].reserve(from.size());
        for (const int64_t x : from) {
            TORCH_CHECK(x >= 0 && x <= 0x7fffffff, "page ids must fit 32 bits, got ", x);
            ids[i].push_back(static_cast<int32_t>(x));
        }
    }
    copy_ids(k, v, ids[0].data(), ids[1].data(), static_cast<int64_t>(src.size()));
}

}  // namespace

PYBIND11_MODULE(_w4a16_torch, m) {
    m.doc() = "torch fast path of the W4A16 quantized linear (calls the C ABI of libdrofell_w4a16.so)";
    m.def("linear", &linear, "Y = X W (+ bias) on PATH_AUTO", pybind11::arg("handle"), pybind11::arg("x"),
          pybind11::arg("bias") = pybind11::none());
    m.def("gemm_gather", &gemm_gather, "this rank's columns of X W into every rank's Y (w4a16_gemm_gather)",
          pybind11::arg("handle"), pybind11::arg("comm"), pybind11::arg("x"), pybind11::arg("y_all"),
          pybind11::arg("ld"), pybind11::arg("col0"));
    m.def("release", &release, "free the workspaces kept for a handle");
    m.def("append_kv", &append_kv, "store new k and v into pages, rotate q (w4a16_append_kv)");
    m.def("paged_attention", &paged_attention, "attention over pages (w4a16_paged_attention)");
    m.def("copy_pages", &copy_pages, "copy whole pages of every layer (w4a16_copy_pages)");
    m.def("copy_page_lists", &copy_page_lists, "copy_pages with the ids as lists");
}
