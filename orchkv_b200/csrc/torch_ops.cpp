// torch_ops.cpp — the paged operators on torch tensors (orchkv_torch module,
// used by orchkv_b200/paged.py).
//
// A decode step makes each of these calls once a layer, and the kernels of a
// small step take a few microseconds: checking a dozen tensors from Python
// takes longer than that, so the checks, the outputs' allocation and the
// stream are taken care of here.  Arguments that do not fit raise ValueError,
// a failed call RuntimeError.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>

#include "orchkv/paged_ops.h"
#include "paged_overlap.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void refuse(const std::string &what) { throw py::value_error(what); }

void run(int rc, const char *name)
{
    if (rc != ORCHKV_OK) throw std::runtime_error(std::string("orchkv_") + name + " failed: " + std::to_string(rc));
}

at::ScalarType scalar_of(int dtype)
{
    return dtype == DTYPE_BF16 ? at::kBFloat16 : dtype == DTYPE_FP16 ? at::kHalf : at::kFloat;
}

// One cache's pages on one device.
class Pages {
public:
    // heads 0: pages of one head each, as many heads as a call's table has
    Pages(int device, uintptr_t k, uintptr_t v, int64_t page, int64_t head, int64_t token, uint32_t n_pages,
          uint32_t page_tokens, uint32_t heads, uint32_t d_head, int dtype, OptTensor k_pages, OptTensor v_pages)
        : dev_(device), slab_(heads == 0), type_(scalar_of(dtype)), k_pages_(std::move(k_pages)),
          v_pages_(std::move(v_pages)),
          pg_{reinterpret_cast<void *>(k), reinterpret_cast<void *>(v), page, head, token, n_pages, page_tokens,
              heads, d_head, dtype}
    {
    }

    py::object append(const Tensor &k, const Tensor &v, const Tensor &table, const Tensor &lens,
                      const Tensor &starts, const OptTensor &q, const OptTensor &turns, bool interleaved,
                      double scale, const OptTensor &positions, const OptTensor &q_norm,
                      const OptTensor &k_norm, double eps, OptTensor q_out) const
    {
        const int64_t rows = k.dim() == 3 ? k.size(0) : -1;
        no_gradient_of_pages();
        orchkv_batch_t b;
        const orchkv_pages_t pg = batch(table, lens, starts, rows, std::nullopt, &b);
        orchkv_append_args_t a = {};
        a.k = row_tensor(k, "k", pg.n_kv_heads, rows);
        a.v = row_tensor(v, "v", pg.n_kv_heads, rows);
        if (q) {
            a.q = row_tensor(*q, "q", -1, rows);
            a.n_q_heads = (uint32_t)q->size(1);
            if (!q_out) q_out = at::empty(q->sizes(), q->options());
            a.q_out = row_tensor(*q_out, "q_out", a.n_q_heads, rows);
            const okv::RowSpan qs = span(a.q, a.n_q_heads, rows), os = span(a.q_out, a.n_q_heads, rows);
            if (!okv::same_rows(qs, os) && okv::overlap(qs, os)) refuse("q_out must be q itself or not overlap it");
            if (okv::overlaps_itself(os)) refuse("q_out: rows and heads must not overlap");
            if (okv::overlap(os, span(a.k, pg.n_kv_heads, rows)) || okv::overlap(os, span(a.v, pg.n_kv_heads, rows)))
                refuse("q_out must not overlap k and v");
        } else if (q_out || q_norm) {
            refuse("q_out and q_norm go with q");
        }
        if (positions) {
            if ((positions->scalar_type() != at::kInt && positions->scalar_type() != at::kLong) ||
                positions->dim() != 1 || positions->size(0) != rows || !positions->is_contiguous() ||
                !here(*positions))
                refuse("positions must be int32 or int64 [rows], contiguous, on the pages' device");
            a.positions = positions->data_ptr();
            a.positions_64 = positions->scalar_type() == at::kLong;
        }
        a.q_norm = norm(q_norm, "q_norm");
        a.k_norm = norm(k_norm, "k_norm");
        a.eps = (float)eps;
        a.scale = (float)scale;
        a.interleaved = interleaved;
        if (turns) {
            if (turns->scalar_type() != at::kDouble || turns->dim() != 1 || !turns->is_contiguous() ||
                !here(*turns) || 2 * turns->size(0) > (int64_t)pg.d_head)
                refuse("rotary wider than a head, or on another device");
            no_gradient(*turns, "rotary");
            a.turns = turns->data_ptr<double>();
            a.rot_dim = 2 * (uint32_t)turns->size(0);
        }
        if ((!pg.page_stride && pg.n_pages > 1) || (!pg.token_stride && pg.page_tokens > 1) ||
            (!pg.head_stride && !b.table_head_stride && pg.n_kv_heads > 1))
            refuse("pages to write into must not be broadcast over pages, tokens or heads");
        c10::cuda::CUDAGuard guard(dev_);
        run(orchkv_paged_append(&pg, &b, &a, stream()), "paged_append");
        if (k_pages_) written(*k_pages_);
        if (v_pages_) written(*v_pages_);
        if (q_out) written(*q_out);
        return q_out ? py::cast(*q_out) : py::none();
    }

    py::object attend(const Tensor &q, const Tensor &table, const Tensor &lens, const Tensor &starts,
                      std::optional<double> scale, int64_t window, std::optional<int64_t> max_new,
                      bool return_lse, OptTensor out) const
    {
        orchkv_batch_t b;
        orchkv_attend_args_t a = {};
        no_gradient_of_pages();
        a.q = row_tensor(q, "q", -1, -1);
        const int64_t rows = q.size(0), hq = q.size(1);
        const orchkv_pages_t pg = batch(table, lens, starts, rows, max_new, &b);
        common(pg, hq, scale, window, &a.n_q_heads, &a.scale, &a.window);
        c10::cuda::CUDAGuard guard(dev_);
        if (!out) out = at::empty(q.sizes(), q.options());
        a.out = row_tensor(*out, "out", hq, rows);
        if (okv::overlap(span(a.q, hq, rows), span(a.out, hq, rows))) refuse("out must not overlap q");
        if (okv::overlaps_itself(span(a.out, hq, rows))) refuse("out: rows and heads must not overlap");
        Tensor lse;
        if (return_lse) {
            lse = at::empty({rows, hq}, q.options().dtype(at::kFloat));
            a.lse = lse.data_ptr<float>();
        }
        const size_t need = orchkv_paged_attend_workspace(&pg, &b, &a);
        Tensor ws;
        if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        run(orchkv_paged_attend(&pg, &b, &a, need ? ws.data_ptr() : nullptr, need, stream()), "paged_attend");
        written(*out);
        if (return_lse) return py::make_tuple(*out, lse);
        return py::cast(*out);
    }

    py::object block_mass(const Tensor &q, const Tensor &lse, const Tensor &table, const Tensor &lens,
                          const Tensor &starts, std::optional<double> scale, int64_t window,
                          std::optional<int64_t> max_new, OptTensor out) const
    {
        orchkv_batch_t b;
        orchkv_mass_args_t a = {};
        no_gradient_of_pages();
        a.q = row_tensor(q, "q", -1, -1);
        const int64_t rows = q.size(0), hq = q.size(1);
        const orchkv_pages_t pg = batch(table, lens, starts, rows, max_new, &b);
        common(pg, hq, scale, window, &a.n_q_heads, &a.scale, &a.window);
        if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != rows || lse.size(1) != hq ||
            !lse.is_contiguous() || !here(lse))
            refuse("lse must be fp32 [rows, query heads], contiguous, on the pages' device");
        no_gradient(lse, "lse");
        a.lse = lse.data_ptr<float>();
        c10::cuda::CUDAGuard guard(dev_);
        const int64_t shape[3] = {b.n_seqs, pg.n_kv_heads, b.table_width};
        if (!out) {
            out = at::empty(shape, q.options().dtype(at::kFloat));
        } else if (out->scalar_type() != at::kFloat || out->sizes() != at::IntArrayRef(shape, 3) ||
                   !out->is_contiguous() || !here(*out)) {
            refuse("out must be fp32 [sequences, KV heads, table width], contiguous, on the pages' device");
        }
        no_gradient(*out, "out");
        a.mass = out->data_ptr<float>();
        if (okv::mass_overlaps(a.mass, shape[0], shape[1], shape[2], span(a.q, hq, rows), a.lse))
            refuse("out must not overlap q or lse");
        const size_t need = orchkv_paged_block_mass_workspace(&pg, &b, &a);
        Tensor ws;
        if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        run(orchkv_paged_block_mass(&pg, &b, &a, need ? ws.data_ptr() : nullptr, need, stream()),
            "paged_block_mass");
        written(*out);
        return py::cast(*out);
    }

private:
    bool here(const Tensor &t) const { return t.is_cuda() && t.get_device() == dev_; }
    // Every tensor a result depends on: a gradient, backward or forward, would be
    // dropped here.
    static void no_gradient(const Tensor &x, const char *name)
    {
        const c10::AutogradState &on = c10::AutogradState::get_tls_state();
        if ((on.get_grad_mode() && x.requires_grad()) || (on.get_fw_grad_mode() && x._fw_grad(0).defined()))
            refuse(std::string(name) + " requires a gradient, which these operators do not have");
    }
    void no_gradient_of_pages() const
    {
        if (k_pages_) no_gradient(*k_pages_, "k pages");
        if (v_pages_) no_gradient(*v_pages_, "v pages");
    }
    // A tensor that a backward pass has saved is known to have changed.
    static void written(const Tensor &x)
    {
        if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
    }
    void *stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev_).stream(); }

    // The pages as this call's tables see them, and its sequences.
    orchkv_pages_t batch(const Tensor &table, const Tensor &lens, const Tensor &starts, int64_t rows,
                         std::optional<int64_t> max_new, orchkv_batch_t *b) const
    {
        if (rows < 0) refuse("row tensors have three dimensions: rows, heads, head_dim");
        if (table.scalar_type() != at::kInt || lens.scalar_type() != at::kInt || starts.scalar_type() != at::kInt)
            refuse("table, lens and starts must be int32");
        if (table.dim() != (slab_ ? 3 : 2))
            refuse(slab_ ? "table must be [sequences, KV heads, width]" : "table must be [sequences, width]");
        const int64_t n = table.size(0), width = table.size(-1);
        if (lens.dim() != 1 || starts.dim() != 1 || lens.size(0) != n || starts.size(0) != n + 1)
            refuse("table, lens and starts must have n, n and n + 1 entries");
        if (table.stride(-1) != 1 || !lens.is_contiguous() || !starts.is_contiguous())
            refuse("table rows, lens and starts must be contiguous");
        if (width == 0 || (slab_ && table.size(1) == 0)) refuse("a table of no blocks");
        if (!here(table) || !here(lens) || !here(starts)) refuse("every tensor must be on the pages' device");
        if (max_new && *max_new < 0) refuse("max_new must not be negative");
        orchkv_pages_t pg = pg_;
        if (slab_) pg.n_kv_heads = (uint32_t)table.size(1);
        b->table = table.data_ptr<int32_t>();
        b->table_seq_stride = table.stride(0);
        b->table_head_stride = slab_ ? table.stride(1) : 0;
        b->table_width = (uint32_t)width;
        b->n_seqs = (uint32_t)n;
        b->lens = lens.data_ptr<int32_t>();
        b->starts = starts.data_ptr<int32_t>();
        b->n_rows = (uint32_t)rows;
        b->max_new = (uint32_t)(max_new && *max_new < rows ? *max_new : rows);
        return pg;
    }

    orchkv_rows_t row_tensor(const Tensor &x, const char *name, int64_t heads, int64_t rows) const
    {
        if (x.dim() != 3 || x.size(2) != (int64_t)pg_.d_head || (heads >= 0 && x.size(1) != heads) ||
            (rows >= 0 && x.size(0) != rows))
            refuse(std::string(name) + " must be [rows, heads, " + std::to_string(pg_.d_head) + "]" +
                   (heads >= 0 ? " with " + std::to_string(heads) + " heads" : "") +
                   (rows >= 0 ? " and " + std::to_string(rows) + " rows" : ""));
        if (x.scalar_type() != type_) refuse(std::string(name) + " must have the pages' dtype");
        const int64_t align = 16 / x.element_size();
        if (x.numel() && (x.stride(2) != 1 || x.stride(0) % align || x.stride(1) % align ||
                          reinterpret_cast<uintptr_t>(x.data_ptr()) % 16))
            refuse(std::string(name) + ": heads must be contiguous, pointer and strides multiples of 16 bytes");
        if (!here(x)) refuse(std::string(name) + " must be on the pages' device");
        no_gradient(x, name);
        return orchkv_rows_t{x.data_ptr(), x.stride(0), x.stride(1)};
    }

    okv::RowSpan span(const orchkv_rows_t &r, int64_t heads, int64_t rows) const
    {
        const int64_t e = type_ == at::kFloat ? 4 : 2;
        return okv::row_span(r, rows, heads, pg_.d_head * e, e);
    }

    const void *norm(const OptTensor &w, const char *name) const
    {
        if (!w) return nullptr;
        if (w->dim() != 1 || w->size(0) != (int64_t)pg_.d_head || w->scalar_type() != type_ ||
            !w->is_contiguous() || !here(*w))
            refuse(std::string(name) + " must be [" + std::to_string(pg_.d_head) +
                   "] of the pages' dtype, contiguous, on the pages' device");
        no_gradient(*w, name);
        return w->data_ptr();
    }

    void common(const orchkv_pages_t &pg, int64_t hq, std::optional<double> scale, int64_t window,
                uint32_t *hq_out, float *scale_out, uint32_t *window_out) const
    {
        if (hq == 0 || hq % pg.n_kv_heads)
            refuse(std::to_string(hq) + " query heads do not share " + std::to_string(pg.n_kv_heads) + " KV heads");
        if (window < 0) refuse("window must not be negative");
        *hq_out = (uint32_t)hq;
        *scale_out = scale ? (float)*scale : (float)(1.0 / std::sqrt((double)pg.d_head));
        // no sequence is longer than 2^30: a larger window is no window
        *window_out = window > (1 << 30) ? 0 : (uint32_t)window;
    }

    int dev_;
    bool slab_;
    at::ScalarType type_;
    OptTensor k_pages_, v_pages_;          // none: memory that is no tensor
    orchkv_pages_t pg_;
};

}  // namespace

PYBIND11_MODULE(orchkv_torch, m)
{
    m.doc() = "OrchKvCache (B200): operators over paged caches on torch tensors";
    py::class_<Pages>(m, "Pages")
        .def(py::init<int, uintptr_t, uintptr_t, int64_t, int64_t, int64_t, uint32_t, uint32_t, uint32_t, uint32_t,
                      int, OptTensor, OptTensor>(),
             py::arg("device"), py::arg("k_ptr"), py::arg("v_ptr"), py::arg("page_stride"), py::arg("head_stride"),
             py::arg("token_stride"), py::arg("n_pages"), py::arg("page_tokens"), py::arg("heads"),
             py::arg("d_head"), py::arg("dtype"), py::arg("k_pages"), py::arg("v_pages"))
        .def("append", &Pages::append)
        .def("attend", &Pages::attend)
        .def("block_mass", &Pages::block_mass);
}
