// torch_attn.cpp -- the attention ops of crispybits_kernels._ext (prompt_attention, kv4_append, kv4_read,
// kv4_attention) over the C ABI of include/crispybits_attention.h.  As in torch_ext.cpp: tensor checks fail through
// TORCH_CHECK, outputs and scratch come from torch's caching allocator on the tensors' device, the kernels run on
// torch's current HIP stream of that device.  Host code only.
#include <torch/extension.h>
#include <c10/hip/HIPStream.h>

#include "crispybits_attention.h"

namespace {

using at::Tensor;
using OptT = c10::optional<Tensor>;

void ok(int rc) { TORCH_CHECK(rc == CBK_OK, cbk_last_error()); }

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kHalf: return CBK_F16;
        case at::kBFloat16: return CBK_BF16;
        case at::kFloat: return CBK_F32;
        default: return -1;
    }
}

void* stream_of(int device) { return c10::hip::getCurrentHIPStream(device).stream(); }

void check_values(const Tensor& t, const char* name, int64_t dim) {
    TORCH_CHECK(t.is_cuda(), name, " must be CUDA");
    TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimensions");
    TORCH_CHECK(dtype_of(t.scalar_type()) >= 0, name, " must be fp16/bf16/fp32");
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
                " requires a gradient: these ops have no backward (use torch.no_grad())");
}

// t itself where the kernels can step through its rows in 16-byte pieces, else a contiguous copy.
Tensor rows_of(const Tensor& t) {
    const int64_t unit = 16 / t.element_size();
    bool fits = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) fits = fits && t.stride(i) >= 0 && (t.size(i) <= 1 || t.stride(i) % unit == 0);
    fits = fits && (t.size(0) <= 1 || t.stride(0) <= (1 << 23));
    return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A stride that is never stepped by may be anything: 0 then.
int64_t step(const Tensor& t, int64_t i) { return t.size(i) <= 1 ? 0 : t.stride(i); }

Tensor whole(const Tensor& t) {
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone(at::MemoryFormat::Contiguous);
}

const int32_t* index_ptr(const Tensor& t, const Tensor& with, const char* name, int64_t dim) {
    TORCH_CHECK(t.is_cuda() && t.device() == with.device(), name, " must be on the same device as the other tensors");
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == dim, name, " must be contiguous int32 with ",
                dim, " dimension(s)");
    return t.data_ptr<int32_t>();
}

bool overlap(const Tensor& a, const Tensor& b) {
    auto span = [](const Tensor& t) {
        int64_t n = 1;
        for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
        const char* p = static_cast<const char*>(t.data_ptr());
        return std::make_pair(p, p + n * t.element_size());
    };
    if (a.numel() == 0 || b.numel() == 0) return false;
    const auto x = span(a), y = span(b);
    return x.first < y.second && y.first < x.second;
}

Tensor out_for(const OptT& out, const Tensor& q, std::initializer_list<const Tensor*> read) {
    if (!out.has_value()) return at::empty(q.sizes(), q.options());
    TORCH_CHECK(out->is_cuda() && out->device() == q.device() && out->scalar_type() == q.scalar_type() &&
                out->sizes() == q.sizes() && out->is_contiguous() &&
                reinterpret_cast<uintptr_t>(out->data_ptr()) % 16 == 0,
                "out must be a contiguous, 16-byte aligned tensor of q's shape, dtype and device");
    TORCH_CHECK(!(at::GradMode::is_enabled() && out->requires_grad()), "out requires a gradient");
    for (const Tensor* t : read) TORCH_CHECK(!overlap(*out, *t), "out overlaps an input");
    return *out;
}

struct Pool {
    int32_t* pages;
    int64_t num_pages, heads, page_size, width, seqs;
    int head_dim;
    const int32_t *table, *lens, *cu;
    int device;
};

Pool pool_of(const Tensor& pages, int64_t page_size, int64_t head_dim, const Tensor& table, const Tensor& lens,
             const OptT& cu) {
    TORCH_CHECK(pages.is_cuda() && pages.scalar_type() == at::kInt && pages.dim() == 3 && pages.is_contiguous(),
                "pages must be a contiguous CUDA int32 tensor [pages, kv heads, words]");
    const int64_t words = head_dim > 0 && head_dim <= 256 ? cbk_kv4_page_words((int)head_dim, page_size) : -1;
    TORCH_CHECK(words > 0, "head_dim must be a multiple of 8 up to 256, page_size a power of two from 32 to 65536");
    TORCH_CHECK(pages.size(2) == words, "pages of ", page_size, " tokens and head_dim ", head_dim, " have ", words,
                " words, not ", pages.size(2));
    Pool p;
    p.table = index_ptr(table, pages, "block_table", 2);
    p.lens = index_ptr(lens, pages, "seq_lens", 1);
    TORCH_CHECK(table.size(0) == lens.size(0), "block_table and seq_lens must have one row per sequence");
    p.cu = nullptr;
    if (cu.has_value()) {
        p.cu = index_ptr(*cu, pages, "cu_seqlens", 1);
        TORCH_CHECK(cu->size(0) == lens.size(0) + 1, "cu_seqlens must have one more entry than there are sequences");
    }
    p.pages = pages.data_ptr<int32_t>();
    p.num_pages = pages.size(0), p.heads = pages.size(1), p.page_size = page_size;
    p.width = table.size(1), p.seqs = lens.size(0), p.head_dim = (int)head_dim;
    p.device = pages.get_device();
    return p;
}

int64_t kv4_page_words(int64_t head_dim, int64_t page_size) {
    const int64_t n = head_dim > 0 && head_dim < (1 << 20) ? cbk_kv4_page_words((int)head_dim, page_size) : -1;
    TORCH_CHECK(n > 0, "head_dim must be a multiple of 8 up to 256, page_size a power of two from 32 to 65536");
    return n;
}

void kv4_append(const Tensor& pages, int64_t page_size, int64_t head_dim, const Tensor& k, const Tensor& v,
                const Tensor& table, const Tensor& lens, const OptT& cu) {
    check_values(k, "k", 3);
    check_values(v, "v", 3);
    const Pool p = pool_of(pages, page_size, head_dim, table, lens, cu);
    TORCH_CHECK(k.device() == pages.device() && v.device() == pages.device(), "k, v and pages on different devices");
    TORCH_CHECK(k.scalar_type() == v.scalar_type() && k.sizes() == v.sizes(), "k and v must have one shape and dtype");
    TORCH_CHECK(k.size(1) == p.heads && k.size(2) == head_dim, "k and v must be [rows, ", p.heads, ", ", head_dim, "]");
    TORCH_CHECK(cu.has_value() || k.size(0) == p.seqs, "without cu_seqlens k and v have one row per sequence");
    const Tensor kr = rows_of(k), vr = rows_of(v);
    ok(cbk_kv4_append(p.pages, p.num_pages, p.heads, p.head_dim, p.page_size, kr.data_ptr(), vr.data_ptr(),
                      dtype_of(k.scalar_type()), k.size(0), step(kr, 0), step(kr, 1), step(vr, 0), step(vr, 1), p.table,
                      p.width, p.lens, p.cu, p.seqs, p.device, stream_of(p.device)));
}

std::tuple<Tensor, Tensor> kv4_read(const Tensor& pages, int64_t page_size, int64_t head_dim, const Tensor& table,
                                    const Tensor& lens, const OptT& cu, int64_t rows, py::object dtype) {
    const Pool p = pool_of(pages, page_size, head_dim, table, lens, cu);
    const at::ScalarType t = torch::python::detail::py_object_to_dtype(dtype);
    TORCH_CHECK(dtype_of(t) >= 0, "dtype must be fp16/bf16/fp32");
    TORCH_CHECK(rows >= 0, "rows must not be negative");
    TORCH_CHECK(cu.has_value() || rows == p.seqs, "without cu_seqlens there is one row per sequence");
    Tensor k = at::empty({rows, p.heads, head_dim}, pages.options().dtype(t)), v = at::empty_like(k);
    ok(cbk_kv4_read(p.pages, p.num_pages, p.heads, p.head_dim, p.page_size, k.data_ptr(), v.data_ptr(), dtype_of(t), rows,
                    p.table, p.width, p.lens, p.cu, p.seqs, p.device, stream_of(p.device)));
    return {k, v};
}

Tensor kv4_attention(const Tensor& q, const Tensor& pages, int64_t page_size, int64_t head_dim, const Tensor& table,
                     const Tensor& lens, double scale, const OptT& out) {
    check_values(q, "q", 4);
    const Pool p = pool_of(pages, page_size, head_dim, table, lens, c10::nullopt);
    TORCH_CHECK(q.device() == pages.device(), "q and pages on different devices");
    TORCH_CHECK(q.size(0) == p.seqs && q.size(3) == head_dim, "q must be [", p.seqs, ", new tokens, heads, ", head_dim, "]");
    const Tensor qc = whole(q);
    const Tensor o = out_for(out, q, {&q, &pages});
    if (o.numel() == 0) return o;
    const int64_t n = cbk_kv4_attention_partial_floats(p.seqs, q.size(1), q.size(2), p.heads, p.head_dim, p.page_size,
                                                       p.width);
    const Tensor part = n > 0 ? at::empty({n}, q.options().dtype(at::kFloat)) : Tensor();
    ok(cbk_kv4_attention(qc.data_ptr(), dtype_of(q.scalar_type()), p.seqs, q.size(1), q.size(2), p.pages, p.num_pages,
                         p.heads, p.head_dim, p.page_size, p.table, p.width, p.lens, (float)scale,
                         n > 0 ? part.data_ptr<float>() : nullptr, n, o.data_ptr(), p.device, stream_of(p.device)));
    return o;
}

Tensor prompt_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, int64_t max_seqlen,
                        double scale, const OptT& out) {
    check_values(q, "q", 3);
    check_values(k, "k", 3);
    check_values(v, "v", 3);
    TORCH_CHECK(k.device() == q.device() && v.device() == q.device(), "q, k and v on different devices");
    TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "q, k and v must have one dtype");
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2),
                "k and v must be [rows, kv heads, head_dim] with q's rows and head_dim");
    TORCH_CHECK(q.size(2) <= 256, "prompt_attention: head_dim must be a multiple of 8 up to 256");
    const int32_t* c = index_ptr(cu, q, "cu_seqlens", 1);
    TORCH_CHECK(cu.size(0) >= 1, "cu_seqlens must have one more entry than there are sequences");
    const Tensor qr = rows_of(q), kr = rows_of(k), vr = rows_of(v);
    const Tensor o = out_for(out, q, {&q, &k, &v});
    const int dev = q.get_device();
    ok(cbk_prompt_attention(qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), dtype_of(q.scalar_type()), q.size(0), q.size(1),
                            k.size(1), (int)q.size(2), step(qr, 0), step(qr, 1), step(kr, 0), step(kr, 1), step(vr, 0),
                            step(vr, 1), c, cu.size(0) - 1, max_seqlen, (float)scale, out.has_value() ? 0 : 1,
                            o.data_ptr(), dev, stream_of(dev)));
    return o;
}

}  // namespace

void bind_attention(py::module& m) {
    m.def("kv4_page_words", &kv4_page_words, "int32 words of one page and kv head of the 4-bit cache");
    m.def("kv4_append", &kv4_append, "Quantize new tokens' keys and values into the paged 4-bit cache");
    m.def("kv4_read", &kv4_read, "Stored tokens of the 4-bit cache as values");
    m.def("kv4_attention", &kv4_attention, "Attention of the newest tokens over the paged 4-bit cache");
    m.def("prompt_attention", &prompt_attention, "Causal attention over packed prompts");
}
