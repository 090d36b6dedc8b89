// Python entry points of the paged KV cache (fcci_paged.h), part of the `attn_varlen` module.
#pragma once
#include "binding_common.h"
#include "fcci_paged.h"

namespace fcci_py {

using OptTensor = c10::optional<at::Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// Stride of a dimension; one of extent 1 is never stepped along, whatever the view says.
inline int64_t step_of(const at::Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }

inline void check_same_device(const at::Tensor& t, const at::Device& dev, const char* name) {
    TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", where the pages are");
}

// [n, H, D] fp16 with a contiguous last dimension
inline void check_heads(const at::Tensor& t, int64_t n, int64_t H, int64_t D, const at::Device& dev, const char* name) {
    check_half_cuda(t, name);
    check_same_device(t, dev, name);
    TORCH_CHECK(t.dim() == 3 && t.size(0) == n && t.size(1) == H && t.size(2) == D && (t.stride(2) == 1 || D == 1), name,
                " must be [", n, ", ", H, ", ", D, "] with a contiguous last dimension");
}

inline void bind_scales(const OptTensor& t, int64_t pages, int64_t H, const at::Device& dev, const char* name,
                        uint8_t** ptr, int64_t* sp, int64_t* sh) {
    TORCH_CHECK(given(t), "an e4m3 cache needs ", name);
    TORCH_CHECK(t->is_cuda() && (t->scalar_type() == at::ScalarType::Float8_e8m0fnu || t->scalar_type() == at::kByte),
                name, " must be a float8_e8m0fnu (or uint8) CUDA tensor");
    check_same_device(*t, dev, name);
    TORCH_CHECK(t->dim() == 2 && t->size(0) == pages && t->size(1) == H, name, " must be [num_pages, Hkv]");
    *ptr = static_cast<uint8_t*>(t->data_ptr());
    *sp = step_of(*t, 0);
    *sh = step_of(*t, 1);
}

struct PagedCall {
    fcci_paged_desc d;
    at::Tensor ws;
    PagedCall() { std::memset(&d, 0, sizeof(d)); }
};

inline at::Tensor make_paged_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t total_q,
                                       int64_t max_seqlen_q, int64_t max_kv_tokens, const at::Device& dev) {
    for (int64_t x : {B, Hq, Hkv, D, total_q, max_seqlen_q, max_kv_tokens})
        TORCH_CHECK(x >= 0 && x < ((int64_t)1 << 31), "make_paged_workspace: sizes must fit in int32");
    const size_t bytes = fcci_paged_workspace_bytes((int32_t)B, (int32_t)Hq, (int32_t)Hkv, (int32_t)D, (int32_t)total_q,
                                                    (int32_t)max_seqlen_q, (int32_t)max_kv_tokens, (int)dev.index());
    TORCH_CHECK(bytes > 0, "fcci_paged_workspace_bytes: invalid shape");
    at::Tensor ws = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
    check_rc(fcci_paged_workspace_init(ws.data_ptr(), bytes, current_stream()), "fcci_paged_workspace_init");
    return ws;
}

// The pools, the page table and the lengths, which every call has. B from the page table.
inline void bind_cache(PagedCall& c, const at::Tensor& k_pages, const at::Tensor& v_pages, const OptTensor& k_scales,
                       const OptTensor& v_scales, const at::Tensor& page_table, const at::Tensor& seq_lens) {
    fcci_paged_desc& d = c.d;
    d.abi_version = FCCI_PAGED_ABI_VERSION;
    TORCH_CHECK(k_pages.is_cuda() && v_pages.is_cuda(), "k_pages and v_pages must be CUDA tensors");
    const at::Device dev = k_pages.device();
    const auto type = k_pages.scalar_type();
    TORCH_CHECK(type == at::kHalf || type == at::ScalarType::Float8_e4m3fn, "pages must be fp16 or float8_e4m3fn");
    TORCH_CHECK(v_pages.scalar_type() == type, "k_pages and v_pages must have one type");
    TORCH_CHECK(k_pages.dim() == 4 && v_pages.sizes() == k_pages.sizes(),
                "k_pages and v_pages must be [num_pages, Hkv, page_size, D]");
    TORCH_CHECK(k_pages.stride(3) == 1 && v_pages.stride(3) == 1, "pages must have a contiguous head_dim");
    check_same_device(v_pages, dev, "v_pages");
    TORCH_CHECK(page_table.is_cuda() && page_table.scalar_type() == at::kInt && page_table.dim() == 2,
                "page_table must be an int32 CUDA tensor [B, max_pages]");
    TORCH_CHECK(page_table.size(1) <= 1 || page_table.stride(1) == 1, "page_table rows must be contiguous");
    check_same_device(page_table, dev, "page_table");
    check_int32_cuda(seq_lens, "seq_lens");
    check_same_device(seq_lens, dev, "seq_lens");
    TORCH_CHECK(seq_lens.numel() == page_table.size(0), "seq_lens must have one entry per page_table row");
    for (int64_t x : {k_pages.size(0), k_pages.size(1), page_table.size(0), page_table.size(1)})
        TORCH_CHECK(x > 0 && x < ((int64_t)1 << 31), "empty or oversized pools or page_table");
    d.B = (int32_t)page_table.size(0);
    d.Hkv = (int32_t)k_pages.size(1);
    d.D = (int32_t)std::min<int64_t>(k_pages.size(3), 1 << 20);
    d.page_size = (int32_t)std::min<int64_t>(k_pages.size(2), 1 << 20);
    d.num_pages = (int32_t)k_pages.size(0);
    d.max_pages = (int32_t)page_table.size(1);
    d.k_pages = k_pages.data_ptr();
    d.v_pages = v_pages.data_ptr();
    d.k_stride_p = step_of(k_pages, 0), d.k_stride_h = step_of(k_pages, 1), d.k_stride_t = k_pages.stride(2);
    d.v_stride_p = step_of(v_pages, 0), d.v_stride_h = step_of(v_pages, 1), d.v_stride_t = v_pages.stride(2);
    if (type == at::kHalf) {
        TORCH_CHECK(!given(k_scales) && !given(v_scales), "an fp16 cache has no scales");
        d.cache_type = FCCI_PAGED_F16;
    } else {
        d.cache_type = FCCI_PAGED_E4M3;
        bind_scales(k_scales, d.num_pages, d.Hkv, dev, "k_scales", &d.k_scales, &d.k_scales_stride_p, &d.k_scales_stride_h);
        bind_scales(v_scales, d.num_pages, d.Hkv, dev, "v_scales", &d.v_scales, &d.v_scales_stride_p, &d.v_scales_stride_h);
    }
    d.page_table = page_table.data_ptr<int32_t>();
    d.page_table_stride = step_of(page_table, 0);
    d.seq_lens = seq_lens.data_ptr<int32_t>();
}

inline void bind_new(PagedCall& c, const at::Tensor& k_new, const at::Tensor& v_new, const at::Device& dev) {
    check_heads(k_new, c.d.total_q, c.d.Hkv, c.d.D, dev, "k_new");
    check_heads(v_new, c.d.total_q, c.d.Hkv, c.d.D, dev, "v_new");
    // a call of no tokens has no address to give: the descriptor's never-read pointer stands in
    c.d.k_new = c.d.total_q ? k_new.data_ptr() : c.d.k_pages;
    c.d.k_new_stride_t = step_of(k_new, 0), c.d.k_new_stride_h = step_of(k_new, 1);
    c.d.v_new = c.d.total_q ? v_new.data_ptr() : c.d.v_pages;
    c.d.v_new_stride_t = step_of(v_new, 0), c.d.v_new_stride_h = step_of(v_new, 1);
}

inline void bind_rows(PagedCall& c, int64_t total, const OptTensor& cu, int64_t max_seqlen_q, const at::Device& dev) {
    TORCH_CHECK(total < ((int64_t)1 << 31), "too many tokens");
    c.d.total_q = (int32_t)total;
    if (given(cu)) {
        check_int32_cuda(*cu, "cu_seqlens_q");
        check_same_device(*cu, dev, "cu_seqlens_q");
        TORCH_CHECK(cu->dim() == 1 && cu->numel() == (int64_t)c.d.B + 1, "cu_seqlens_q must have B+1 entries");
        TORCH_CHECK(max_seqlen_q >= 0 && max_seqlen_q < ((int64_t)1 << 31), "cu_seqlens_q needs max_seqlen_q");
        c.d.cu_seqlens_q = cu->data_ptr<int32_t>();
        c.d.max_seqlen_q = (int32_t)max_seqlen_q;
    } else {
        TORCH_CHECK(total == c.d.B, "one new token per sequence (or cu_seqlens_q)");
        c.d.max_seqlen_q = 1;
    }
}

// A caller's workspace, or one made for this call (its memory returns to the caching allocator in stream
// order; under capture it comes from the graph's own pool and is zeroed inside the graph).
inline void bind_paged_workspace(PagedCall& c, const OptTensor& workspace, const at::Device& dev) {
    fcci_paged_desc& d = c.d;
    if (given(workspace)) {
        TORCH_CHECK(workspace->is_cuda() && workspace->scalar_type() == at::kByte && workspace->is_contiguous(),
                    "workspace must be a contiguous uint8 CUDA tensor from make_paged_workspace()");
        check_same_device(*workspace, dev, "workspace");
        c.ws = *workspace;
    } else {
        c.ws = make_paged_workspace(d.B, d.Hq, d.Hkv, d.D, d.total_q, d.max_seqlen_q, d.max_kv_tokens, dev);
    }
    d.workspace = c.ws.data_ptr();
    d.workspace_bytes = (size_t)c.ws.numel();
}

inline void bind_rope(PagedCall& c, double rope_theta, int64_t rotary_dim, bool turn_by_default) {
    c.d.rope_theta = (float)rope_theta;
    const int64_t r = rotary_dim < 0 ? (turn_by_default ? c.d.D : 0) : rotary_dim;
    c.d.rotary_dim = (int32_t)std::min<int64_t>(r, 1 << 20);
}

inline void paged_append(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& k_pages,
                         const at::Tensor& v_pages, const at::Tensor& page_table, const at::Tensor& seq_lens,
                         const OptTensor& k_scales, const OptTensor& v_scales, const OptTensor& q,
                         const OptTensor& q_rot_out, const OptTensor& cu_seqlens_q, int64_t max_seqlen_q,
                         double rope_theta, int64_t rotary_dim, bool advance, const OptTensor& workspace) {
    PagedCall c;
    bind_cache(c, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens);
    const at::Device dev = k_pages.device();
    TORCH_CHECK(k_new.dim() == 3, "k_new must be [tokens, Hkv, D]");
    bind_rows(c, k_new.size(0), cu_seqlens_q, max_seqlen_q, dev);
    bind_new(c, k_new, v_new, dev);
    c.d.Hq = c.d.Hkv;
    TORCH_CHECK(given(q) == given(q_rot_out), "q and q_rot_out go together");
    c10::cuda::CUDAGuard guard(dev);
    if (given(q) && c.d.total_q) {
        TORCH_CHECK(q->dim() == 3 && q->size(1) > 0 && q->size(1) < 65536, "q must be [tokens, Hq, D]");
        c.d.Hq = (int32_t)q->size(1);
        check_heads(*q, c.d.total_q, c.d.Hq, c.d.D, dev, "q");
        check_rows(*q_rot_out, q->numel(), "q_rot_out");
        check_same_device(*q_rot_out, dev, "q_rot_out");
        c.d.q = q->data_ptr();
        c.d.q_stride_t = step_of(*q, 0), c.d.q_stride_h = step_of(*q, 1);
        c.d.q_rot_out = q_rot_out->data_ptr();
    }
    bind_rope(c, rope_theta, rotary_dim, true);
    c.d.advance = advance ? 1 : 0;
    bind_paged_workspace(c, workspace, dev);
    check_rc(fcci_paged_append(&c.d, current_stream()), "attn_varlen.paged_append");
}

// q, out and the scale of an attention call
inline void bind_attention(PagedCall& c, const at::Tensor& q, const at::Tensor& out, double scale, const at::Device& dev) {
    c.d.Hq = (int32_t)std::min<int64_t>(q.size(1), 1 << 20);
    check_heads(q, c.d.total_q, c.d.Hq, c.d.D, dev, "q");
    check_heads(out, c.d.total_q, c.d.Hq, c.d.D, dev, "out");
    c.d.q = c.d.total_q ? q.data_ptr() : c.d.k_pages;
    c.d.q_stride_t = step_of(q, 0), c.d.q_stride_h = step_of(q, 1);
    c.d.out = c.d.total_q ? out.data_ptr() : c.d.k_pages;
    c.d.out_stride_t = step_of(out, 0), c.d.out_stride_h = step_of(out, 1);
    c.d.scale = scale > 0 ? (float)scale : (float)(1.0 / std::sqrt((double)c.d.D));
}

inline void paged_decode(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& out,
                         const at::Tensor& page_table, const at::Tensor& seq_lens, const OptTensor& k_scales,
                         const OptTensor& v_scales, const OptTensor& k_new, const OptTensor& v_new, double scale,
                         double rope_theta, int64_t rotary_dim, bool advance, const OptTensor& q_rot_out,
                         const OptTensor& workspace, bool prefetch_kv) {
    PagedCall c;
    bind_cache(c, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens);
    const at::Device dev = k_pages.device();
    TORCH_CHECK(q.dim() == 3, "q must be [B, Hq, D]");
    bind_rows(c, q.size(0), c10::nullopt, 1, dev);
    bind_attention(c, q, out, scale, dev);
    TORCH_CHECK(given(k_new) == given(v_new), "k_new and v_new go together");
    if (given(k_new)) bind_new(c, *k_new, *v_new, dev);
    TORCH_CHECK(!advance || given(k_new), "advance needs k_new and v_new");
    c10::cuda::CUDAGuard guard(dev);
    if (given(q_rot_out)) {
        check_rows(*q_rot_out, q.numel(), "q_rot_out");
        check_same_device(*q_rot_out, dev, "q_rot_out");
        c.d.q_rot_out = q_rot_out->data_ptr();
    }
    bind_rope(c, rope_theta, rotary_dim, given(k_new));
    c.d.advance = advance ? 1 : 0;
    bind_paged_workspace(c, workspace, dev);
    c.d.flags = prefetch_kv ? FCCI_PAGED_PREFETCH_KV : 0u;
    check_rc(fcci_paged_decode(&c.d, current_stream()), "attn_varlen.paged_decode");
}

inline void paged_prefill(const at::Tensor& q, const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& k_pages,
                          const at::Tensor& v_pages, const at::Tensor& out, const at::Tensor& page_table,
                          const at::Tensor& seq_lens, const at::Tensor& cu_seqlens_q, int64_t max_seqlen_q,
                          const OptTensor& k_scales, const OptTensor& v_scales, double scale, double rope_theta,
                          int64_t rotary_dim, bool advance, int64_t max_kv_tokens, const OptTensor& workspace) {
    PagedCall c;
    bind_cache(c, k_pages, v_pages, k_scales, v_scales, page_table, seq_lens);
    const at::Device dev = k_pages.device();
    TORCH_CHECK(q.dim() == 3, "q must be [tokens, Hq, D]");
    bind_rows(c, q.size(0), cu_seqlens_q, max_seqlen_q, dev);
    bind_attention(c, q, out, scale, dev);
    bind_new(c, k_new, v_new, dev);
    bind_rope(c, rope_theta, rotary_dim, true);
    c.d.advance = advance ? 1 : 0;
    // without a bound: what the given workspace has room for, or every row of the page table
    int64_t kv = max_kv_tokens;
    if (kv < 0) kv = given(workspace) ? -1 : (int64_t)c.d.B * c.d.max_pages * c.d.page_size;
    TORCH_CHECK(kv < ((int64_t)1 << 31), "give max_kv_tokens (a bound on the keys of all sequences) below 2^31");
    c.d.max_kv_tokens = (int32_t)kv;
    c10::cuda::CUDAGuard guard(dev);
    bind_paged_workspace(c, workspace, dev);
    check_rc(fcci_paged_prefill(&c.d, current_stream()), "attn_varlen.paged_prefill");
}

inline int64_t paged_read_error(const at::Tensor& workspace, bool clear) {
    TORCH_CHECK(workspace.is_cuda() && workspace.scalar_type() == at::kByte, "workspace must be a uint8 CUDA tensor");
    c10::cuda::CUDAGuard guard(workspace.device());
    uint32_t flags = 0;
    check_rc(fcci_paged_read_error(workspace.data_ptr(), &flags, clear ? 1 : 0, current_stream()),
             "attn_varlen.paged_read_error");
    return (int64_t)flags;
}

inline void def_paged(py::module& m) {
    m.def("paged_append", &paged_append,
          "RoPE on k_new (and q) at T_b + i and append of k/v into the pages of a paged cache (no attention)",
          py::arg("k_new"), py::arg("v_new"), py::arg("k_pages"), py::arg("v_pages"), py::arg("page_table"),
          py::arg("seq_lens"), py::kw_only(), py::arg("k_scales") = py::none(), py::arg("v_scales") = py::none(),
          py::arg("q") = py::none(), py::arg("q_rot_out") = py::none(), py::arg("cu_seqlens_q") = py::none(),
          py::arg("max_seqlen_q") = -1, py::arg("rope_theta") = 10000.0, py::arg("rotary_dim") = -1,
          py::arg("advance") = false, py::arg("workspace") = py::none());
    m.def("paged_decode", &paged_decode,
          "Decode step over a paged cache: RoPE(q,k_new) at T, append at T, split-KV GQA attention over T+1 keys",
          py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("out"), py::arg("page_table"),
          py::arg("seq_lens"), py::kw_only(), py::arg("k_scales") = py::none(), py::arg("v_scales") = py::none(),
          py::arg("k_new") = py::none(), py::arg("v_new") = py::none(), py::arg("scale") = -1.0,
          py::arg("rope_theta") = 10000.0, py::arg("rotary_dim") = -1, py::arg("advance") = false,
          py::arg("q_rot_out") = py::none(), py::arg("workspace") = py::none(), py::arg("prefetch_kv") = false);
    m.def("paged_prefill", &paged_prefill,
          "Prompts (or chunks) over a paged cache: RoPE(q,k_new) at T_b+i, append, causal attention over T_b+n_b keys",
          py::arg("q"), py::arg("k_new"), py::arg("v_new"), py::arg("k_pages"), py::arg("v_pages"), py::arg("out"),
          py::arg("page_table"), py::arg("seq_lens"), py::arg("cu_seqlens_q"), py::arg("max_seqlen_q"), py::kw_only(),
          py::arg("k_scales") = py::none(), py::arg("v_scales") = py::none(), py::arg("scale") = -1.0,
          py::arg("rope_theta") = 10000.0, py::arg("rotary_dim") = -1, py::arg("advance") = false,
          py::arg("max_kv_tokens") = -1, py::arg("workspace") = py::none());
    m.def(
        "make_paged_workspace",
        [](int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t total_q, int64_t max_seqlen_q, int64_t max_kv_tokens,
           c10::optional<at::Device> device) {
            at::Device dev = device.has_value() ? *device : at::Device(at::kCUDA, c10::cuda::current_device());
            if (!dev.has_index()) dev = at::Device(at::kCUDA, c10::cuda::current_device());
            c10::cuda::CUDAGuard guard(dev);
            return make_paged_workspace(B, Hq, Hkv, D, total_q, max_seqlen_q, max_kv_tokens, dev);
        },
        "Zeroed workspace for the paged calls of up to total_q new tokens (allocate outside graph capture); "
        "max_kv_tokens bounds the keys of all sequences in a paged_prefill",
        py::arg("B"), py::arg("Hq"), py::arg("Hkv"), py::arg("D"), py::arg("total_q"), py::arg("max_seqlen_q") = 1,
        py::arg("max_kv_tokens") = 0, py::arg("device") = py::none());
    m.def("paged_read_error", &paged_read_error, "Device error word of a paged workspace (synchronises)",
          py::arg("workspace"), py::arg("clear") = true);
}

}  // namespace fcci_py
