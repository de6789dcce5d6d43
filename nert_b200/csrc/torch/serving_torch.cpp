// torch binding of the serving rows: argument checks, output tensors and the
// call of the C ABI (include/nert_b200.h) on torch's current stream.
//
// The smallest serving calls run for a few microseconds on the GPU, so what a
// call costs on the host counts: checked and launched from here a call takes
// about a third of what the same checks take through ctypes. The library itself
// has no torch dependency; this file is a module of its own.

#include "../../../include/nert_b200.h"

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void raise(int status) {
    py::object cls = py::module_::import("nert_b200._lib").attr("NB2Error");
    PyErr_SetObject(cls.ptr(), cls(status, nb2_last_error()).ptr());
    throw py::error_already_set();
}

void check(int status) {
    if (status != NB2_OK) {
        raise(status);
    }
}

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

// The GPU of a call, with its index.
c10::Device gpu(c10::Device device) {
    NEED(device.is_cuda(), "expected tensors on a GPU");
    return device.has_index() ? device : c10::Device(c10::kCUDA, c10::cuda::current_device());
}

// The library makes a context's GPU current for the thread. Every function that
// Python calls holds one of these, so that torch's current GPU is the caller's again after it.
using OnGpu = c10::cuda::CUDAGuard;

// The context of torch's current stream on the tensor's GPU, made on first use
// and kept: torch hands out streams from fixed pools.
nb2_device* context(c10::Device device) {
    const c10::cuda::CUDAStream s = c10::cuda::getCurrentCUDAStream(device.index());
    struct Entry {
        int device;
        cudaStream_t stream;
        nb2_device* dev;
    };
    static std::vector<Entry> known; // under the interpreter's lock
    for (const Entry& e : known) {
        if (e.stream == s.stream() && e.device == s.device_index()) {
            return e.dev;
        }
    }
    nb2_device* dev = nullptr;
    check(nb2_device_on_stream(s.device_index(), s.stream(), &dev));
    known.push_back({s.device_index(), s.stream(), dev});
    return dev;
}

int dtype_code(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
    case at::kFloat:
        return NB2_F32;
    case at::kHalf:
        return NB2_F16;
    case at::kBFloat16:
        return NB2_BF16;
    default:
        NEED(false, name, ": the type must be float32, float16 or bfloat16");
    }
    return -1;
}

// Contiguous int32 data on `device`; null for none.
const int32_t* ints(const OptTensor& t, const char* name, c10::Device device, int64_t dim = 1) {
    if (!t.has_value()) {
        return nullptr;
    }
    NEED(t->scalar_type() == at::kInt && t->dim() == dim && t->device() == device && t->is_contiguous(), name,
         ": expected a contiguous ", dim, "-d int32 tensor on the GPU of the others");
    return static_cast<const int32_t*>(t->data_ptr());
}

const float* floats(const OptTensor& t, const char* name, c10::Device device, int64_t n) {
    if (!t.has_value()) {
        return nullptr;
    }
    NEED(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n && t->device() == device &&
             t->is_contiguous(),
         name, ": expected ", n, " contiguous float32 values on the GPU of the others");
    return static_cast<const float*>(t->data_ptr());
}

// [tokens, heads, dim] of q's type with contiguous heads.
void heads(const Tensor& t, const char* name, const Tensor& q) {
    NEED(t.dim() == 3 && t.size(0) == q.size(0) && t.size(2) == q.size(2) && t.scalar_type() == q.scalar_type() &&
             t.device() == q.device(),
         name, ": expected [", q.size(0), ", heads, ", q.size(2), "] of q's type on its GPU");
    NEED(t.stride(2) == 1 || t.size(2) == 1, name, ": a head's elements must be contiguous");
}

void caches(const Tensor& k, const Tensor& v, const Tensor& q, int64_t kv_heads) {
    for (const Tensor* c : {&k, &v}) {
        const char* name = c == &k ? "k_cache" : "v_cache";
        NEED(c->dim() == 4 && c->size(2) == kv_heads && c->size(3) == q.size(2) && c->scalar_type() == q.scalar_type() &&
                 c->device() == q.device(),
             name, ": expected [blocks, block_size, ", kv_heads, ", ", q.size(2), "] of q's type on its GPU");
        NEED(c->stride(3) == 1 || c->size(3) == 1, name, ": a head's elements must be contiguous");
    }
    NEED(k.sizes() == v.sizes(), "k_cache and v_cache differ in shape");
}

// The address of a [batch, blocks] table, and its row stride.
int32_t* block_table(const Tensor& t, int64_t batch, c10::Device device, int64_t& stride) {
    NEED(t.dim() == 2 && t.size(0) == batch && t.scalar_type() == at::kInt && t.device() == device &&
             (t.stride(1) == 1 || t.size(1) <= 1),
         "block_table: expected [", batch, ", blocks] int32 on the GPU of the others");
    stride = batch > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1));
    return static_cast<int32_t*>(t.data_ptr());
}

void* address(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

std::tuple<Tensor, Tensor, Tensor, Tensor, OptTensor, Tensor>
page_plan(const Tensor& seq_lens, const Tensor& new_lens, const Tensor& table, const Tensor& free_blocks,
          int64_t block_size, int64_t tokens, const OptTensor& parents, int64_t mask_words, const OptTensor& free_head) {
    const c10::Device on = gpu(seq_lens.device());
    const OnGpu guard(on);
    nb2_device* dev = context(on);
    const int32_t* old = ints(seq_lens, "seq_lens", on);
    const int32_t* fresh = ints(new_lens, "new_lens", on);
    const int32_t* pool = ints(free_blocks, "free_blocks", on);
    const int32_t* head = ints(free_head, "free_head", on);
    const int32_t* up = ints(parents, "parents", on);
    const int64_t batch = seq_lens.size(0);
    NEED(tokens >= 0, "tokens: negative");
    NEED(new_lens.size(0) == batch, "new_lens and seq_lens differ in length");
    NEED(head == nullptr || free_head->size(0) == 1, "free_head: expected one value");
    NEED(!parents.has_value() || parents->size(0) >= tokens, "parents: fewer than tokens");
    NEED(parents.has_value() == (mask_words > 0), "parents and mask_words come together");
    nb2_page_plan_geom g{};
    int32_t* t = block_table(table, batch, on, g.table_stride);
    g.batch = batch;
    g.tokens = tokens;
    g.block_size = block_size;
    g.table_blocks = table.size(1);
    g.free_blocks = free_blocks.size(0);
    g.mask_words = mask_words;
    // one allocation, cut: the outputs are small and a step has many of them
    const int64_t words = parents.has_value() ? mask_words : 0;
    const auto pad = [](int64_t n) { return (n + 3) / 4 * 4; };
    const int64_t at_total = 4, at_off = at_total + pad(batch), at_slot = at_off + pad(batch + 1),
                  at_pos = at_slot + pad(tokens), at_mask = at_pos + pad(tokens),
                  all = at_mask + tokens * words + 4;
    const Tensor buf = at::empty({all}, seq_lens.options());
    int32_t* b = static_cast<int32_t*>(buf.data_ptr());
    if (parents.has_value() && up == nullptr) {
        up = b; // no token is new: never read
    }
    check(nb2_page_plan(dev, &g, old, fresh, pool, head, up, t, b + at_total, b + at_off, b, b + at_slot, b + at_pos,
                        words > 0 ? b + at_mask : nullptr));
    OptTensor mask;
    if (words > 0) {
        mask = buf.as_strided({tokens, words}, {words, 1}, at_mask);
    }
    return {buf.as_strided({batch}, {1}, at_total), buf.as_strided({batch + 1}, {1}, at_off),
            buf.as_strided({tokens}, {1}, at_slot), buf.as_strided({tokens}, {1}, at_pos), mask,
            buf.as_strided({1}, {1}, 0)};
}

// axis_of as the bytes of one axis a frequency, its largest + 1 in axes
std::tuple<Tensor, OptTensor> rope_append(const Tensor& q, const Tensor& k, const OptTensor& v, const Tensor& table,
                                          const Tensor& positions, const std::optional<py::bytes>& axis_of, int axes,
                                          bool interleaved, const OptTensor& slots, const OptTensor& k_cache,
                                          const OptTensor& v_cache, const OptTensor& q_out, const OptTensor& k_out) {
    const c10::Device on = gpu(q.device());
    const OnGpu guard(on);
    nb2_device* dev = context(on);
    NEED(q.dim() == 3, "q: expected [tokens, heads, head_dim]");
    nb2_rope_geom g{};
    g.dtype = dtype_code(q, "q");
    heads(q, "q", q);
    heads(k, "k", q);
    g.tokens = q.size(0);
    g.q_heads = q.size(1);
    g.kv_heads = k.size(1);
    g.head_dim = q.size(2);
    NEED(table.dim() == 2 && table.scalar_type() == at::kFloat && table.is_contiguous() && table.device() == on,
         "table: expected contiguous [length, rot_dim] float32 on the GPU of the others");
    g.table_len = table.size(0);
    g.rot_dim = table.size(1);
    g.axes = axes;
    if (axis_of.has_value()) {
        char* bytes = nullptr;
        Py_ssize_t n = 0;
        PyBytes_AsStringAndSize(axis_of->ptr(), &bytes, &n);
        NEED(n == g.rot_dim / 2 && n <= 256, "axis_of: expected ", g.rot_dim / 2, " frequencies (at most 256)");
        std::copy(bytes, bytes + n, g.axis_of);
    }
    if (positions.dim() == 1) {
        NEED(axes == 1 && positions.size(0) >= g.tokens, "positions: expected one row of tokens for each axis");
        ints(positions, "positions", on);
    } else {
        NEED(positions.dim() == 2 && positions.size(0) >= axes && positions.size(1) >= g.tokens &&
                 positions.scalar_type() == at::kInt && positions.device() == on &&
                 (positions.stride(1) == 1 || positions.size(1) <= 1),
             "positions: expected [axes, tokens] int32 on the GPU of the others");
        g.axis_stride = positions.stride(0);
    }
    const bool cached = k_cache.has_value();
    if (cached) {
        NEED(v.has_value() && v_cache.has_value() && slots.has_value(), "a cache needs v, v_cache and slots");
        heads(*v, "v", q);
        NEED(v->size(1) == g.kv_heads, "v: heads differ from k's");
        caches(*k_cache, *v_cache, q, g.kv_heads);
        NEED(slots->dim() == 1 && slots->size(0) >= g.tokens, "slots: fewer than tokens");
        g.v_stride = v->stride(0);
        g.v_head_stride = v->stride(1);
        g.num_blocks = k_cache->size(0);
        g.block_size = k_cache->size(1);
        g.kc_block_stride = k_cache->stride(0);
        g.kc_place_stride = k_cache->stride(1);
        g.kc_head_stride = k_cache->stride(2);
        g.vc_block_stride = v_cache->stride(0);
        g.vc_place_stride = v_cache->stride(1);
        g.vc_head_stride = v_cache->stride(2);
    } else {
        NEED(!v.has_value() && !v_cache.has_value() && !slots.has_value(), "v and slots belong to a cache");
    }
    const Tensor qo = q_out.has_value() ? *q_out : at::empty({g.tokens, g.q_heads, g.head_dim}, q.options());
    OptTensor ko = k_out;
    if (!ko.has_value() && !cached) {
        ko = at::empty({g.tokens, g.kv_heads, g.head_dim}, q.options());
    }
    heads(qo, "q_out", q);
    NEED(qo.size(1) == g.q_heads, "q_out: heads differ from q's");
    if (ko.has_value()) {
        heads(*ko, "k_out", q);
        NEED(ko->size(1) == g.kv_heads, "k_out: heads differ from k's");
        g.ko_stride = ko->stride(0);
        g.ko_head_stride = ko->stride(1);
    }
    g.q_stride = q.stride(0);
    g.q_head_stride = q.stride(1);
    g.k_stride = k.stride(0);
    g.k_head_stride = k.stride(1);
    g.qo_stride = qo.stride(0);
    g.qo_head_stride = qo.stride(1);
    g.interleaved = interleaved ? 1 : 0;
    if (g.tokens > 0) {
        check(nb2_rope_append(dev, &g, q.data_ptr(), k.data_ptr(), address(v), static_cast<const float*>(table.data_ptr()),
                              static_cast<const int32_t*>(positions.data_ptr()), ints(slots, "slots", on), qo.data_ptr(),
                              address(ko), address(k_cache), address(v_cache)));
    }
    return {qo, ko};
}

std::tuple<Tensor, OptTensor> tree_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                             const Tensor& table, const Tensor& seq_lens, const Tensor& token_offsets,
                                             const OptTensor& tree_mask, std::optional<int64_t> max_new,
                                             std::optional<double> scale, bool return_lse, const OptTensor& out) {
    const c10::Device on = gpu(q.device());
    const OnGpu guard(on);
    nb2_device* dev = context(on);
    NEED(q.dim() == 3, "q: expected [tokens, heads, head_dim]");
    nb2_tree_attn_geom g{};
    g.dtype = dtype_code(q, "q");
    heads(q, "q", q);
    NEED(k_cache.dim() == 4, "k_cache: expected [blocks, block_size, heads, head_dim]");
    g.kv_heads = k_cache.size(2);
    caches(k_cache, v_cache, q, g.kv_heads);
    const int32_t* total = ints(seq_lens, "seq_lens", on);
    const int32_t* offsets = ints(token_offsets, "token_offsets", on);
    const int32_t* mask = ints(tree_mask, "tree_mask", on, 2);
    g.batch = seq_lens.size(0);
    NEED(token_offsets.size(0) == g.batch + 1, "token_offsets: expected batch + 1 values");
    const int32_t* t = block_table(table, g.batch, on, g.table_stride);
    g.tokens = q.size(0);
    g.q_heads = q.size(1);
    g.head_dim = q.size(2);
    if (tree_mask.has_value()) {
        NEED(tree_mask->size(0) >= g.tokens && tree_mask->size(1) > 0, "tree_mask: expected [tokens, words]");
        g.mask_words = tree_mask->size(1);
    }
    g.max_new = max_new.value_or(g.tokens);
    g.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(g.head_dim)));
    const Tensor o = out.has_value() ? *out : at::empty({g.tokens, g.q_heads, g.head_dim}, q.options());
    heads(o, "out", q);
    NEED(o.size(1) == g.q_heads, "out: heads differ from q's");
    OptTensor lse;
    if (return_lse) {
        lse = at::empty({g.tokens, g.q_heads}, q.options().dtype(at::kFloat));
    }
    g.q_stride = q.stride(0);
    g.q_head_stride = q.stride(1);
    g.o_stride = o.stride(0);
    g.o_head_stride = o.stride(1);
    g.num_blocks = k_cache.size(0);
    g.block_size = k_cache.size(1);
    g.table_blocks = table.size(1);
    g.kc_block_stride = k_cache.stride(0);
    g.kc_place_stride = k_cache.stride(1);
    g.kc_head_stride = k_cache.stride(2);
    g.vc_block_stride = v_cache.stride(0);
    g.vc_place_stride = v_cache.stride(1);
    g.vc_head_stride = v_cache.stride(2);
    if (g.tokens > 0) {
        check(nb2_tree_attention(dev, &g, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), t, total, offsets, mask,
                                 o.data_ptr(), static_cast<float*>(address(lse))));
    }
    return {o, lse};
}

// The library takes a null list or mask for none. One that is given and holds nothing has no address of its own: it gets
// another's, so that what points into it (offsets, rows) is checked against its count, 0, and nothing is read from it.
template <typename T>
const T* given(const T* p, const void* other) {
    return p != nullptr ? p : static_cast<const T*>(other);
}

using List = std::optional<std::tuple<Tensor, Tensor>>;

void list(const List& l, const char* name, c10::Device on, int64_t requests, const int32_t*& ids, const int32_t*& offsets,
          int64_t& count) {
    if (l.has_value()) {
        offsets = ints(std::get<1>(*l), name, on);
        ids = given(ints(std::get<0>(*l), name, on), offsets);
        NEED(std::get<1>(*l).size(0) == requests + 1, name, ": expected requests + 1 offsets");
        count = std::get<0>(*l).size(0);
    }
}

Tensor logits_process(const Tensor& logits, const List& prompt, const List& output, const OptTensor& row_request,
                      const OptTensor& repetition, const OptTensor& presence, const OptTensor& frequency,
                      const std::optional<std::tuple<Tensor, Tensor, Tensor>>& bias,
                      const std::optional<std::tuple<Tensor, OptTensor>>& grammar, std::optional<at::ScalarType> out_dtype,
                      const OptTensor& out, std::optional<int64_t> n_requests) {
    const c10::Device on = gpu(logits.device());
    const OnGpu guard(on);
    nb2_device* dev = context(on);
    NEED(logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1), "logits: expected [rows, vocab]");
    nb2_logits_geom g{};
    g.rows = logits.size(0);
    g.vocab = logits.size(1);
    g.in_dtype = dtype_code(logits, "logits");
    Tensor o;
    if (out.has_value()) {
        o = *out;
        NEED(o.sizes() == logits.sizes() && o.device() == on && (g.vocab <= 1 || o.stride(1) == 1) &&
                 (!out_dtype.has_value() || o.scalar_type() == *out_dtype),
             "out: expected the logits' shape on their GPU");
    } else {
        o = at::empty({g.rows, g.vocab}, logits.options().dtype(out_dtype.value_or(logits.scalar_type())));
    }
    g.out_dtype = dtype_code(o, "out");
    int64_t requests = g.rows;
    if (n_requests.has_value()) {
        requests = *n_requests;
    } else {
        for (const OptTensor* t : {&repetition, &presence, &frequency}) {
            if (t->has_value() && (*t)->dim() == 1) {
                requests = (*t)->size(0);
            }
        }
        for (const List* l : {&prompt, &output}) {
            if (l->has_value() && std::get<1>(**l).dim() == 1) {
                requests = std::get<1>(**l).size(0) - 1;
            }
        }
        if (bias.has_value() && std::get<2>(*bias).dim() == 1) {
            requests = std::get<2>(*bias).size(0) - 1;
        }
    }
    NEED(row_request.has_value() || requests >= g.rows || g.rows == 0, "row_request: rows and requests differ");
    const int32_t* rr = ints(row_request, "row_request", on);
    NEED(!row_request.has_value() || row_request->size(0) == g.rows, "row_request: expected one request a row");
    g.requests = requests;
    const int32_t *p_ids = nullptr, *p_off = nullptr, *o_ids = nullptr, *o_off = nullptr, *b_ids = nullptr,
                  *b_off = nullptr, *m = nullptr, *m_rows = nullptr;
    const float* b_val = nullptr;
    list(prompt, "prompt", on, requests, p_ids, p_off, g.prompt_count);
    list(output, "output", on, requests, o_ids, o_off, g.output_count);
    if (bias.has_value()) {
        list(std::make_tuple(std::get<0>(*bias), std::get<2>(*bias)), "bias", on, requests, b_ids, b_off, g.bias_count);
        b_val = given(floats(std::get<1>(*bias), "bias values", on, g.bias_count), b_off);
    }
    if (grammar.has_value()) {
        const Tensor& mask = std::get<0>(*grammar);
        const OptTensor& rows = std::get<1>(*grammar);
        NEED(mask.dim() == 2 && mask.scalar_type() == at::kInt && mask.device() == on &&
                 (mask.size(1) <= 1 || mask.stride(1) == 1) && mask.size(1) * 32 >= g.vocab,
             "grammar: expected [n, ceil(vocab / 32)] int32 words on the GPU of the others");
        NEED(!rows.has_value() || (rows->dim() == 1 && rows->size(0) == g.rows), "grammar rows: expected one a row");
        m = given(static_cast<const int32_t*>(mask.data_ptr()), logits.data_ptr());
        m_rows = ints(rows, "grammar rows", on);
        g.grammar_count = mask.size(0);
        g.grammar_stride = mask.size(0) > 1 ? mask.stride(0) : mask.size(1);
    }
    g.in_stride = logits.stride(0);
    g.out_stride = o.stride(0);
    check(nb2_logits_process(dev, &g, logits.data_ptr(), o.data_ptr(), rr, p_ids, p_off, o_ids, o_off,
                             floats(repetition, "repetition", on, requests), floats(presence, "presence", on, requests),
                             floats(frequency, "frequency", on, requests), b_ids, b_val, b_off, m, m_rows));
    return o;
}

void synchronize(c10::Device device) {
    const c10::Device on = gpu(device);
    const OnGpu guard(on);
    nb2_device* dev = context(on);
    int status;
    {
        py::gil_scoped_release free; // other threads run while this one waits
        status = nb2_device_synchronize(dev);
    }
    check(status);
}

int64_t context_address(c10::Device device) {
    const c10::Device on = gpu(device);
    const OnGpu guard(on);
    return reinterpret_cast<int64_t>(context(on));
}

} // namespace

PYBIND11_MODULE(nert_b200_torch, m) {
    m.def("page_plan", &page_plan);
    m.def("rope_append", &rope_append);
    m.def("tree_attention", &tree_attention);
    m.def("logits_process", &logits_process);
    m.def("synchronize", &synchronize);
    m.def("context", &context_address);
}
