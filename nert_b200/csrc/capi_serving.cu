// extern "C" entry points of the serving rows (include/nert_b200.h): what the
// host can check is checked here, then the row is launched on the device's
// stream. C++ exceptions never cross the boundary.

#include "serving.cuh"

#include <cmath>
#include <new>
#include <string>

using namespace nb2;

namespace {

template <typename F>
int guard(F&& f) {
    try {
        f();
        return NB2_OK;
    } catch (const Error& e) {
        set_last_error(e.what());
        return e.code;
    } catch (const std::bad_alloc&) {
        set_last_error("out of host memory");
        return NB2_ERR_NOMEM;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return NB2_ERR_INVALID;
    }
}

void need(bool ok, const char* msg) {
    if (!ok) {
        fail(kStatusInvalid, msg);
    }
}

void bind(nb2_device* dev) {
    need(dev != nullptr, "null device");
    dev->make_current();
}

bool float_type(int dtype) { return dtype == kF32 || dtype == kF16 || dtype == kBF16; }

constexpr int64_t kMaxI32 = 0x7fffffff;

bool in_i32(int64_t v) { return v >= 0 && v <= kMaxI32; }

// The stride of a dimension of one element says nothing, whatever it is: a caller's views may hold any. It becomes a
// head's length, which every check of alignment allows.
void level(int64_t extent, int64_t& stride, int64_t head_dim) {
    if (extent <= 1) {
        stride = head_dim;
    }
}

} // namespace

extern "C" {

int nb2_page_plan(nb2_device* dev, const nb2_page_plan_geom* g, const int32_t* seq_lens, const int32_t* new_lens,
                  const int32_t* free_blocks, const int32_t* free_head, const int32_t* parents, int32_t* block_table,
                  int32_t* new_total, int32_t* token_offsets, int32_t* free_head_out, int32_t* slots,
                  int32_t* positions, int32_t* tree_mask) {
    return guard([&] {
        need(g != nullptr, "PagePlan: null geometry");
        need(in_i32(g->tokens) && in_i32(g->free_blocks) && in_i32(g->table_blocks), "PagePlan: bad extents");
        need(g->batch >= 0, "PagePlan: negative batch");
        if (g->batch > kPlanMaxBatch) {
            fail(kStatusUnsupported, "PagePlan: at most 8192 requests");
        }
        need(g->block_size > 0 && g->block_size <= kMaxI32, "PagePlan: the block size must be positive");
        need(g->table_stride >= g->table_blocks, "PagePlan: table rows overlap");
        need(g->mask_words >= 0, "PagePlan: negative mask width");
        if (g->mask_words > kPlanMaxWords) {
            fail(kStatusUnsupported, "PagePlan: at most 1024 drafted tokens a request");
        }
        need((parents != nullptr) == (g->mask_words > 0), "PagePlan: parents and a tree mask come together");
        need((parents != nullptr) == (tree_mask != nullptr), "PagePlan: parents and a tree mask come together");
        need(token_offsets != nullptr && free_head_out != nullptr, "PagePlan: null buffer");
        need(g->batch == 0 || (seq_lens && new_lens && new_total), "PagePlan: null buffer");
        need(g->batch == 0 || g->table_blocks == 0 || block_table != nullptr, "PagePlan: null buffer");
        need(g->tokens == 0 || (slots && positions), "PagePlan: null buffer");
        need(g->free_blocks == 0 || free_blocks != nullptr, "PagePlan: null buffer");
        need(new_total != seq_lens || g->batch == 0, "PagePlan: new_total may not be seq_lens");
        need(free_head_out != free_head, "PagePlan: free_head_out may not be free_head");
        bind(dev);
        page_plan(dev, PagePlanArgs{*g, seq_lens, new_lens, free_blocks, free_head, parents, block_table, new_total,
                                    token_offsets, free_head_out, slots, positions,
                                    reinterpret_cast<uint32_t*>(tree_mask), nullptr});
    });
}

int nb2_rope_append(nb2_device* dev, const nb2_rope_geom* g, const void* q, const void* k, const void* v,
                    const float* table, const int32_t* positions, const int32_t* slots, void* q_out, void* k_out,
                    void* k_cache, void* v_cache) {
    return guard([&] {
        need(g != nullptr, "RopeAppend: null geometry");
        need(in_i32(g->tokens), "RopeAppend: bad token count");
        need(float_type(g->dtype), "RopeAppend: the type must be float32, float16 or bfloat16");
        need(g->q_heads > 0 && g->kv_heads > 0 && g->q_heads <= 65535 && g->kv_heads <= 65535,
             "RopeAppend: between 1 and 65535 heads");
        need(g->head_dim > 0 && g->head_dim % 2 == 0, "RopeAppend: the head dimension must be even");
        need(g->rot_dim > 0 && g->rot_dim % 2 == 0 && g->rot_dim <= g->head_dim,
             "RopeAppend: the rotated part must be even and within the head");
        if (g->head_dim > 512) {
            fail(kStatusUnsupported, "RopeAppend: at most 512 elements a head");
        }
        need(g->axes >= 1 && g->axes <= 8, "RopeAppend: between 1 and 8 axes");
        for (int64_t f = 0; f < g->rot_dim / 2; ++f) {
            need(g->axis_of[f] < g->axes, "RopeAppend: a frequency's axis is out of range");
        }
        need(in_i32(g->table_len) && g->table_len > 0, "RopeAppend: the table is empty");
        if (g->tokens == 0) {
            return;
        }
        need(q && k && table && positions && q_out, "RopeAppend: null buffer");
        need((k_cache != nullptr) == (v_cache != nullptr) && (k_cache != nullptr) == (v != nullptr) &&
                 (k_cache != nullptr) == (slots != nullptr),
             "RopeAppend: v, slots and both caches come together");
        need(k_cache != nullptr || k_out != nullptr, "RopeAppend: the keys have nowhere to go");
        need(k_cache == nullptr || (g->block_size > 0 && g->block_size <= kMaxI32 && in_i32(g->num_blocks)),
             "RopeAppend: bad cache extents");
        nb2_rope_geom e = *g;
        for (int64_t* s : {&e.q_stride, &e.k_stride, &e.v_stride, &e.qo_stride, &e.ko_stride}) {
            level(g->tokens, *s, g->head_dim);
        }
        for (int64_t* s : {&e.q_head_stride, &e.qo_head_stride}) {
            level(g->q_heads, *s, g->head_dim);
        }
        for (int64_t* s : {&e.k_head_stride, &e.v_head_stride, &e.ko_head_stride, &e.kc_head_stride, &e.vc_head_stride}) {
            level(g->kv_heads, *s, g->head_dim);
        }
        for (int64_t* s : {&e.kc_block_stride, &e.vc_block_stride}) {
            level(g->num_blocks, *s, g->head_dim);
        }
        for (int64_t* s : {&e.kc_place_stride, &e.vc_place_stride}) {
            level(g->block_size, *s, g->head_dim);
        }
        need(q_out != q || (e.qo_stride == e.q_stride && e.qo_head_stride == e.q_head_stride),
             "RopeAppend: in place needs equal strides");
        need(k_out != k || (e.ko_stride == e.k_stride && e.ko_head_stride == e.k_head_stride),
             "RopeAppend: in place needs equal strides");
        bind(dev);
        rope_append(dev, RopeArgs{e, q, k, v, table, positions, slots, q_out, k_out, k_cache, v_cache, nullptr});
    });
}

int nb2_tree_attention(nb2_device* dev, const nb2_tree_attn_geom* g, const void* q, const void* k_cache,
                       const void* v_cache, const int32_t* block_table, const int32_t* total_lens,
                       const int32_t* token_offsets, const int32_t* tree_mask, void* out, float* lse) {
    return guard([&] {
        need(g != nullptr, "TreeAttention: null geometry");
        need(in_i32(g->tokens) && g->batch >= 0, "TreeAttention: bad extents");
        if (g->batch > kPlanMaxBatch) {
            fail(kStatusUnsupported, "TreeAttention: at most 8192 requests");
        }
        need(float_type(g->dtype), "TreeAttention: the type must be float32, float16 or bfloat16");
        need(g->q_heads > 0 && g->kv_heads > 0 && g->q_heads % g->kv_heads == 0 && g->q_heads <= 65535,
             "TreeAttention: query heads must be a multiple of the key/value heads");
        need(g->head_dim > 0 && g->head_dim % 8 == 0, "TreeAttention: the head dimension must be a multiple of 8");
        if (g->head_dim > 256) {
            fail(kStatusUnsupported, "TreeAttention: at most 256 elements a head");
        }
        if (g->tokens * (g->q_heads / g->kv_heads) > kMaxI32 - 1024) {
            fail(kStatusUnsupported, "TreeAttention: at most 2^31 - 1025 rows a key/value head");
        }
        need(g->max_new >= 0 && g->max_new <= kMaxI32, "TreeAttention: bad bound of new tokens");
        need(g->block_size > 0 && g->block_size <= kMaxI32 && in_i32(g->num_blocks), "TreeAttention: bad cache extents");
        need(in_i32(g->table_blocks) && g->table_stride >= g->table_blocks, "TreeAttention: bad block table extents");
        need((tree_mask != nullptr) == (g->mask_words > 0), "TreeAttention: a tree mask needs its width");
        need(std::isfinite(g->scale), "TreeAttention: the scale must be finite");
        if (g->tokens == 0) {
            return;
        }
        need(q && out && token_offsets, "TreeAttention: null buffer");
        need(g->batch == 0 || total_lens != nullptr, "TreeAttention: null buffer");
        need(g->batch == 0 || g->table_blocks == 0 || block_table != nullptr, "TreeAttention: null buffer");
        need(g->num_blocks == 0 || (k_cache && v_cache), "TreeAttention: null buffer");
        nb2_tree_attn_geom e = *g;
        for (int64_t* s : {&e.q_stride, &e.o_stride}) {
            level(g->tokens, *s, g->head_dim);
        }
        for (int64_t* s : {&e.q_head_stride, &e.o_head_stride}) {
            level(g->q_heads, *s, g->head_dim);
        }
        for (int64_t* s : {&e.kc_head_stride, &e.vc_head_stride}) {
            level(g->kv_heads, *s, g->head_dim);
        }
        for (int64_t* s : {&e.kc_block_stride, &e.vc_block_stride}) {
            level(g->num_blocks, *s, g->head_dim);
        }
        for (int64_t* s : {&e.kc_place_stride, &e.vc_place_stride}) {
            level(g->block_size, *s, g->head_dim);
        }
        const int64_t unit = 16 / dtype_bytes(g->dtype);
        for (int64_t s : {e.q_stride, e.q_head_stride, e.o_stride, e.o_head_stride, e.kc_block_stride, e.kc_place_stride,
                          e.kc_head_stride, e.vc_block_stride, e.vc_place_stride, e.vc_head_stride}) {
            need(s % unit == 0, "TreeAttention: strides must be multiples of 16 bytes");
        }
        for (const void* p : {q, k_cache, v_cache, static_cast<const void*>(out)}) {
            need((reinterpret_cast<uintptr_t>(p) & 15) == 0, "TreeAttention: buffers must be 16-byte aligned");
        }
        need(out != q || (e.o_stride == e.q_stride && e.o_head_stride == e.q_head_stride),
             "TreeAttention: in place needs equal strides");
        bind(dev);
        tree_attention(dev, TreeAttnArgs{e, q, k_cache, v_cache, block_table, total_lens, token_offsets,
                                         reinterpret_cast<const uint32_t*>(tree_mask), out, lse, nullptr});
    });
}

int nb2_logits_process(nb2_device* dev, const nb2_logits_geom* g, const void* logits, void* out,
                       const int32_t* row_request, const int32_t* prompt_ids, const int32_t* prompt_offsets,
                       const int32_t* output_ids, const int32_t* output_offsets, const float* repetition,
                       const float* presence, const float* frequency, const int32_t* bias_ids,
                       const float* bias_values, const int32_t* bias_offsets, const int32_t* grammar,
                       const int32_t* grammar_rows) {
    return guard([&] {
        need(g != nullptr, "LogitsProcess: null geometry");
        need(in_i32(g->rows) && in_i32(g->vocab) && g->requests >= 0, "LogitsProcess: bad extents");
        need(float_type(g->in_dtype) && float_type(g->out_dtype),
             "LogitsProcess: the types must be float32, float16 or bfloat16");
        need((prompt_ids == nullptr || prompt_offsets != nullptr) && (output_ids == nullptr || output_offsets != nullptr),
             "LogitsProcess: a list needs its offsets");
        need(bias_ids == nullptr || (bias_values != nullptr && bias_offsets != nullptr),
             "LogitsProcess: a bias list needs its values and offsets");
        constexpr int64_t kMaxList = int64_t{1} << 30; // a count of one token must fit 30 bits
        need(g->prompt_count >= 0 && g->prompt_count < kMaxList && g->output_count >= 0 &&
                 g->output_count < kMaxList && g->bias_count >= 0 && g->bias_count < kMaxList,
             "LogitsProcess: a list holds between 0 and 2^30 - 1 ids");
        need(grammar == nullptr || g->grammar_stride >= (g->vocab + 31) / 32, "LogitsProcess: a grammar row is too short");
        if (g->rows == 0 || g->vocab == 0) {
            return;
        }
        need(logits != nullptr && out != nullptr, "LogitsProcess: null buffer");
        need(g->out_stride >= g->vocab || g->rows == 1, "LogitsProcess: output rows overlap");
        need(out != logits || (g->in_dtype == g->out_dtype && g->in_stride == g->out_stride),
             "LogitsProcess: in place needs equal types and strides");
        bind(dev);
        logits_process(dev, LogitsArgs{*g, logits, out, row_request, prompt_ids, prompt_offsets, output_ids,
                                       output_offsets, repetition, presence, frequency, bias_ids, bias_values,
                                       bias_offsets, reinterpret_cast<const uint32_t*>(grammar), grammar_rows, nullptr});
    });
}

} // extern "C"
