// Logit rules: repeated-token penalties, biases and grammar masks, one pass
// over the logits.
//
// The rules that depend on a request's texts touch few of the vocabulary's
// tokens; what has to be moved is the row itself, in and out, so the kernel is
// bound by HBM. A CTA takes one chunk of one row's vocabulary. It first walks the
// request's lists and keeps, in shared memory, one word a token of its chunk
// (bits 0-30: count in the output list, bit 31: in the prompt list; integer
// atomics, so no order shows in the result) and, with a bias list, a second
// word with the list index + 1 of the token's last bias (a maximum, again
// without order). Then it streams its chunk once.

#include "serving.cuh"

namespace nb2 {

namespace {

constexpr int kLogitThreads = 256;
constexpr int kLogitChunk = 4096;

__device__ __forceinline__ void list_range(const int32_t* offsets, int64_t r, int64_t count, int64_t& lo, int64_t& hi,
                                           bool& bad) {
    lo = offsets[r];
    hi = offsets[r + 1];
    if (lo < 0 || hi < lo || hi > count) {
        bad = true;
        lo = hi = 0;
    }
}

template <typename TI, typename TO>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(LogitsArgs a) {
    extern __shared__ uint32_t logit_smem[];
    const nb2_logits_geom& g = a.g;
    const int64_t row = blockIdx.x;
    const int64_t v0 = static_cast<int64_t>(blockIdx.y) * kLogitChunk;
    const int n = static_cast<int>(min(static_cast<int64_t>(kLogitChunk), g.vocab - v0));
    uint32_t* counts = logit_smem;
    uint32_t* last = logit_smem + kLogitChunk;
    bool bad = false;
    int64_t r = a.row_request != nullptr ? a.row_request[row] : row;
    const bool rules = r >= 0 && r < g.requests;
    bad = !rules;
    for (int i = threadIdx.x; i < n; i += kLogitThreads) {
        counts[i] = 0;
        if (a.bias_ids != nullptr) {
            last[i] = 0;
        }
    }
    __syncthreads();
    if (rules) {
        int64_t lo, hi;
        if (a.prompt_ids != nullptr) {
            list_range(a.prompt_offsets, r, g.prompt_count, lo, hi, bad);
            for (int64_t i = lo + threadIdx.x; i < hi; i += kLogitThreads) {
                const int64_t v = a.prompt_ids[i];
                bad = bad || v < 0 || v >= g.vocab;
                if (v >= v0 && v < v0 + n) {
                    atomicOr(&counts[v - v0], 0x80000000u);
                }
            }
        }
        if (a.output_ids != nullptr) {
            list_range(a.output_offsets, r, g.output_count, lo, hi, bad);
            for (int64_t i = lo + threadIdx.x; i < hi; i += kLogitThreads) {
                const int64_t v = a.output_ids[i];
                bad = bad || v < 0 || v >= g.vocab;
                if (v >= v0 && v < v0 + n) {
                    atomicAdd(&counts[v - v0], 1u);
                }
            }
        }
        if (a.bias_ids != nullptr) {
            list_range(a.bias_offsets, r, g.bias_count, lo, hi, bad);
            for (int64_t i = lo + threadIdx.x; i < hi; i += kLogitThreads) {
                const int64_t v = a.bias_ids[i];
                bad = bad || v < 0 || v >= g.vocab;
                if (v >= v0 && v < v0 + n) {
                    atomicMax(&last[v - v0], static_cast<uint32_t>(i + 1));
                }
            }
        }
    }
    __syncthreads();
    const float rep = rules && a.repetition != nullptr ? a.repetition[r] : 1.0f;
    const float pres = rules && a.presence != nullptr ? a.presence[r] : 0.0f;
    const float freq = rules && a.frequency != nullptr ? a.frequency[r] : 0.0f;
    const uint32_t* words = nullptr;
    if (a.grammar != nullptr) {
        const int64_t m = a.grammar_rows != nullptr ? a.grammar_rows[row] : row;
        if (m >= g.grammar_count) {
            bad = true;
        } else if (m >= 0) {
            words = a.grammar + m * g.grammar_stride;
        }
    }
    const TI* in = static_cast<const TI*>(a.logits) + row * g.in_stride + v0;
    TO* out = static_cast<TO*>(a.out) + row * g.out_stride + v0;
    for (int i = threadIdx.x; i < n; i += kLogitThreads) {
        float x = to_f32(in[i]);
        const uint32_t c = counts[i];
        if (c != 0) {
            const uint32_t used = c & 0x7fffffffu;
            x = x > 0.0f ? x / rep : x * rep;
            x -= __fadd_rn(__fmul_rn(freq, static_cast<float>(used)), used != 0 ? pres : 0.0f);
        }
        if (a.bias_ids != nullptr && last[i] != 0) {
            x += a.bias_values[last[i] - 1];
        }
        if (words != nullptr && ((words[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u) == 0) {
            x = -INFINITY;
        }
        out[i] = from_f32<TO>(x);
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    }
}

template <typename TI, typename TO>
void launch_logits(nb2_device* dev, const LogitsArgs& a) {
    const size_t smem = kLogitChunk * 4 * (a.bias_ids != nullptr ? 2 : 1);
    const int64_t chunks = (a.g.vocab + kLogitChunk - 1) / kLogitChunk;
    if (a.g.rows > 0x7fffffffLL || chunks > 65535) {
        fail(kStatusUnsupported, "logits: too many rows or tokens");
    }
    const dim3 grid(static_cast<unsigned>(a.g.rows), static_cast<unsigned>(chunks));
    logits_kernel<TI, TO><<<grid, kLogitThreads, smem, dev->stream>>>(a);
    check_cuda(cudaGetLastError(), "logits launch");
}

template <typename TI>
void pick_logits(nb2_device* dev, const LogitsArgs& a) {
    if (a.g.out_dtype == kF32) {
        launch_logits<TI, float>(dev, a);
    } else if (a.g.out_dtype == kF16) {
        launch_logits<TI, __half>(dev, a);
    } else {
        launch_logits<TI, __nv_bfloat16>(dev, a);
    }
}

} // namespace

void logits_process(nb2_device* dev, LogitsArgs a) {
    if (a.g.rows == 0) {
        return;
    }
    a.err = dev->err_word;
    if (a.g.in_dtype == kF32) {
        pick_logits<float>(dev, a);
    } else if (a.g.in_dtype == kF16) {
        pick_logits<__half>(dev, a);
    } else {
        pick_logits<__nv_bfloat16>(dev, a);
    }
}

} // namespace nb2
