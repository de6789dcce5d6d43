// Logit rules: repeated-token penalties, biases and grammar masks, one pass
// over the logits.
//
// The rules that depend on a request's texts touch few of the vocabulary's
// tokens; what has to be moved is the rows themselves, in and out, so the
// kernel is bound by HBM. A CTA takes one chunk of the vocabulary for some
// consecutive rows.
// For each request among them it first walks the request's lists (read again by
// every chunk, from L2, which is why a CTA keeps one request's rows together) and keeps one word a
// token of its chunk in shared memory: bits 0-29 the count in the output list, bit 30 that it has
// a bias, bit 31 that it is in the prompt list; with a bias list a second word, the list index + 1 of
// its last bias. Sums, maxima and bits of integers: no order shows in the result. The words then
// become what the request's rows have in common: the float bias - frequency * count - presence,
// and a bitmap of the tokens that the repetition factor applies to. Then the chunk of
// every row of the request is streamed, the next row's loads in flight, every element through the same
// few instructions: x * (x > 0 ? 1/rep : rep or 1) + word.
// Measured (408 rows of 128,000 tokens in bfloat16 to float32, 313 MB, 24 requests of up to 8,000
// tokens): 84 us among other passes, 3.8 TB/s. Rules only where a bitmap has a bit, inside the stream (some lane of nearly every warp
// has one; 37 instructions an element): 115 us. Plain stream, then single stores at the touched
// tokens (each a read and a partial write of a sector in L2): 150 us. Five CTAs an SM leave 48 registers, which suit
// 16-bit logits; the float32 forms spill 80 bytes a thread there.

#include "serving.cuh"

namespace nb2 {

namespace {

constexpr int kLogitThreads = 256;
constexpr int kLogitChunk = 4096;
constexpr int kLogitWords = kLogitChunk / 32;
constexpr int kMaxRows = 32; // rows of a CTA
constexpr uint32_t kInPrompt = 1u << 31, kHasBias = 1u << 30, kCount = kHasBias - 1;

__device__ __forceinline__ void list_range(const int32_t* offsets, int64_t r, int64_t count, int& lo, int& hi, bool& bad) {
    lo = offsets[r];
    hi = offsets[r + 1];
    if (lo < 0 || hi < lo || hi > count) {
        bad = true;
        lo = hi = 0;
    }
}

// ids [lo, hi) of a list that fall into the chunk, to `hit(index in the chunk, index in the list)`.
template <typename F>
__device__ __forceinline__ void walk_list(const int32_t* ids, int lo, int hi, int64_t v0, int n, int64_t vocab, bool& bad,
                                          F hit) {
    constexpr int kAhead = 8; // loads of a thread in flight
    for (int64_t i = lo + static_cast<int>(threadIdx.x); i < hi; i += kAhead * kLogitThreads) {
        int v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            v[u] = i + u * kLogitThreads < hi ? __ldg(ids + i + u * kLogitThreads) : 0;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i + u * kLogitThreads < hi) {
                bad = bad || v[u] < 0 || v[u] >= vocab;
                const int64_t at = v[u] - v0;
                if (at >= 0 && at < n) {
                    hit(static_cast<int>(at), static_cast<int>(i + u * kLogitThreads));
                }
            }
        }
    }
}

// kLevel: every row starts on a whole pack, in the logits and in the results.
template <typename TI, typename TO, bool kBias, bool kLevel>
__global__ void __launch_bounds__(kLogitThreads, kLevel ? 5 : 1)
    logits_kernel(const __grid_constant__ LogitsArgs a, int rows_per_cta) {
    extern __shared__ uint32_t logit_smem[];
    // logits of a thread and step: the wider side is 16 bytes, so that a warp's loads and stores have no gaps
    constexpr int V = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO));
    constexpr int kSteps = kLogitChunk / V / kLogitThreads;
    using PI = Pack<TI, V>;
    using PO = Pack<TO, V>;
    const nb2_logits_geom& g = a.g;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * rows_per_cta;
    const int64_t end = min(g.rows, first + rows_per_cta);
    const int64_t v0 = static_cast<int64_t>(blockIdx.y) * kLogitChunk;
    const int n = static_cast<int>(min(static_cast<int64_t>(kLogitChunk), g.vocab - v0));
    uint32_t* seen = logit_smem; // tokens with a repetition penalty
    uint32_t* counts = seen + kLogitWords;
    float* add = reinterpret_cast<float*>(counts);
    uint32_t* last = counts + kLogitChunk; // with a bias list
    const int tid = threadIdx.x;
    bool bad = false;
    int64_t held = -2; // the request whose lists are in shared memory
    float rep = 1.0f, inv = 1.0f;

    // each row's request (-1: none) and grammar row (-1: none)
    __shared__ int64_t row_of[kMaxRows], mask_of[kMaxRows];
    const int rows = static_cast<int>(end - first);
    if (tid < rows) {
        int64_t r = a.row_request != nullptr ? a.row_request[first + tid] : first + tid;
        if (r < 0 || r >= g.requests) {
            bad = true;
            r = -1;
        }
        int64_t m = -1;
        if (a.grammar != nullptr) {
            m = a.grammar_rows != nullptr ? a.grammar_rows[first + tid] : first + tid;
            if (m >= g.grammar_count) {
                bad = true;
                m = -1;
            }
        }
        row_of[tid] = r;
        mask_of[tid] = m;
    }
    __syncthreads();

    // `body` packs of a row from token `head` on start on a whole pack in the logits and in the results (none
    // where the two can't).
    const TI* in = static_cast<const TI*>(a.logits) + first * g.in_stride + v0;
    TO* out = static_cast<TO*>(a.out) + first * g.out_stride + v0;
    auto parts = [&](const TI* x, const TO* y, int& head, int& body) {
        head = 0;
        body = n / V;
        if constexpr (!kLevel) {
            head = min(n, static_cast<int>((alignof(PI) - reinterpret_cast<uintptr_t>(x) % alignof(PI)) % alignof(PI) /
                                           sizeof(TI)));
            body = reinterpret_cast<uintptr_t>(y + head) % alignof(PO) == 0 ? (n - head) / V : 0;
        }
    };
    auto words_of = [&](int row) { // null: no grammar
        return mask_of[row] >= 0 ? a.grammar + mask_of[row] * g.grammar_stride + (v0 >> 5) : nullptr;
    };
    const int last_word = (n - 1) >> 5;
    // A row's packs and grammar bits of a thread. kLevel: a warp's kSteps * V words come as one load, word m of step k
    // in lane k * V + m, and reach their lanes when they are used.
    constexpr int kMine = kLevel ? 1 : kSteps;
    auto fetch = [&](const TI* src, const uint32_t* words, int head, int body, PI (&x)[kSteps], uint32_t (&keep)[kMine]) {
        if constexpr (kLevel) {
            static_assert(kSteps * V <= 32, "a warp's words of a row are one load");
            const int w = (tid & 31) / V * (kLogitThreads * V / 32) + (tid >> 5) * V + (tid & 31) % V;
            keep[0] = words != nullptr && (tid & 31) < kSteps * V && w <= last_word ? words[w] : 0xffffffffu;
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int i = tid + k * kLogitThreads;
            if constexpr (!kLevel) {
                keep[k] = 0xffffffffu;
            }
            if (i < body) {
                x[k] = *reinterpret_cast<const PI*>(src + head + i * V);
                if (!kLevel && words != nullptr) {
                    const int bit = head + i * V, w = bit >> 5;
                    keep[kLevel ? 0 : k] = words[w] >> (bit & 31);
                    if ((bit & 31) > 32 - V && w < last_word) { // a pack over two words
                        keep[kLevel ? 0 : k] |= words[w + 1] << (32 - (bit & 31));
                    }
                }
            }
        }
    };
    PI x[kSteps];
    uint32_t keep[kMine];
    int head, body;
    const uint32_t* words = words_of(0);
    parts(in, out, head, body);
    fetch(in, words, head, body, x, keep);

    for (int row = 0; row < rows; ++row) {
        const int64_t r = row_of[row];
        if (r != held) {
            __syncthreads(); // the rows before are done with the words
            const uint4 zero = make_uint4(0, 0, 0, 0);
            for (int i = tid; i < kLogitChunk / 4; i += kLogitThreads) {
                reinterpret_cast<uint4*>(counts)[i] = zero;
                if (kBias) {
                    reinterpret_cast<uint4*>(last)[i] = zero;
                }
            }
            __syncthreads();
            int lo, hi;
            if (r >= 0 && a.prompt_ids != nullptr) {
                list_range(a.prompt_offsets, r, g.prompt_count, lo, hi, bad);
                walk_list(a.prompt_ids, lo, hi, v0, n, g.vocab, bad, [&](int at, int) {
                    atomicOr(&counts[at], kInPrompt);
                });
            }
            if (r >= 0 && a.output_ids != nullptr) {
                list_range(a.output_offsets, r, g.output_count, lo, hi, bad);
                walk_list(a.output_ids, lo, hi, v0, n, g.vocab, bad, [&](int at, int) {
                    atomicAdd(&counts[at], 1u);
                });
            }
            if (kBias && r >= 0) {
                list_range(a.bias_offsets, r, g.bias_count, lo, hi, bad);
                walk_list(a.bias_ids, lo, hi, v0, n, g.vocab, bad, [&](int at, int i) {
                    atomicMax(&last[at], static_cast<uint32_t>(i) + 1u);
                    atomicOr(&counts[at], kHasBias);
                });
            }
            rep = r >= 0 && a.repetition != nullptr ? a.repetition[r] : 1.0f;
            inv = 1.0f / rep;
            const float pres = r >= 0 && a.presence != nullptr ? a.presence[r] : 0.0f;
            const float freq = r >= 0 && a.frequency != nullptr ? a.frequency[r] : 0.0f;
            held = r;
            __syncthreads();
            for (int at = tid; at < kLogitChunk; at += kLogitThreads) {
                const uint32_t c = counts[at], used = c & kCount;
                const uint32_t some = __ballot_sync(0xffffffffu, (c & (kInPrompt | kCount)) != 0);
                if ((tid & 31) == 0) {
                    seen[at >> 5] = some;
                }
                float d = used != 0 ? -fmaf(freq, static_cast<float>(used), pres) : 0.0f;
                if (kBias && (c & kHasBias) != 0) {
                    d += a.bias_values[last[at] - 1];
                }
                add[at] = d;
            }
            __syncthreads();
        }
        // the next row's loads, in flight while this one is written
        PI next_x[kSteps];
        uint32_t next_keep[kMine];
        int next_head = 0, next_body = 0;
        const uint32_t* next_words = nullptr;
        if (row + 1 < rows) {
            next_words = words_of(row + 1);
            parts(in + g.in_stride, out + g.out_stride, next_head, next_body);
            fetch(in + g.in_stride, next_words, next_head, next_body, next_x, next_keep);
        }
        auto ruled = [&](float x, bool penalty, float more) {
            return x * (penalty ? (x > 0.0f ? inv : rep) : 1.0f) + more;
        };
        auto one = [&](int i) {
            const float y = ruled(to_f32(in[i]), (seen[i >> 5] >> (i & 31)) & 1u, add[i]);
            const bool allowed = words == nullptr || ((words[i >> 5] >> (i & 31)) & 1u) != 0;
            out[i] = from_f32<TO>(allowed ? y : -INFINITY);
        };
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int i = tid + k * kLogitThreads;
            uint32_t allowed = keep[kLevel ? 0 : k];
            if constexpr (kLevel) {
                allowed = __shfl_sync(0xffffffffu, allowed, k * V + (tid & 31) * V / 32) >> (tid * V & 31);
            }
            if (i < body) {
                const int at = head + i * V, s = at & 31;
                float more[V];
                uint32_t penalty = seen[at >> 5] >> s;
                if (kLevel) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(add + at + j);
                        more[j] = f.x, more[j + 1] = f.y, more[j + 2] = f.z, more[j + 3] = f.w;
                    }
                } else {
                    if (s > 32 - V && (at >> 5) + 1 < kLogitWords) { // a pack over two words
                        penalty |= seen[(at >> 5) + 1] << (32 - s);
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        more[j] = add[at + j];
                    }
                }
                PO o;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float y = ruled(to_f32(x[k].e[j]), (penalty >> j) & 1u, more[j]);
                    o.e[j] = from_f32<TO>((allowed >> j) & 1u ? y : -INFINITY);
                }
                *reinterpret_cast<PO*>(out + at) = o;
            }
        }
        if (body > 0) {
            for (int i = tid; i < head; i += kLogitThreads) {
                one(i);
            }
        }
        for (int i = (body > 0 ? head + body * V : 0) + tid; i < n; i += kLogitThreads) {
            one(i);
        }
        in += g.in_stride;
        out += g.out_stride;
        words = next_words;
        head = next_head;
        body = next_body;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            x[k] = next_x[k];
        }
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            keep[k] = next_keep[k];
        }
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    }
}

template <typename TI, typename TO, bool kBias, bool kLevel>
void launch_logits(nb2_device* dev, const LogitsArgs& a) {
    auto kernel = logits_kernel<TI, TO, kBias, kLevel>;
    const int smem = 4 * (kLogitWords + kLogitChunk * (kBias ? 2 : 1));
    static bool set[64] = {};
    if (!set[dev->ordinal]) {
        check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                   "cudaFuncSetAttribute(logits)");
        set[dev->ordinal] = true;
    }
    const int64_t chunks = (a.g.vocab + kLogitChunk - 1) / kLogitChunk;
    if (chunks > 65535) {
        fail(kStatusUnsupported, "LogitsProcess: too many tokens");
    }
    // rows of a CTA: as many as leave each SM four CTAs to run one after another or at once, and whole requests where
    // those have so few rows (a CTA that meets a second request walks lists twice)
    int64_t rows = std::min<int64_t>(kMaxRows, std::max<int64_t>(1, a.g.rows * chunks / (4 * dev->num_sms)));
    const int64_t each = a.g.requests > 0 ? a.g.rows / a.g.requests : 1;
    if (each > 1 && rows > each) {
        rows = rows / each * each;
    }
    const dim3 grid(static_cast<unsigned>((a.g.rows + rows - 1) / rows), static_cast<unsigned>(chunks));
    kernel<<<grid, kLogitThreads, smem, dev->stream>>>(a, static_cast<int>(rows));
    check_cuda(cudaGetLastError(), "logits launch");
}

template <typename TI, typename TO>
void pick_bias(nb2_device* dev, const LogitsArgs& a) {
    constexpr int kPack = 16 / static_cast<int>(std::max(sizeof(TI), sizeof(TO))); // logits of a step
    const bool level = reinterpret_cast<uintptr_t>(a.logits) % (kPack * sizeof(TI)) == 0 && a.g.in_stride % kPack == 0 &&
                       reinterpret_cast<uintptr_t>(a.out) % (kPack * sizeof(TO)) == 0 && a.g.out_stride % kPack == 0;
    if (a.bias_ids != nullptr) {
        level ? launch_logits<TI, TO, true, true>(dev, a) : launch_logits<TI, TO, true, false>(dev, a);
    } else {
        level ? launch_logits<TI, TO, false, true>(dev, a) : launch_logits<TI, TO, false, false>(dev, a);
    }
}

template <typename TI>
void pick_logits(nb2_device* dev, const LogitsArgs& a) {
    if (a.g.out_dtype == kF32) {
        pick_bias<TI, float>(dev, a);
    } else if (a.g.out_dtype == kF16) {
        pick_bias<TI, __half>(dev, a);
    } else {
        pick_bias<TI, __nv_bfloat16>(dev, a);
    }
}

} // namespace

void logits_process(nb2_device* dev, LogitsArgs a) {
    if (a.g.rows == 0) {
        return;
    }
    a.err = dev->error_word();
    if (a.g.in_dtype == kF32) {
        pick_logits<float>(dev, a);
    } else if (a.g.in_dtype == kF16) {
        pick_logits<__half>(dev, a);
    } else {
        pick_logits<__nv_bfloat16>(dev, a);
    }
}

} // namespace nb2
