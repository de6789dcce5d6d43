// Block tables, slots, positions and tree masks of one serving step, in one
// launch: nothing but lengths is known on the host.
//
// With l = cached and n = new tokens of request r and s = block size, the
// request takes a_r = ceil((l+n)/s) - ceil(l/s) blocks, from the exclusive prefix
// sum of a on; new token i sits at place l + i. The work is a few bytes a
// token, so latency is what it costs: the prefix sums are not handed from one
// CTA to the next. Every CTA of the token part sums all lengths itself
// (two 4-byte words a request, read from L2) and then places its own 512
// tokens by binary search in the sums; every CTA of the tree part handles one
// request and sums the lengths before it.
// Measured: 129 requests with trees of up to 64 tokens 10 us with cold caches, 64 single tokens 6; one CTA's chain of
// dependent reads (lengths, sums, table or free list, store) is what it costs.
// Ancestors by pointer doubling: after round k a token's mask holds its 2^k
// nearest ancestors and jump[i] is the 2^k-th, so a chain of N takes log2 N
// rounds instead of N dependent reads. depth = ancestors = popcount(mask) - 1.

#include "serving.cuh"

#include <algorithm>
#include <mutex>

namespace nb2 {

namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 512; // tokens placed by one CTA of the token part (2,048: a step of 129 trees 16 us, 512: 10)
constexpr int kTreeRows = kPlanMaxWords * 32 / kPlanThreads;

struct ReqLens {
    int64_t old, fresh, have, want; // tokens cached / added; blocks before / after
};

// ceil(n / s) of values below 2^31, in 32 bits (a 64-bit division is a routine of a hundred instructions)
__device__ __forceinline__ int64_t blocks_of(int64_t n, int64_t s) {
    return (static_cast<uint32_t>(n) + static_cast<uint32_t>(s) - 1u) / static_cast<uint32_t>(s);
}

// Lengths of request r, negative ones and a sum past int32 taken as nothing.
__device__ __forceinline__ ReqLens lens_of(const PagePlanArgs& a, int r, bool& bad) {
    ReqLens x;
    x.old = a.seq_lens[r];
    x.fresh = a.new_lens[r];
    if (x.old < 0 || x.fresh < 0 || x.old + x.fresh > 0x7fffffffLL) {
        bad = true;
        x.old = x.old < 0 ? 0 : x.old;
        x.fresh = 0;
    }
    x.have = blocks_of(x.old, a.g.block_size);
    x.want = blocks_of(x.old + x.fresh, a.g.block_size);
    return x;
}

__device__ __forceinline__ int clamp_i32(int64_t v) { return v > 0x7fffffffLL ? 0x7fffffff : static_cast<int>(v); }

// Largest r with first[r] <= i (first is ascending, first[0] = 0; i < first[n]).
__device__ __forceinline__ int owner(const int* first, int n, int i) {
    int lo = 0, hi = n; // first[lo] <= i < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= i) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__device__ void token_part(const PagePlanArgs& a, int part, int parts, int* smem) {
    const int B = static_cast<int>(a.g.batch);
    int* tok = smem;         // [B + 1] first token of each request
    int* blk = smem + B + 1; // [B + 1] first new block of each request
    __shared__ int64_t warp_tok[kPlanThreads / 32], warp_blk[kPlanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    bool bad = false;
    const int per = (B + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(B, tid * per), r1 = min(B, r0 + per);
    int64_t st = 0, sb = 0;
    for (int r = r0; r < r1; ++r) {
        const ReqLens x = lens_of(a, r, bad);
        st += x.fresh;
        sb += x.want - x.have;
    }
    int64_t it = st, ib = sb; // inclusive over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t ut = __shfl_up_sync(0xffffffffu, it, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) {
            it += ut;
            ib += ub;
        }
    }
    if (lane == 31) {
        warp_tok[warp] = it;
        warp_blk[warp] = ib;
    }
    __syncthreads();
    int64_t bt = it - st, bb = ib - sb;
    for (int w = 0; w < warp; ++w) {
        bt += warp_tok[w];
        bb += warp_blk[w];
    }
    for (int r = r0; r < r1; ++r) {
        const ReqLens x = lens_of(a, r, bad);
        tok[r] = clamp_i32(bt);
        blk[r] = clamp_i32(bb);
        if (part == 0) {
            a.offsets[r] = clamp_i32(bt);
            a.new_total[r] = static_cast<int32_t>(x.old + x.fresh);
        }
        bt += x.fresh;
        bb += x.want - x.have;
    }
    const int64_t head = a.free_head != nullptr ? a.free_head[0] : 0;
    if (head < 0) {
        bad = true;
    }
    if (tid == kPlanThreads - 1) {
        tok[B] = clamp_i32(bt);
        blk[B] = clamp_i32(bb);
        if (part == 0) {
            a.offsets[B] = clamp_i32(bt);
            a.free_head_out[0] = clamp_i32(head + bb);
            bad = bad || bt > a.g.tokens;
        }
    }
    __syncthreads();

    // new blocks into the table
    bool short_list = false;
    const int n_blk = blk[B];
    for (int64_t i = static_cast<int64_t>(part) * kPlanThreads + tid; i < n_blk;
         i += static_cast<int64_t>(parts) * kPlanThreads) {
        const int r = owner(blk, B, static_cast<int>(i));
        const ReqLens x = lens_of(a, r, bad);
        const int64_t j = x.have + (i - blk[r]), f = head + i;
        const bool ok = f >= 0 && f < a.g.free_blocks;
        short_list |= !ok;
        if (j < a.g.table_blocks) {
            a.table[r * a.g.table_stride + j] = ok ? a.free_blocks[f] : -1;
        } else {
            short_list = true;
        }
    }
    // this CTA's tokens
    const int n_tok = tok[B];
    for (int64_t t = static_cast<int64_t>(part) * kPlanTokens + tid;
         t < min(a.g.tokens, static_cast<int64_t>(part + 1) * kPlanTokens); t += kPlanThreads) {
        if (t >= n_tok) {
            a.slots[t] = -1;
            a.positions[t] = 0;
            for (int w = 0; w < a.g.mask_words; ++w) {
                a.mask[t * a.g.mask_words + w] = 0;
            }
            continue;
        }
        const int r = owner(tok, B, static_cast<int>(t));
        const ReqLens x = lens_of(a, r, bad);
        const int64_t p = x.old + (t - tok[r]);
        const uint32_t size = static_cast<uint32_t>(a.g.block_size), j = static_cast<uint32_t>(p) / size;
        int64_t block = -1;
        if (j < a.g.table_blocks) {
            if (j < x.have) {
                block = a.table[r * a.g.table_stride + j];
            } else { // taken in this launch, maybe by another CTA: read it at its source
                const int64_t f = head + blk[r] + (static_cast<int64_t>(j) - x.have);
                block = f >= 0 && f < a.g.free_blocks ? a.free_blocks[f] : -1;
            }
        }
        int64_t slot = block * a.g.block_size + (static_cast<uint32_t>(p) - j * size);
        if (block < 0 || slot > 0x7fffffffLL) {
            slot = -1;
            short_list = true;
        }
        a.slots[t] = static_cast<int32_t>(slot);
        if (a.parents == nullptr) {
            a.positions[t] = static_cast<int32_t>(p);
        }
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    } else if (short_list) {
        record_error(a.err, kDevNoBlock);
    }
}

__device__ void tree_part(const PagePlanArgs& a, int r, int* smem) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int W = static_cast<int>(a.g.mask_words);
    __shared__ int64_t warp_tok[kPlanThreads / 32];
    bool bad = false;
    int64_t before = 0;
    for (int i = tid; i < r; i += kPlanThreads) {
        before += lens_of(a, i, bad).fresh;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) {
        warp_tok[warp] = before;
    }
    __syncthreads();
    int64_t first = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        first += warp_tok[w];
    }
    const ReqLens x = lens_of(a, r, bad);
    int64_t all = x.fresh;
    if (first + all > a.g.tokens) { // more tokens than the outputs hold
        bad = true;
        all = first < a.g.tokens ? a.g.tokens - first : 0;
    }
    const int n = static_cast<int>(all < W * 32 ? all : W * 32);
    int* jump = smem;                                       // [32 W]
    uint32_t* seen = reinterpret_cast<uint32_t*>(smem + 32 * W); // [32 W][W]
    int up[kTreeRows];
#pragma unroll
    for (int k = 0; k < kTreeRows; ++k) {
        const int i = tid + k * kPlanThreads;
        up[k] = -1;
        if (i < n) {
            up[k] = a.parents[first + i];
            if (up[k] >= i) {
                bad = true;
                up[k] = -1;
            }
            up[k] = up[k] < 0 ? -1 : up[k];
            jump[i] = up[k];
            for (int w = 0; w < W; ++w) {
                const uint32_t self = w == (i >> 5) ? 1u << (i & 31) : 0u;
                seen[i * W + w] = self | (up[k] >= 0 && w == (up[k] >> 5) ? 1u << (up[k] & 31) : 0u);
            }
        }
    }
    // mask holds the 2^k nearest ancestors, up[] the 2^k-th
    while (__syncthreads_or([&] {
        bool any = false;
#pragma unroll
        for (int k = 0; k < kTreeRows; ++k) {
            any |= up[k] >= 0;
        }
        return any;
    }())) {
        for (int w = 0; w < W; ++w) {
            uint32_t more[kTreeRows];
#pragma unroll
            for (int k = 0; k < kTreeRows; ++k) {
                more[k] = up[k] >= 0 ? seen[up[k] * W + w] : 0u;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kTreeRows; ++k) {
                if (up[k] >= 0) {
                    seen[(tid + k * kPlanThreads) * W + w] |= more[k];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kTreeRows; ++k) {
            up[k] = up[k] >= 0 ? jump[up[k]] : -1;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kTreeRows; ++k) {
            if (tid + k * kPlanThreads < n) {
                jump[tid + k * kPlanThreads] = up[k];
            }
        }
    }
    for (int64_t i = tid; i < all; i += kPlanThreads) {
        int depth = static_cast<int>(i < 0x7fffffff ? i : 0);
        if (i < n) {
            depth = -1;
            for (int w = 0; w < W; ++w) {
                depth += __popc(seen[i * W + w]);
            }
        } else {
            bad = true; // no room in the mask: the token sees no drafted one
        }
        a.positions[first + i] = static_cast<int32_t>(x.old + depth);
    }
    for (int64_t i = tid; i < all * W; i += kPlanThreads) {
        a.mask[first * W + i] = i < static_cast<int64_t>(n) * W ? seen[i] : 0u;
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    }
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(PagePlanArgs a, int token_parts) {
    extern __shared__ int plan_smem[];
    const int part = static_cast<int>(blockIdx.x);
    if (part < token_parts) {
        token_part(a, part, token_parts, plan_smem);
    } else {
        tree_part(a, part - token_parts, plan_smem);
    }
}

} // namespace

void page_plan(nb2_device* dev, PagePlanArgs a) {
    a.err = dev->error_word();
    const int64_t parts = std::max<int64_t>(1, (a.g.tokens + kPlanTokens - 1) / kPlanTokens);
    const int64_t trees = a.parents != nullptr ? a.g.batch : 0;
    if (parts + trees > 0x7fffffffLL) {
        fail(kStatusUnsupported, "page plan: too many tokens");
    }
    const int64_t w = a.g.mask_words;
    const size_t smem = static_cast<size_t>(std::max(2 * (a.g.batch + 1), trees > 0 ? 32 * w * (w + 1) : 0)) * 4;
    // Asked for once a GPU, whatever this call's size: the 48 KB that need no asking hold the static part too, and a value
    // that followed the calls could be lowered by one thread between another's request and its launch.
    constexpr int64_t kMostSmem = 4 * std::max(2 * (kPlanMaxBatch + 1), 32 * kPlanMaxWords * (kPlanMaxWords + 1));
    static std::once_flag asked[64];
    std::call_once(asked[dev->ordinal], [] {
        check_cuda(cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(kMostSmem)),
                   "cudaFuncSetAttribute(page plan)");
    });
    page_plan_kernel<<<static_cast<unsigned>(parts + trees), kPlanThreads, smem, dev->stream>>>(
        a, static_cast<int>(parts));
    check_cuda(cudaGetLastError(), "page plan launch");
}

} // namespace nb2
