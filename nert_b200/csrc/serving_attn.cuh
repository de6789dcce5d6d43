// Shared by the tree attention kernels: the split of the work over the grid and
// the join of the pieces. The split is explained in serving_attn.cu.
#pragma once

#include "serving.cuh"

#include <algorithm>

namespace nb2 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ---- the split of the work ----------------------------------------------------

struct Request {
    int64_t first;  // its first token
    int n, total;   // new tokens, places (0 where the lengths cannot be right)
    int row_blocks; // blocks of its n * group rows
    int tiles;      // tiles of its places, at least one so that rows without places are written
    bool bad;
    int extra;      // what beginning and ending an item costs a CTA, in tiles: Q, the pipeline's fill, the stores
    __device__ __forceinline__ int per_item() const { return tiles + extra; }
    __device__ __forceinline__ int64_t units(int64_t kv_heads) const {
        return static_cast<int64_t>(row_blocks) * kv_heads * per_item();
    }
};

template <int RT, int KT>
__device__ __forceinline__ Request request_at(const TreeAttnArgs& a, int r, int group) {
    Request q{};
    const int64_t lo = a.offsets[r], hi = a.offsets[r + 1];
    const int64_t total = a.total[r];
    if (lo < 0 || hi < lo || hi > a.g.tokens) {
        q.bad = true;
        return q;
    }
    q.first = lo;
    q.n = static_cast<int>(hi - lo);
    if (q.n == 0) {
        return q;
    }
    constexpr int64_t kMostPlaces = 0x7fffff00; // a tile past the end still counts in 32 bits
    q.bad = total < q.n || total > kMostPlaces || total > a.g.table_blocks * a.g.block_size || q.n > a.g.max_new;
    q.total = q.bad ? 0 : static_cast<int>(total);
    q.row_blocks = static_cast<int>((static_cast<int64_t>(q.n) * group + RT - 1) / RT);
    q.tiles = max(1, (q.total + KT - 1) / KT);
    q.extra = KT == 128 ? 5 : 2; // measured: fewer or more are slower by 5% on mixed lengths
    return q;
}

// CTA whose span holds unit w, of `grid` spans [c W / grid, (c + 1) W / grid).
__device__ __forceinline__ int cta_of(int64_t w, int64_t W, int64_t grid) {
    return static_cast<int>(((w + 1) * grid - 1) / W);
}

template <int NT>
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        red[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    int64_t s = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        s += red[w];
    }
    return s;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Bits of places k0 .. k0 + 31, counted from the first new token, that a row's token sees.
__device__ __forceinline__ uint32_t see_bits(const uint32_t* mask, int64_t words, int tok, int k0) {
    if (k0 <= -32) {
        return 0xffffffffu;
    }
    if (mask == nullptr) { // a chain: up to the token itself
        const int n = tok - k0 + 1;
        return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
    }
    if (k0 < 0) {
        return (mask[0] << -k0) | ((1u << -k0) - 1u);
    }
    const int w = k0 >> 5, s = k0 & 31;
    const uint32_t lo = w < words ? mask[w] : 0u, hi = w + 1 < words ? mask[w + 1] : 0u;
    return __funnelshift_r(lo, hi, s);
}

// ---- the join ------------------------------------------------------------------

// Elements d .. d + 3 of a finished row (unnormalised sums x, maximum m in base 2, sum of weights z).
template <typename T>
__device__ __forceinline__ void store_row4(const TreeAttnArgs& a, int64_t first, int64_t kvh, int group, int rho, int d,
                                           float4 x, float m, float z) {
    const int tok = rho / group;
    const int64_t h = kvh * group + (rho - tok * group), t = first + tok;
    const bool none = z == 0.0f; // no place was seen
    const float inv = 1.0f / z;
    Pack<T, 4> y;
    y.e[0] = from_f32<T>(none ? 0.0f : x.x * inv);
    y.e[1] = from_f32<T>(none ? 0.0f : x.y * inv);
    y.e[2] = from_f32<T>(none ? 0.0f : x.z * inv);
    y.e[3] = from_f32<T>(none ? 0.0f : x.w * inv);
    *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(a.out) + t * a.g.o_stride + h * a.g.o_head_stride + d) = y;
    if (d == 0 && a.lse != nullptr) {
        a.lse[t * a.g.q_heads + h] = none ? -INFINITY : m * kLn2 + logf(z);
    }
}

// The pieces of an item in the slots of CTAs c0 .. c1 (the first left its piece in its second slot,
// the others theirs in their first), added in that order and stored; NT threads. A thread takes kElems groups of
// four elements through kPieces pieces at a time, all their loads in flight: one after another the loads of a short
// item's pieces (up to one a tile) took longer than its tiles. kColumns: pieces lie four elements by four, the rows together;
// a warp takes 8 rows x 16 elements. `step` threads share the item.
template <typename T, int DP, int RT, int NT, int kElems, int kPieces, bool kColumns>
__device__ __forceinline__ void join_pieces_as(const TreeAttnArgs& a, const float* part_o, const float2* part_ml, int c0,
                                               int c1, int64_t first, int64_t kvh, int group, int rho0, int rows, int tid,
                                               int step) {
    static_assert(!kColumns || kElems == 1, "the columns' order is that of one element a thread");
    auto place = [](int i, int& row, int& d) {
        if constexpr (kColumns) {
            const int r = i >> 5;
            row = r / (DP / 16) * 8 + ((i >> 2) & 7);
            d = r % (DP / 16) * 16 + (i & 3) * 4;
        } else {
            row = i / (DP / 4);
            d = (i - row * (DP / 4)) * 4;
        }
    };
    const int all = (kColumns ? (rows + 7) / 8 * 8 : rows) * (DP / 4);
    for (int i0 = tid; i0 < all; i0 += kElems * step) {
        float m[kElems], z[kElems];
        float4 x[kElems];
#pragma unroll
        for (int u = 0; u < kElems; ++u) {
            m[u] = -INFINITY;
            z[u] = 0.0f;
            x[u] = make_float4(0, 0, 0, 0);
        }
#pragma unroll 1
        for (int c = c0; c <= c1; c += kPieces) {
            float2 ml[kPieces][kElems];
            float4 y[kPieces][kElems];
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
                const int64_t slot = 2 * static_cast<int64_t>(c + p) + (c + p == c0 ? 1 : 0);
#pragma unroll
                for (int u = 0; u < kElems; ++u) {
                    int row, d;
                    place(i0 + u * step, row, d);
                    ml[p][u] = make_float2(-INFINITY, 0.0f);
                    if (c + p <= c1 && row < rows && d < a.g.head_dim) {
                        ml[p][u] = __ldcg(&part_ml[slot * RT + row]);
                        y[p][u] = __ldcg(reinterpret_cast<const float4*>(
                            part_o + (kColumns ? (slot * (DP / 4) + d / 4) * RT * 4 + row * 4 : (slot * RT + row) * DP + d)));
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
#pragma unroll
                for (int u = 0; u < kElems; ++u) {
                    const float to = fmaxf(m[u], ml[p][u].x), ref = to == -INFINITY ? 0.0f : to;
                    const float f = exp2_fast(m[u] - ref), h = exp2_fast(ml[p][u].x - ref);
                    m[u] = to;
                    z[u] = f * z[u] + h * ml[p][u].y;
                    x[u].x *= f, x[u].y *= f, x[u].z *= f, x[u].w *= f;
                    if (h != 0.0f) { // a piece that saw nothing adds nothing
                        x[u].x += h * y[p][u].x, x[u].y += h * y[p][u].y, x[u].z += h * y[p][u].z, x[u].w += h * y[p][u].w;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kElems; ++u) {
            int row, d;
            place(i0 + u * step, row, d);
            if (row < rows && d < a.g.head_dim) {
                store_row4<T>(a, first, kvh, group, rho0 + row, d, x[u], m[u], z[u]);
            }
        }
    }
}

template <typename T, int DP, int RT, int NT>
__device__ __forceinline__ void join_pieces(const TreeAttnArgs& a, const float* part_o, const float2* part_ml, int c0, int c1,
                                            int64_t first, int64_t kvh, int group, int rho0, int rows, int tid) {
    if (rows * (DP / 4) <= 2 * NT) {
        join_pieces_as<T, DP, RT, NT, 1, 8, false>(a, part_o, part_ml, c0, c1, first, kvh, group, rho0, rows, tid, NT);
    } else {
        join_pieces_as<T, DP, RT, NT, 4, 2, false>(a, part_o, part_ml, c0, c1, first, kvh, group, rho0, rows, tid, NT);
    }
}

// Zero rows for the tokens that belong to no request.
template <typename T>
__device__ __forceinline__ void spare_tokens(const TreeAttnArgs& a, int tid, int nt) {
    const nb2_tree_attn_geom& g = a.g;
    const int64_t lo = g.batch > 0 ? a.offsets[0] : 0, hi = g.batch > 0 ? a.offsets[g.batch] : 0;
    const int64_t before = min(max(lo, int64_t{0}), g.tokens), after = min(max(hi, before), g.tokens);
    const int64_t spare = (before + g.tokens - after) * g.q_heads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * nt + tid; i < spare; i += static_cast<int64_t>(gridDim.x) * nt) {
        int64_t t = i / g.q_heads;
        const int64_t h = i - t * g.q_heads;
        t = t < before ? t : t - before + after;
        T* row = static_cast<T*>(a.out) + t * g.o_stride + h * g.o_head_stride;
        for (int d = 0; d < g.head_dim; ++d) {
            row[d] = from_f32<T>(0.0f);
        }
        if (a.lse != nullptr) {
            a.lse[t * g.q_heads + h] = -INFINITY;
        }
    }
}

// Spans shorter than kMinSpan units are not made once `least` CTAs have one: each adds a piece to a join, whose pieces
// take about a third of a tile each.
constexpr int kMinSpan = 4;

// This CTA's span of the W units, and the request that its first unit is in. All NT threads.
__device__ __forceinline__ int64_t span_count(int64_t W, int64_t ctas, int least) { // none is empty
    return min(ctas, max(W / kMinSpan, min(W, static_cast<int64_t>(least))));
}

struct Span {
    int64_t W, grid, w0, w1;
    int request;          // holds unit w0
    int64_t request_unit; // first unit of that request
    __device__ __forceinline__ void set(int64_t cta, int least) {
        grid = span_count(W, gridDim.x, least);
        w0 = cta < grid ? cta * W / grid : 0;
        w1 = cta < grid ? (cta + 1) * W / grid : 0;
    }
};

template <int RT, int KT, int NT>
__device__ __forceinline__ Span find_span(const TreeAttnArgs& a, int group, int least, int64_t* red, int64_t* found,
                                          bool& bad) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int B = static_cast<int>(a.g.batch);
    const int64_t cta = blockIdx.x;
    Span s{};
    if (B <= 32) { // every warp for itself: no barrier
        const Request q = lane < B ? request_at<RT, KT>(a, lane, group) : Request{};
        bad |= q.bad;
        const int64_t u = q.units(a.g.kv_heads);
        int64_t inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
            inc += lane >= o ? up : 0;
        }
        s.W = __shfl_sync(0xffffffffu, inc, 31);
        s.set(cta, least);
        const uint32_t hit = __ballot_sync(0xffffffffu, s.w0 < s.w1 && inc - u <= s.w0 && s.w0 < inc);
        s.request = hit != 0 ? __ffs(hit) - 1 : 0;
        s.request_unit = __shfl_sync(0xffffffffu, inc - u, s.request);
        return s;
    }
    int64_t mine = 0; // units of request tid
    for (int r = tid; r < B; r += NT) {
        const Request q = request_at<RT, KT>(a, r, group);
        bad |= q.bad;
        s.W += q.units(a.g.kv_heads);
        mine = r == tid ? s.W : mine;
    }
    s.W = block_sum<NT>(s.W, red);
    s.set(cta, least);
    if (s.w0 == s.w1) {
        return s;
    }
    int64_t base = 0;
    for (int c = 0; c < B; c += NT) {
        const int64_t u = c == 0 ? mine : c + tid < B ? request_at<RT, KT>(a, c + tid, group).units(a.g.kv_heads) : 0;
        int64_t inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
            inc += lane >= o ? up : 0;
        }
        __syncthreads();
        if (lane == 31) {
            red[warp] = inc;
        }
        __syncthreads();
        int64_t all = 0;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) {
            inc += w < warp ? red[w] : 0;
            all += red[w];
        }
        inc += base;
        if (inc - u <= s.w0 && s.w0 < inc) {
            found[0] = c + tid;
            found[1] = inc - u;
        }
        base += all;
        if (base > s.w0) {
            break;
        }
    }
    __syncthreads();
    s.request = static_cast<int>(found[0]);
    s.request_unit = found[1];
    return s;
}

// ---- the join of few items, by a launch of its own ----------------------------------

// An item's pieces are joined by one CTA when it has a few; where few items share the GPU (one long context), each is in
// many, which that CTA reads one after another while the others are gone: then a second launch joins them, a slice
// of an item's elements a CTA. By the CTA / by the launch, bfloat16, 60,000 places: 64 tokens, 32/8 heads of 128 (18 pieces
// of 128 KB) 123 / 99 us, 8/1 heads (74 pieces) 152 / 58; 8 tokens, 32/8 heads (18 of 16 KB) 96 / 93; 8,000 places, 33 tokens 57 / 40.
// One token (37 of 2 KB) takes 61 us and 57 with no join at all, so nothing would be gained there.
constexpr int kJoinThreads = 256;
constexpr int64_t kJoinApart = 256 << 10; // bytes of an item's pieces from which on that is faster

inline bool join_apart(const TreeAttnArgs& a, int ctas, int RT, int DP, dim3& grid) {
    const nb2_tree_attn_geom& g = a.g;
    const int64_t rows = std::min(g.max_new, g.tokens) * (g.q_heads / g.kv_heads);
    const int64_t items = g.batch * g.kv_heads * ((rows + RT - 1) / RT), most = (std::min<int64_t>(rows, RT) + 7) / 8 * 8;
    grid = dim3(static_cast<unsigned>((most * (DP / 4) + kJoinThreads - 1) / kJoinThreads), static_cast<unsigned>(items));
    return items > 0 && g.batch <= kJoinThreads && items <= 65535 && most * DP * 4 * ctas > kJoinApart * items;
}

template <typename T, int DP, int RT, int KT, bool kColumns>
__global__ void __launch_bounds__(kJoinThreads)
    join_kernel(const __grid_constant__ TreeAttnArgs a, int group, int ctas, int least, const float* part_o,
                const float2* part_ml) {
    __shared__ int64_t warp_items[kJoinThreads / 32], warp_units[kJoinThreads / 32], found[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t kv_heads = a.g.kv_heads, wanted = blockIdx.y;
    Request q{};
    if (tid < a.g.batch) {
        q = request_at<RT, KT>(a, tid, group);
    }
    // A request out of its bounds may have more rows than the grid was sized for. Its items are of one tile, which is never
    // cut, so they need no join and are not counted.
    const int64_t items = q.bad ? 0 : q.row_blocks * kv_heads, units = q.units(kv_heads);
    int64_t items_to = items, units_to = units, W = 0, all = 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, items_to, o), y = __shfl_up_sync(0xffffffffu, units_to, o);
        items_to += lane >= o ? x : 0;
        units_to += lane >= o ? y : 0;
    }
    if (lane == 31) {
        warp_items[warp] = items_to;
        warp_units[warp] = units_to;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) {
        items_to += w < warp ? warp_items[w] : 0;
        units_to += w < warp ? warp_units[w] : 0;
        all += warp_items[w];
        W += warp_units[w];
    }
    if (items_to - items <= wanted && wanted < items_to) {
        found[0] = tid;
        found[1] = wanted - (items_to - items);
        found[2] = units_to - units;
    }
    __syncthreads();
    if (wanted >= all) {
        return;
    }
    const Request rq = request_at<RT, KT>(a, static_cast<int>(found[0]), group);
    const int64_t item = found[1], w0 = found[2] + item * rq.per_item() + rq.extra, n = span_count(W, ctas, least);
    const int64_t kvh = item / rq.row_blocks;
    const int rb = static_cast<int>(item - kvh * rq.row_blocks), rows = min(RT, rq.n * group - rb * RT);
    const int c0 = cta_of(w0, W, n), c1 = cta_of(w0 + rq.tiles - 1, W, n);
    if (c0 < c1) { // otherwise one CTA had all of it, and stored it
        join_pieces_as<T, DP, RT, kJoinThreads, 1, 8, kColumns>(a, part_o, part_ml, c0, c1, rq.first, kvh, group, rb * RT, rows,
                                                                static_cast<int>(blockIdx.x) * kJoinThreads + tid,
                                                                static_cast<int>(gridDim.x) * kJoinThreads);
    }
}

// The tensor-core kernel for many rows (serving_attn_tc.cu): whether it takes the call, and the call.
bool tree_attention_tc_takes(const TreeAttnArgs& a, int sms);
void tree_attention_tc(nb2_device* dev, const TreeAttnArgs& a);

} // namespace nb2
