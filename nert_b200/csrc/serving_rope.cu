// Rotary positions with several axes, fused with the cache write.
//
// Each pair (x1, x2) of a head is one complex number turned by the angle of
// its frequency at the position that the frequency's axis gives: six flops
// for two loads and two stores, so the kernel is bound by HBM: q, k and v
// once in and once out. The angles come as a table of cosines and sines in 32
// bits (the caller's: any base, scaling or length rule), gathered by position.
//
// A thread owns V consecutive frequencies of one token and walks over some of
// its heads, so cos and sin are loaded once for all of them; the next head's two
// V-element packs are loaded before the present one is turned and stored. Both halves
// of every pair are read before either is written, which is what makes the
// in-place form safe. The walk is a rolled loop: what bounds the kernel is how many loads an
// SM holds in flight, and 64 registers a thread (1,024 threads of 64 bytes each) took 76 us
// for 297 MB (16,001 tokens, 28 + 4 + 4 heads of 128 in bfloat16; 3.9 TB/s), four heads unrolled in
// 122 registers 117 us, 48 registers with spills 125 us.

#include "serving.cuh"

namespace nb2 {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kWalk = 4;

template <typename T, int V, bool kPairs, bool kOneAxis>
__global__ void __launch_bounds__(kRopeThreads, 4)
    rope_kernel(const __grid_constant__ RopeArgs a, int lanes, int groups, int tokens_per_cta) {
    using P = Pack<T, V>;
    const nb2_rope_geom& g = a.g;
    const int work = lanes * groups;
    const int local = static_cast<int>(threadIdx.x) / work;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * tokens_per_cta + local;
    if (local >= tokens_per_cta || t >= g.tokens) {
        return;
    }
    const int half = static_cast<int>(g.rot_dim / 2);
    const int turn = half / V; // lanes that turn pairs; the rest copy what is past rot_dim
    const int q_heads = static_cast<int>(g.q_heads), kv_heads = static_cast<int>(g.kv_heads);
    const int heads = q_heads + kv_heads + (a.v != nullptr ? kv_heads : 0);
    const int w = static_cast<int>(threadIdx.x) - local * work;
    const int group = w / lanes, lane = w - group * lanes;
    const bool turns = lane < turn;
    // element offsets of the two packs in a head
    const int e0 = !turns ? static_cast<int>(g.rot_dim) + (lane - turn) * 2 * V : kPairs ? lane * 2 * V : lane * V;
    const int e1 = turns && !kPairs ? half + e0 : e0 + V;

    auto source = [&](int h) -> const T* { // a row: one head of the token, over q's, k's and v's heads
        if (h < q_heads) {
            return static_cast<const T*>(a.q) + t * g.q_stride + h * g.q_head_stride;
        }
        h -= q_heads;
        if (h < kv_heads) {
            return static_cast<const T*>(a.k) + t * g.k_stride + h * g.k_head_stride;
        }
        return static_cast<const T*>(a.v) + t * g.v_stride + (h - kv_heads) * g.v_head_stride;
    };
    P x0, x1;
    {
        const T* row = source(group);
        x0 = *reinterpret_cast<const P*>(row + e0);
        x1 = *reinterpret_cast<const P*>(row + e1);
    }
    int64_t k_at = -1, v_at = -1; // the token's place in the caches
    if (a.slots != nullptr) {
        const int slot = a.slots[t];
        if (slot >= 0) {
            const int size = static_cast<int>(g.block_size);
            const int block = slot / size, place = slot - block * size;
            if (block < g.num_blocks) {
                k_at = block * g.kc_block_stride + place * g.kc_place_stride;
                v_at = block * g.vc_block_stride + place * g.vc_place_stride;
            } else {
                record_error(a.err, kDevIndexOutOfRange);
            }
        }
    }
    float c[V], s[V];
    auto position = [&](int f) -> int64_t {
        const int64_t p = a.positions[g.axis_of[f] * g.axis_stride + t];
        if (p < 0 || p >= g.table_len) {
            record_error(a.err, kDevIndexOutOfRange);
            return 0;
        }
        return p;
    };
    if (turns && kOneAxis) { // the lane's frequencies share a position: one row of the table
        using F = Pack<float, V>;
        const float* row = a.table + position(lane * V) * g.rot_dim + lane * V;
        const F fc = *reinterpret_cast<const F*>(row), fs = *reinterpret_cast<const F*>(row + half);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            c[j] = fc.e[j];
            s[j] = fs.e[j];
        }
    } else if (turns) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int f = lane * V + j;
            const float* row = a.table + position(f) * g.rot_dim + f;
            c[j] = row[0];
            s[j] = row[half];
        }
    }
#pragma unroll 1
    for (int h = group; h < heads; h += groups) {
        P n0, n1;
        if (h + groups < heads) {
            const T* row = source(h + groups);
            n0 = *reinterpret_cast<const P*>(row + e0);
            n1 = *reinterpret_cast<const P*>(row + e1);
        }
        if (turns && h < q_heads + kv_heads) {
            if constexpr (kPairs) { // pair j: elements 2j, 2j + 1 of the two packs together
                T x[2 * V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    x[j] = x0.e[j];
                    x[V + j] = x1.e[j];
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = to_f32(x[2 * j]), v = to_f32(x[2 * j + 1]);
                    x[2 * j] = from_f32<T>(u * c[j] - v * s[j]);
                    x[2 * j + 1] = from_f32<T>(v * c[j] + u * s[j]);
                }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    x0.e[j] = x[j];
                    x1.e[j] = x[V + j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float u = to_f32(x0.e[j]), v = to_f32(x1.e[j]);
                    x0.e[j] = from_f32<T>(u * c[j] - v * s[j]);
                    x1.e[j] = from_f32<T>(v * c[j] + u * s[j]);
                }
            }
        }
        auto store = [&](T* row) {
            *reinterpret_cast<P*>(row + e0) = x0;
            *reinterpret_cast<P*>(row + e1) = x1;
        };
        const int hk = h - q_heads;
        if (hk < 0) {
            store(static_cast<T*>(a.q_out) + t * g.qo_stride + h * g.qo_head_stride);
        } else if (hk < kv_heads) {
            if (a.k_out != nullptr) {
                store(static_cast<T*>(a.k_out) + t * g.ko_stride + hk * g.ko_head_stride);
            }
            if (a.k_cache != nullptr && k_at >= 0) {
                store(static_cast<T*>(a.k_cache) + k_at + hk * g.kc_head_stride);
            }
        } else if (v_at >= 0) {
            store(static_cast<T*>(a.v_cache) + v_at + (hk - kv_heads) * g.vc_head_stride);
        }
        x0 = n0;
        x1 = n1;
    }
}

template <typename T, int V, bool kPairs, bool kOneAxis>
void launch_rope_as(nb2_device* dev, const RopeArgs& a) {
    const nb2_rope_geom& g = a.g;
    const int64_t heads = g.q_heads + g.kv_heads + (a.v != nullptr ? g.kv_heads : 0);
    const int lanes = static_cast<int>(g.rot_dim / 2 / V + (g.head_dim - g.rot_dim) / 2 / V);
    // Heads of one thread: one while the tokens do not fill the GPU (latency
    // counts), else kWalk (the table's rows are then read 1/kWalk as often).
    const int64_t fill = static_cast<int64_t>(dev->num_sms) * 1024;
    const int walk = g.tokens * heads * lanes >= kWalk * fill ? kWalk : 1;
    int groups = static_cast<int>((heads + walk - 1) / walk);
    groups = std::min(groups, std::max(1, kRopeThreads / lanes));
    const int work = lanes * groups;
    const int per = std::max(1, kRopeThreads / work);
    const int64_t grid = (g.tokens + per - 1) / per;
    if (grid > 0x7fffffffLL) {
        fail(kStatusUnsupported, "rope: too many tokens");
    }
    rope_kernel<T, V, kPairs, kOneAxis>
        <<<static_cast<unsigned>(grid), (work * per + 31) / 32 * 32, 0, dev->stream>>>(a, lanes, groups, per);
    check_cuda(cudaGetLastError(), "rope launch");
}

template <typename T, int V>
void launch_rope(nb2_device* dev, const RopeArgs& a) {
    const nb2_rope_geom& g = a.g;
    bool one_axis = V > 1 && (reinterpret_cast<uintptr_t>(a.table) & 15) == 0 && g.rot_dim / 2 % 4 == 0;
    for (int64_t f = 0; f < g.rot_dim / 2; ++f) {
        one_axis = one_axis && g.axis_of[f] == g.axis_of[f / V * V];
    }
    if constexpr (V > 1) {
        if (one_axis) {
            g.interleaved ? launch_rope_as<T, V, true, true>(dev, a) : launch_rope_as<T, V, false, true>(dev, a);
            return;
        }
    }
    g.interleaved ? launch_rope_as<T, V, true, false>(dev, a) : launch_rope_as<T, V, false, false>(dev, a);
}

// V elements can be moved at once where the pairs and the copied rest come in
// whole packs and every address is aligned to a pack.
bool packs(const RopeArgs& a, int V, int64_t bytes) {
    const nb2_rope_geom& g = a.g;
    if (g.rot_dim / 2 % V != 0 || (g.head_dim - g.rot_dim) % (2 * V) != 0) {
        return false;
    }
    for (int64_t s : {g.q_stride, g.q_head_stride, g.k_stride, g.k_head_stride, g.qo_stride, g.qo_head_stride}) {
        if (s % V != 0) {
            return false;
        }
    }
    if (a.v != nullptr && (g.v_stride % V != 0 || g.v_head_stride % V != 0)) {
        return false;
    }
    if (a.k_out != nullptr && (g.ko_stride % V != 0 || g.ko_head_stride % V != 0)) {
        return false;
    }
    if (a.k_cache != nullptr) {
        for (int64_t s : {g.kc_block_stride, g.kc_place_stride, g.kc_head_stride, g.vc_block_stride,
                          g.vc_place_stride, g.vc_head_stride}) {
            if (s % V != 0) {
                return false;
            }
        }
    }
    const uintptr_t mask = static_cast<uintptr_t>(std::min<int64_t>(16, V * bytes) - 1);
    for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.q_out), static_cast<const void*>(a.k_out),
                          static_cast<const void*>(a.k_cache), static_cast<const void*>(a.v_cache)}) {
        if ((reinterpret_cast<uintptr_t>(p) & mask) != 0) {
            return false;
        }
    }
    return true;
}

template <typename T>
void pick_rope(nb2_device* dev, const RopeArgs& a) {
    constexpr int kWide = 16 / sizeof(T);
    if (packs(a, kWide, sizeof(T))) {
        launch_rope<T, kWide>(dev, a);
    } else if (kWide > 4 && packs(a, 4, sizeof(T))) {
        launch_rope<T, 4>(dev, a);
    } else {
        launch_rope<T, 1>(dev, a);
    }
}

} // namespace

void rope_append(nb2_device* dev, RopeArgs a) {
    if (a.g.tokens == 0) {
        return;
    }
    a.err = dev->err_word;
    if (a.g.dtype == kF32) {
        pick_rope<float>(dev, a);
    } else if (a.g.dtype == kF16) {
        pick_rope<__half>(dev, a);
    } else {
        pick_rope<__nv_bfloat16>(dev, a);
    }
}

} // namespace nb2
