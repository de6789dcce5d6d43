// Rotary positions with several axes, fused with the cache write.
//
// Each pair (x1, x2) of a head is one complex number turned by the angle of
// its frequency at the position that the frequency's axis gives: six flops
// for two loads and two stores, so the kernel is bound by HBM: q, k and v
// once in and once out. The angles come as a table of cosines and sines in 32
// bits (the caller's: any base, scaling or length rule), gathered by position.
//
// A CTA takes heads of q, of k or of v. A thread owns V consecutive frequencies of one token and walks over some of
// the token's heads, so cos and sin are loaded once for all of them; the next head's two V-element packs are loaded
// before the present one is turned and stored. Both halves of every pair are read before either is written, which
// is what makes the in-place form safe. What bounds the kernel is how many loads an SM holds in flight, that is,
// registers: a rolled walk over one tensor needs about 64 (1,024 threads of 64 bytes each; ptxas spills 8 bytes of the
// bfloat16 half-split form, 44 where axes change inside a lane, and nothing of the others).
// Measured at 16,001 tokens, 28 + 4 + 4 heads of 128 in bfloat16 (297 MB): 56 us, 5.3 TB/s. Walking over all three
// tensors in the same registers took 72 us, four heads unrolled in 122 registers 117 us, 48 registers with spills 94 us.

#include "serving.cuh"

namespace nb2 {

namespace {

constexpr int kRopeThreads = 256;
// Heads of a thread where there are tokens enough: the table's rows are read that much less often. 16-bit types: 8 heads
// 56 us, 4 heads 60, 2 heads 69; float32 (6,304 tokens, 12 + 12 heads of 64): 2 heads 16 us, 4 heads 18, 8 heads 20.
constexpr int walk_of(size_t bytes) { return bytes == 2 ? 8 : 2; }

// How the heads of one tensor are spread over CTAs.
struct Spread {
    int heads;
    int groups; // threads that share a token's heads at one lane
    int tokens; // of a CTA
    int64_t ctas;
};

template <typename T, int V, bool kPairs, bool kOneAxis>
__global__ void __launch_bounds__(kRopeThreads, 4)
    rope_kernel(const __grid_constant__ RopeArgs a, int lanes, const __grid_constant__ Spread sq,
                const __grid_constant__ Spread sk) {
    using P = Pack<T, V>;
    const nb2_rope_geom& g = a.g;
    const int64_t cta = blockIdx.x;
    const int role = cta < sq.ctas ? 0 : cta < sq.ctas + sk.ctas ? 1 : 2; // q, k, v
    const int heads = role == 0 ? sq.heads : sk.heads, groups = role == 0 ? sq.groups : sk.groups;
    const int tokens = role == 0 ? sq.tokens : sk.tokens, work = lanes * groups;
    const int local = static_cast<int>(threadIdx.x) / work;
    const int64_t t = (role == 0 ? cta : role == 1 ? cta - sq.ctas : cta - sq.ctas - sk.ctas) * tokens + local;
    if (local >= tokens || t >= g.tokens) {
        return;
    }
    const int half = static_cast<int>(g.rot_dim / 2);
    const int turn = half / V; // lanes that turn pairs; the rest copy what is past rot_dim
    const int w = static_cast<int>(threadIdx.x) - local * work;
    const int group = w / lanes, lane = w - group * lanes;
    const bool turns = role < 2 && lane < turn;
    // element offsets of the two packs in a head
    const int e0 = lane >= turn ? static_cast<int>(g.rot_dim) + (lane - turn) * 2 * V : kPairs ? lane * 2 * V : lane * V;
    const int e1 = lane < turn && !kPairs ? half + e0 : e0 + V;

    const int64_t src_head = role == 0 ? g.q_head_stride : role == 1 ? g.k_head_stride : g.v_head_stride;
    const T* src = (role == 0   ? static_cast<const T*>(a.q) + t * g.q_stride
                    : role == 1 ? static_cast<const T*>(a.k) + t * g.k_stride
                                : static_cast<const T*>(a.v) + t * g.v_stride) +
                   group * src_head;
    P x0 = *reinterpret_cast<const P*>(src + e0), x1 = *reinterpret_cast<const P*>(src + e1);

    // where the heads go: out, and the token's place in a cache (null: nowhere)
    T *out = nullptr, *cache = nullptr;
    int64_t out_head = 0, cache_head = 0;
    if (role == 0) {
        out_head = g.qo_head_stride;
        out = static_cast<T*>(a.q_out) + t * g.qo_stride;
    } else {
        if (role == 1 && a.k_out != nullptr) {
            out_head = g.ko_head_stride;
            out = static_cast<T*>(a.k_out) + t * g.ko_stride;
        }
        const int slot = a.slots != nullptr ? a.slots[t] : -1;
        if (slot >= 0) {
            const int size = static_cast<int>(g.block_size);
            const int block = slot / size, place = slot - block * size;
            if (block >= g.num_blocks) {
                record_error(a.err, kDevIndexOutOfRange);
            } else if (role == 1) {
                cache_head = g.kc_head_stride;
                cache = static_cast<T*>(a.k_cache) + block * g.kc_block_stride + place * g.kc_place_stride;
            } else {
                cache_head = g.vc_head_stride;
                cache = static_cast<T*>(a.v_cache) + block * g.vc_block_stride + place * g.vc_place_stride;
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
        src += groups * src_head;
        if (h + groups < heads) {
            n0 = *reinterpret_cast<const P*>(src + e0);
            n1 = *reinterpret_cast<const P*>(src + e1);
        }
        if (turns) {
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
        if (out != nullptr) {
            T* row = out + h * out_head;
            *reinterpret_cast<P*>(row + e0) = x0;
            *reinterpret_cast<P*>(row + e1) = x1;
        }
        if (cache != nullptr) {
            T* row = cache + h * cache_head;
            *reinterpret_cast<P*>(row + e0) = x0;
            *reinterpret_cast<P*>(row + e1) = x1;
        }
        x0 = n0;
        x1 = n1;
    }
}

template <typename T, int V, bool kPairs, bool kOneAxis>
void launch_rope_as(nb2_device* dev, const RopeArgs& a) {
    const nb2_rope_geom& g = a.g;
    const int lanes = static_cast<int>(g.rot_dim / 2 / V + (g.head_dim - g.rot_dim) / 2 / V);
    const int64_t heads = g.q_heads + g.kv_heads + (a.v != nullptr ? g.kv_heads : 0);
    // one head a thread while the tokens do not fill the GPU (latency counts)
    constexpr int kWalk = walk_of(sizeof(T));
    const int walk = g.tokens * heads * lanes >= kWalk * static_cast<int64_t>(dev->num_sms) * 1024 ? kWalk : 1;
    auto spread = [&](int64_t n) {
        Spread s{};
        s.heads = static_cast<int>(n);
        s.groups = std::min((s.heads + walk - 1) / walk, std::max(1, kRopeThreads / lanes));
        s.tokens = std::max(1, kRopeThreads / (lanes * s.groups));
        s.ctas = (g.tokens + s.tokens - 1) / s.tokens;
        return s;
    };
    const Spread sq = spread(g.q_heads), sk = spread(g.kv_heads);
    const int64_t grid = sq.ctas + sk.ctas * (a.v != nullptr ? 2 : 1);
    if (grid > 0x7fffffffLL) {
        fail(kStatusUnsupported, "RopeAppend: too many tokens");
    }
    rope_kernel<T, V, kPairs, kOneAxis><<<static_cast<unsigned>(grid), kRopeThreads, 0, dev->stream>>>(a, lanes, sq, sk);
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
    a.err = dev->error_word();
    if (a.g.dtype == kF32) {
        pick_rope<float>(dev, a);
    } else if (a.g.dtype == kF16) {
        pick_rope<__half>(dev, a);
    } else {
        pick_rope<__nv_bfloat16>(dev, a);
    }
}

} // namespace nb2
