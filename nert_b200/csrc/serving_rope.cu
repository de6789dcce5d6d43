// Rotary positions with several axes, fused with the cache write.
//
// Each pair (x1, x2) of a head is one complex number turned by the angle of
// its frequency at the position that the frequency's axis gives: six flops
// for two loads and two stores, so the kernel is bound by HBM: q, k and v
// once in and once out. The angles come as a table of cosines and sines in 32
// bits (the caller's: any base, scaling or length rule), gathered by position.
//
// A thread owns V consecutive frequencies of one token and kHeads heads of it,
// so cos and sin are loaded once for all of them and its 2 kHeads V-element
// loads are in flight together. Both halves of every pair are read before
// either is written, which is what makes the in-place form safe.

#include "serving.cuh"

namespace nb2 {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kHeads = 4;

// Where a row (one head of one token) starts, by its index over q, k, v heads.
template <typename T, int V>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeArgs a, int lanes, int groups, int tokens_per_cta) {
    using P = Pack<T, V>;
    const nb2_rope_geom& g = a.g;
    const int half = static_cast<int>(g.rot_dim / 2);
    const int turn = half / V; // lanes that turn pairs; the rest copy what is past rot_dim
    const int heads = static_cast<int>(g.q_heads + g.kv_heads + (a.v != nullptr ? g.kv_heads : 0));
    const int work = lanes * groups;
    const int local = static_cast<int>(threadIdx.x) / work;
    if (local >= tokens_per_cta) {
        return;
    }
    const int64_t t = static_cast<int64_t>(blockIdx.x) * tokens_per_cta + local;
    if (t >= g.tokens) {
        return;
    }
    int64_t block = -1, place = 0;
    if (a.slots != nullptr) {
        const int64_t slot = a.slots[t];
        if (slot >= 0) {
            block = slot / g.block_size;
            place = slot - block * g.block_size;
            if (block >= g.num_blocks) {
                record_error(a.err, kDevIndexOutOfRange);
                block = -1;
            }
        }
    }
    for (int w = static_cast<int>(threadIdx.x) - local * work; w < work; w += blockDim.x) {
        const int group = w / lanes, lane = w - group * lanes;
        const bool turns = lane < turn;
        // element offsets of the two packs in a head
        int e0, e1;
        if (!turns) {
            e0 = static_cast<int>(g.rot_dim) + (lane - turn) * 2 * V;
            e1 = e0 + V;
        } else if (g.interleaved) {
            e0 = lane * 2 * V;
            e1 = e0 + V;
        } else {
            e0 = lane * V;
            e1 = half + e0;
        }
        P x0[kHeads], x1[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            int h = group + i * groups;
            if (h < heads) {
                const T* row;
                if (h < g.q_heads) {
                    row = static_cast<const T*>(a.q) + t * g.q_stride + h * g.q_head_stride;
                } else if ((h -= static_cast<int>(g.q_heads)) < g.kv_heads) {
                    row = static_cast<const T*>(a.k) + t * g.k_stride + h * g.k_head_stride;
                } else {
                    row = static_cast<const T*>(a.v) + t * g.v_stride + (h - g.kv_heads) * g.v_head_stride;
                }
                x0[i] = *reinterpret_cast<const P*>(row + e0);
                x1[i] = *reinterpret_cast<const P*>(row + e1);
            }
        }
        float c[V], s[V];
        if (turns) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int f = lane * V + j;
                int64_t p = a.positions[g.axis_of[f] * g.axis_stride + t];
                if (p < 0 || p >= g.table_len) {
                    record_error(a.err, kDevIndexOutOfRange);
                    p = 0;
                }
                c[j] = a.table[p * g.rot_dim + f];
                s[j] = a.table[p * g.rot_dim + half + f];
            }
        }
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            int h = group + i * groups;
            if (h >= heads) {
                continue;
            }
            const bool is_v = h >= g.q_heads + g.kv_heads;
            if (turns && !is_v) {
                if (g.interleaved) {
                    // pair j sits at elements 2j, 2j + 1 of the two packs together
                    T* flat0 = x0[i].e;
                    T* flat1 = x1[i].e;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        T& u = 2 * j < V ? flat0[2 * j < V ? 2 * j : 0] : flat1[2 * j < V ? 0 : 2 * j - V];
                        T& v = 2 * j + 1 < V ? flat0[2 * j + 1 < V ? 2 * j + 1 : 0]
                                             : flat1[2 * j + 1 < V ? 0 : 2 * j + 1 - V];
                        const float p = to_f32(u), q = to_f32(v);
                        u = from_f32<T>(p * c[j] - q * s[j]);
                        v = from_f32<T>(q * c[j] + p * s[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float p = to_f32(x0[i].e[j]), q = to_f32(x1[i].e[j]);
                        x0[i].e[j] = from_f32<T>(p * c[j] - q * s[j]);
                        x1[i].e[j] = from_f32<T>(q * c[j] + p * s[j]);
                    }
                }
            }
            if (h < g.q_heads) {
                T* row = static_cast<T*>(a.q_out) + t * g.qo_stride + h * g.qo_head_stride;
                *reinterpret_cast<P*>(row + e0) = x0[i];
                *reinterpret_cast<P*>(row + e1) = x1[i];
                continue;
            }
            h -= static_cast<int>(g.q_heads);
            if (!is_v) {
                if (a.k_out != nullptr) {
                    T* row = static_cast<T*>(a.k_out) + t * g.ko_stride + h * g.ko_head_stride;
                    *reinterpret_cast<P*>(row + e0) = x0[i];
                    *reinterpret_cast<P*>(row + e1) = x1[i];
                }
                if (a.k_cache != nullptr && block >= 0) {
                    T* row = static_cast<T*>(a.k_cache) + block * g.kc_block_stride + place * g.kc_place_stride +
                             h * g.kc_head_stride;
                    *reinterpret_cast<P*>(row + e0) = x0[i];
                    *reinterpret_cast<P*>(row + e1) = x1[i];
                }
            } else if (block >= 0) {
                h -= static_cast<int>(g.kv_heads);
                T* row = static_cast<T*>(a.v_cache) + block * g.vc_block_stride + place * g.vc_place_stride +
                         h * g.vc_head_stride;
                *reinterpret_cast<P*>(row + e0) = x0[i];
                *reinterpret_cast<P*>(row + e1) = x1[i];
            }
        }
    }
}

template <typename T, int V>
void launch_rope(nb2_device* dev, const RopeArgs& a) {
    const nb2_rope_geom& g = a.g;
    const int64_t heads = g.q_heads + g.kv_heads + (a.v != nullptr ? g.kv_heads : 0);
    const int lanes = static_cast<int>(g.rot_dim / 2 / V + (g.head_dim - g.rot_dim) / 2 / V);
    const int groups = static_cast<int>((heads + kHeads - 1) / kHeads);
    const int work = lanes * groups;
    const int per = std::max(1, kRopeThreads / work);
    const int64_t grid = (g.tokens + per - 1) / per;
    if (grid > 0x7fffffffLL) {
        fail(kStatusUnsupported, "rope: too many tokens");
    }
    const int threads = std::min(kRopeThreads, (work * per + 31) / 32 * 32);
    rope_kernel<T, V><<<static_cast<unsigned>(grid), threads, 0, dev->stream>>>(a, lanes, groups, per);
    check_cuda(cudaGetLastError(), "rope launch");
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
