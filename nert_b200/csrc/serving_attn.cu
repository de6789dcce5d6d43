// Attention of each request's new tokens over its paged cache and over the
// new tokens that its tree allows.
//
// One CTA per (new token, query head) walks the request's places in tiles of
// 128: a thread scores one place, the tile's maximum and sum update a running
// softmax, and every thread then adds the tile's values to its elements of the
// output. A place that the token does not see, or whose block id is out of
// range, has weight zero and is never read.

#include "serving.cuh"

namespace nb2 {

namespace {

constexpr int kSimpleThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kSimpleThreads) tree_attn_kernel(TreeAttnArgs a) {
    const nb2_tree_attn_geom& g = a.g;
    __shared__ float q[256], p[kSimpleThreads], red[kSimpleThreads / 32];
    __shared__ int64_t at[kSimpleThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t t = blockIdx.x;
    const int64_t h = blockIdx.y, kvh = h / (g.q_heads / g.kv_heads);
    const int D = static_cast<int>(g.head_dim);
    T* out = static_cast<T*>(a.out) + t * g.o_stride + h * g.o_head_stride;
    int lo = 0, hi = static_cast<int>(g.batch); // request of token t
    bool bad = false;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        (a.offsets[mid] <= t ? lo : hi) = mid;
    }
    const int64_t first = g.batch > 0 ? a.offsets[lo] : 0, end = g.batch > 0 ? a.offsets[lo + 1] : 0;
    const int64_t n = end - first, i = t - first;
    int64_t total = i >= 0 && i < n ? a.total[lo] : 0;
    if (total > 0 && (total < n || total > g.table_blocks * g.block_size || n > g.max_new)) {
        bad = true;
        total = 0;
    }
    const int64_t old = total - n;
    for (int d = tid; d < D; d += kSimpleThreads) {
        q[d] = to_f32(static_cast<const T*>(a.q)[t * g.q_stride + h * g.q_head_stride + d]);
    }
    __syncthreads();
    float m = -INFINITY, z = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int64_t j0 = 0; j0 < total; j0 += kSimpleThreads) {
        const int64_t j = j0 + tid;
        bool see = j < total;
        if (see && j >= old) {
            const int64_t k = j - old;
            see = a.mask == nullptr ? k <= i
                                    : k < 32 * g.mask_words && ((a.mask[t * g.mask_words + (k >> 5)] >> (k & 31)) & 1u);
        }
        int64_t block = -1;
        if (see) {
            block = a.table[lo * g.table_stride + j / g.block_size];
            if (block < 0 || block >= g.num_blocks) {
                bad = true;
                see = false;
            }
        }
        float s = -INFINITY;
        if (see) {
            const int64_t place = j % g.block_size;
            const T* k = static_cast<const T*>(a.kc) + block * g.kc_block_stride + place * g.kc_place_stride +
                         kvh * g.kc_head_stride;
            s = 0.0f;
            for (int d = 0; d < D; ++d) {
                s += q[d] * to_f32(k[d]);
            }
            s *= g.scale;
            at[tid] = block * g.vc_block_stride + place * g.vc_place_stride + kvh * g.vc_head_stride;
        } else {
            at[tid] = -1;
        }
        float top = s;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (lane == 0) {
            red[warp] = top;
        }
        __syncthreads();
        top = m;
        for (int w = 0; w < kSimpleThreads / 32; ++w) {
            top = fmaxf(top, red[w]);
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        p[tid] = expf(s - ref);
        __syncthreads();
        const float keep = expf(m - ref);
        m = top;
        z *= keep;
        o0 *= keep;
        o1 *= keep;
        for (int k = 0; k < kSimpleThreads; ++k) {
            if (at[k] < 0) {
                continue;
            }
            z += p[k];
            const T* v = static_cast<const T*>(a.vc) + at[k];
            if (tid < D) {
                o0 += p[k] * to_f32(v[tid]);
            }
            if (tid + kSimpleThreads < D) {
                o1 += p[k] * to_f32(v[tid + kSimpleThreads]);
            }
        }
        __syncthreads();
    }
    const float inv = z > 0.0f ? 1.0f / z : 0.0f;
    if (tid < D) {
        out[tid] = from_f32<T>(o0 * inv);
    }
    if (tid + kSimpleThreads < D) {
        out[tid + kSimpleThreads] = from_f32<T>(o1 * inv);
    }
    if (tid == 0 && a.lse != nullptr) {
        a.lse[t * g.q_heads + h] = z > 0.0f ? m + logf(z) : -INFINITY;
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    }
}

} // namespace

void tree_attention(nb2_device* dev, TreeAttnArgs a) {
    if (a.g.tokens == 0) {
        return;
    }
    a.err = dev->err_word;
    const dim3 grid(static_cast<unsigned>(a.g.tokens), static_cast<unsigned>(a.g.q_heads));
    if (a.g.dtype == kF32) {
        tree_attn_kernel<float><<<grid, kSimpleThreads, 0, dev->stream>>>(a);
    } else if (a.g.dtype == kF16) {
        tree_attn_kernel<__half><<<grid, kSimpleThreads, 0, dev->stream>>>(a);
    } else {
        tree_attn_kernel<__nv_bfloat16><<<grid, kSimpleThreads, 0, dev->stream>>>(a);
    }
    check_cuda(cudaGetLastError(), "tree attention launch");
}

} // namespace nb2
