// Attention of each request's new tokens over its paged cache and over the
// new tokens that its tree allows.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q.k_j
//
// in one pass over the cache with the running maximum m and sum of each row.
// A row is one query head of one new token; the rows of a request that share a
// key/value head (its n tokens times the group of q_heads/kv_heads) are one
// matrix, cut into blocks of 16 WR rows, so a key or value read once from HBM serves
// them all. Few rows: bound by HBM (4 flops a row for each element of the cache);
// many: by the tensor cores.
//
// Work split. The lengths are on the device, so the split is made there: an item is (request,
// key/value head, row block), its units the request's tiles of KT places, and the units of all
// items, in order, are cut into equal spans, one a CTA (a grid that fits the GPU at once), so every
// CTA reads the same number of tiles whatever the lengths. An item inside one span is finished by
// its CTA; of one that is cut, each CTA leaves (O, m, sum) in its own slot (a span cuts at most its
// first and its last item: two slots a CTA) and the CTA that arrives last adds the pieces in span
// order, so the result does not depend on which one that is (where pieces are many, a second launch adds them in the same order).
//
// Within a CTA, WR x WK warps: row group x part of the tile's places. The warps of a row group run
// the softmax on their own places and join at the end of the item. Tiles come by 16-byte cp.async
// through a ring of NS stages, the addresses of a tile's rows looked up in the block table two tiles
// ahead of its copies.
//
// Measured: 4 single tokens over 60-2,000 places, 32/8 heads of 128 in bfloat16 (16 MB): 16 us, bound by latencies (of 29,000
// clocks with cold caches the lengths take 3,000, q 2,400, the first tile 5,000, the join 10,000). 8 trees of 5-24
// tokens over 100-3,000 places, 12 heads of 64 in float32 (76 MB): 55 us, 1.4 TB/s, bound by the three tf32 products of
// each product and their operands' splits at one CTA an SM (233 registers). Heads of more than 128 elements do not fit
// 255 registers: 560-732 bytes a thread are spilled in 16-bit types, 208-232 in float32 (64-element heads in blocks of 32 rows
// spill 192, to leave an SM two CTAs; the rest at most 48).

#include "serving_attn.cuh"

#include <type_traits>

namespace nb2 {

namespace {

// ---- instructions ----------------------------------------------------------------

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    const int n = live ? 16 : 0; // 0: sixteen zero bytes
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ void mma_tf32_8(float (&d)[4], const float (&a)[4], float b0, float b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(__float_as_uint(a[0])), "r"(__float_as_uint(a[1])), "r"(__float_as_uint(a[2])),
                   "r"(__float_as_uint(a[3])), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}

// x = high + low, high rounded to tf32 (nearest, ties away), low exact; the tensor cores read low's first 11 bits, so
// what is lost is 2^-21 of x. In whole-number instructions: with the conversion instruction 8 requests of up to 24
// tokens (12 heads of 64) took 61 us, so 57.
__device__ __forceinline__ void split_tf32(float x, float& high, float& low) {
    high = __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u);
    low = x - high;
}

// Whether 0 times x is not 0 in the products: infinities and NaN, and in float32 what split_tf32 rounds to infinity.
template <typename T>
__device__ __forceinline__ bool spoils(T x) {
    if constexpr (sizeof(T) == 4) {
        return (__float_as_uint(x) & 0x7fffffffu) + 0x1000u >= 0x7f800000u;
    } else {
        return !isfinite(to_f32(x));
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// ---- the kernel -----------------------------------------------------------------

template <typename T, int DP, int WR, int WK>
struct Shape {
    static constexpr bool kF32Type = sizeof(T) == 4;
    static constexpr int kWarps = WR * WK, kThreads = 32 * kWarps;
    static constexpr int RT = 16 * WR;                    // rows of a block
    static constexpr int KT = kF32Type && DP > 64 ? 32 : 64; // places of a tile
    static constexpr int KW = KT / WK;                    // places of a warp
    static constexpr int kChunks = DP * sizeof(T) / 16;   // 16-byte chunks of a row
    static constexpr int kRow = DP * sizeof(T) + (kF32Type ? 16 : 0); // bytes of a row in shared memory
    static constexpr int kTile = KT * kRow;
    // stages of the ring: what fits beside Q
    static constexpr int NS = kF32Type && DP == 64 ? 3 : DP == 64 ? 4 : DP == 128 || (WR == 1 && !kF32Type) ? 3 : 2;
    static constexpr int kRing = NS * 2 * kTile;
    static constexpr int kQ = RT * kRow * (kF32Type ? 2 : 1);
    static constexpr int kJoin = WK * RT * DP * 4;        // the warps' sums, over the ring
    static constexpr int kSmem = (kRing > kJoin ? kRing : kJoin) + kQ + 1024;
    // CTAs that shared memory lets an SM hold: registers are kept to what they leave
    static constexpr int kPerSm = (kThreads == 128 || (WR == 2 && DP == 64)) && (kSmem + 8192) * 2 <= 227 * 1024 ? 2 : 1;
};

template <typename T, int DP, int WR, int WK>
__global__ void __launch_bounds__(32 * WR * WK, Shape<T, DP, WR, WK>::kPerSm)
    tree_attn_kernel(const __grid_constant__ TreeAttnArgs a, int group, int sms, float* part_o, float2* part_ml,
                     uint32_t* tickets) {
    using S = Shape<T, DP, WR, WK>;
    constexpr int NT = S::kThreads, RT = S::RT, KT = S::KT, KW = S::KW, NS = S::NS;
    constexpr int NB = KW / 8; // 8-place column blocks of a warp's scores
    extern __shared__ __align__(1024) uint8_t attn_dyn[];
    uint8_t* ring = attn_dyn;
    uint8_t* qs = attn_dyn + (S::kRing > S::kJoin ? S::kRing : S::kJoin);
    __shared__ int64_t red[NT / 32];
    // element offsets of the rows of the tiles in the ring and of the next, -1: no such place
    __shared__ int64_t k_at[NS + 1][KT], v_at[NS + 1][KT];
    __shared__ uint32_t valid_of[NS + 1][KT / 32]; // bits of the tiles' places that are there
    __shared__ unsigned long long odd_keys;        // places of the tile whose values are not finite
    __shared__ float2 warp_ml[WK][RT];
    __shared__ int64_t found[2];
    __shared__ int is_last;

    const nb2_tree_attn_geom& g = a.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wr = warp / WK, wk = warp % WK;
    const int gq = lane >> 2, cq = lane & 3;
    const int64_t cta = blockIdx.x;
    const int D = static_cast<int>(g.head_dim);
    const float scale2 = g.scale * kLog2e;
    bool bad = false;

    const Span span = find_span<RT, KT, NT>(a, group, sms, red, found, bad);
    spare_tokens<T>(a, tid, NT);
    const int64_t W = span.W, grid = span.grid, w1 = span.w1;
    int r = span.request;
    int64_t r_unit = span.request_unit; // first unit of request r
    Request rq{};
    if (span.w0 < w1) {
        rq = request_at<RT, KT>(a, r, group);
    }
    for (int64_t w = span.w0; w < w1;) { // w: the first unit not yet looked at
        while (w >= r_unit + rq.units(g.kv_heads)) {
            r_unit += rq.units(g.kv_heads);
            rq = request_at<RT, KT>(a, ++r, group);
        }
        // ---- the item and this CTA's tiles of it
        const int64_t item = (w - r_unit) / rq.per_item();
        const int64_t item_w0 = r_unit + item * rq.per_item() + rq.extra, item_w1 = item_w0 + rq.tiles;
        const int64_t from = max(w, item_w0);
        w = min(w1, item_w1);
        if (from >= w) {
            continue; // the span ends before the item's first tile
        }
        const int64_t kvh = item / rq.row_blocks;
        const int rb = static_cast<int>(item - kvh * rq.row_blocks);
        const int t_begin = static_cast<int>(from - item_w0);
        const int t_end = static_cast<int>(w - item_w0);
        const int rows = min(RT, rq.n * group - rb * RT);
        const int old = rq.total - rq.n; // -n where the lengths are wrong: then total is 0 and no place is seen
        const int32_t* table = a.table + r * g.table_stride;

        __syncthreads(); // the last item's use of shared memory is over
        // block of place j of this request, for the row addresses of a tile; -1: none there
        auto look_up = [&](int tile) -> int {
            const int j = tile * KT + tid;
            return tid < KT && tile < t_end && j < rq.total ? table[j / static_cast<int>(g.block_size)] : -1;
        };
        int next = look_up(t_begin);
        // ---- Q rows into shared memory, zero past the block's rows and head_dim
#pragma unroll 1
        for (int i = tid; i < RT * S::kChunks; i += NT) {
            const int row = i / S::kChunks, ch = i - row * S::kChunks;
            constexpr int E = 16 / sizeof(T);
            uint4 x = make_uint4(0, 0, 0, 0);
            if (row < rows && ch * E < D) {
                const int rho = rb * RT + row, tok = rho / group;
                const int64_t h = kvh * group + (rho - tok * group);
                x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (rq.first + tok) * g.q_stride +
                                                    h * g.q_head_stride + ch * E);
            }
            if constexpr (S::kF32Type) { // as tf32 high and low parts
                float f[4] = {__uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w)};
                float hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    split_tf32(f[e], hi[e], lo[e]);
                }
                *reinterpret_cast<float4*>(qs + row * S::kRow + ch * 16) = make_float4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<float4*>(qs + (RT + row) * S::kRow + ch * 16) = make_float4(lo[0], lo[1], lo[2], lo[3]);
            } else {
                *reinterpret_cast<uint4*>(qs + row * S::kRow + ((ch ^ (row & 7)) << 4)) = x;
            }
        }
        // rows of this thread's fragments: the token and its mask row
        int tok0, tok1;
        const uint32_t *mask0 = nullptr, *mask1 = nullptr;
        {
            const int l0 = wr * 16 + gq, l1 = l0 + 8;
            tok0 = l0 < rows ? (rb * RT + l0) / group : -1;
            tok1 = l1 < rows ? (rb * RT + l1) / group : -1;
            if (a.mask != nullptr) {
                mask0 = a.mask + (rq.first + max(tok0, 0)) * g.mask_words;
                mask1 = a.mask + (rq.first + max(tok1, 0)) * g.mask_words;
            }
        }

        auto place_rows = [&](int tile, int block) {
            if (tid < KT && tile < t_end) {
                const int at = tile % (NS + 1), j = tile * KT + tid;
                int64_t ka = -1, va = -1;
                const bool there = block >= 0 && block < g.num_blocks;
                const uint32_t valid = __ballot_sync(0xffffffffu, there);
                if (lane == 0) {
                    valid_of[at][warp] = valid;
                }
                bad |= !there && j < rq.total;
                if (there) {
                    const int p = j % static_cast<int>(g.block_size);
                    ka = block * g.kc_block_stride + p * g.kc_place_stride + kvh * g.kc_head_stride;
                    va = block * g.vc_block_stride + p * g.vc_place_stride + kvh * g.vc_head_stride;
                }
                k_at[at][tid] = ka;
                v_at[at][tid] = va;
            }
        };
        auto copy_tile = [&](int tile) {
            if (tile < t_end) {
                const int st = tile % NS, at = tile % (NS + 1);
                const uint32_t dst = smem_u32(ring + st * 2 * S::kTile);
                constexpr int kPer = NT / S::kChunks > 0 ? NT / S::kChunks : 1; // rows of one pass
                static_assert(NT % S::kChunks == 0 && KT % kPer == 0, "the threads cover whole rows");
                const int ch = tid % S::kChunks, row0 = tid / S::kChunks;
                const bool in = ch * static_cast<int>(16 / sizeof(T)) < D;
                const T* kc = static_cast<const T*>(a.kc) + ch * (16 / sizeof(T));
                const T* vc = static_cast<const T*>(a.vc) + ch * (16 / sizeof(T));
#pragma unroll 4
                for (int i = 0; i < KT / kPer; ++i) {
                    const int row = row0 + i * kPer;
                    const int64_t ka = k_at[at][row], va = v_at[at][row];
                    const uint32_t off = row * S::kRow + (S::kF32Type ? ch * 16 : ((ch ^ (row & 7)) << 4));
                    const bool live = in && ka >= 0;
                    cp_async16(dst + off, kc + (live ? ka : 0), live);
                    cp_async16(dst + S::kTile + off, vc + (live ? va : 0), live);
                }
            }
            cp_commit();
        };

        place_rows(t_begin, next);
        next = look_up(t_begin + 1);
        __syncthreads(); // Q is there

        uint32_t qf[S::kF32Type ? 1 : DP / 16][4];
        if constexpr (!S::kF32Type) {
            const int row = wr * 16 + (lane & 15);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                ldsm4(qf[k], smem_u32(qs + row * S::kRow + (((2 * k + (lane >> 4)) ^ (row & 7)) << 4)));
            }
        }
        float o[DP / 8][4];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        }
        float m0 = -INFINITY, m1 = -INFINITY, z0 = 0.0f, z1 = 0.0f; // of rows gq and gq + 8, this thread's columns

        // The first NS - 1 rounds only fill the ring. A CTA may meet few tiles, so what runs once is
        // kept small: its instructions come from L2.
#pragma unroll 1
        for (int tile = t_begin - (NS - 1); tile < t_end; ++tile) {
            if (tile >= t_begin) {
                cp_wait<NS - 2>();
            }
            __syncthreads(); // the tile has landed, the stage of the one before is free, the next addresses are there
            copy_tile(tile + NS - 1);
            place_rows(tile + NS, next);
            next = look_up(tile + NS + 1);
            if (tile < t_begin) {
                continue;
            }
            const int st = tile % NS, at = tile % (NS + 1);
            const int j0 = tile * KT;
            bool plain = j0 + KT <= old;
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) {
                plain = plain && valid_of[at][i] == 0xffffffffu;
            }
            uint8_t* kt = ring + st * 2 * S::kTile;
            uint8_t* vt = kt + S::kTile;
            uint64_t odd = 0; // places whose values are not finite
            if (!plain) {
                // Values that are not finite (or not in tf32) would reach the rows that do not
                // see them as 0 * inf: taken out of the tile here, added for the rows that do below.
                if (tid == 0) {
                    odd_keys = 0;
                }
                __syncthreads();
#pragma unroll 1
                for (int i = tid; i < KT * S::kChunks; i += NT) {
                    const int row = i / S::kChunks, ch = i - row * S::kChunks;
                    const T* e = reinterpret_cast<const T*>(vt + row * S::kRow + ch * 16);
                    bool found_odd = false;
#pragma unroll
                    for (int x = 0; x < static_cast<int>(16 / sizeof(T)); ++x) {
                        found_odd |= spoils(e[x]);
                    }
                    if (found_odd) {
                        atomicOr(&odd_keys, 1ull << row);
                    }
                }
                __syncthreads();
                odd = odd_keys;
                if (odd != 0) {
#pragma unroll 1
                    for (int i = tid; i < KT * S::kChunks; i += NT) {
                        const int row = i / S::kChunks, ch = i - row * S::kChunks;
                        if ((odd >> row) & 1) {
                            *reinterpret_cast<uint4*>(vt + row * S::kRow + ch * 16) = make_uint4(0, 0, 0, 0);
                        }
                    }
                    __syncthreads();
                }
            }
            // ---- scores of this warp's places
            float s[NB][4];
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
            }
            if constexpr (S::kF32Type) {
#pragma unroll 4
                for (int k = 0; k < DP / 16; ++k) {
                    // dims 16k + 4c .. + 3 of a thread: the contraction's order is free, so k index c and
                    // c + 4 of the two steps are dims 4c, 4c + 1 and 4c + 2, 4c + 3
                    const uint8_t* qa = qs + (wr * 16 + gq) * S::kRow + (4 * k + cq) * 16;
                    const float4 h0 = *reinterpret_cast<const float4*>(qa);
                    const float4 h1 = *reinterpret_cast<const float4*>(qa + 8 * S::kRow);
                    const float4 l0 = *reinterpret_cast<const float4*>(qa + RT * S::kRow);
                    const float4 l1 = *reinterpret_cast<const float4*>(qa + (RT + 8) * S::kRow);
                    const float ah0[4] = {h0.x, h1.x, h0.y, h1.y}, ah1[4] = {h0.z, h1.z, h0.w, h1.w};
                    const float al0[4] = {l0.x, l1.x, l0.y, l1.y}, al1[4] = {l0.z, l1.z, l0.w, l1.w};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const float4 x = *reinterpret_cast<const float4*>(kt + (wk * KW + nb * 8 + gq) * S::kRow +
                                                                          (4 * k + cq) * 16);
                        float bx, by, bz, bw, lx, ly, lz, lw;
                        split_tf32(x.x, bx, lx);
                        split_tf32(x.y, by, ly);
                        split_tf32(x.z, bz, lz);
                        split_tf32(x.w, bw, lw);
                        // the tensor cores truncate where they add: chains are kept short and summed
                        // in round-to-nearest (one long chain measured twice the error)
                        float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_tf32_8(t, al0, bx, by);
                        mma_tf32_8(t, ah0, lx, ly);
                        mma_tf32_8(t, al1, bz, bw);
                        mma_tf32_8(t, ah1, lz, lw);
                        mma_tf32_8(t, ah0, bx, by);
                        mma_tf32_8(t, ah1, bz, bw);
                        s[nb][0] += t[0];
                        s[nb][1] += t[1];
                        s[nb][2] += t[2];
                        s[nb][3] += t[3];
                    }
                }
            } else {
                const uint32_t kb = smem_u32(kt);
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
                    for (int nb = 0; nb < NB; nb += 2) {
                        const int row = wk * KW + nb * 8 + ((lane >> 4) << 3) + (lane & 7);
                        uint32_t b[4];
                        ldsm4(b, kb + row * S::kRow + (((2 * k + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
                        mma16<T>(s[nb], qf[k], b[0], b[1]);
                        mma16<T>(s[nb + 1], qf[k], b[2], b[3]);
                    }
                }
            }
            // ---- running softmax in base 2
            if (plain) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[nb][e] *= scale2;
                    }
                }
            } else {
                // the warp's places (at most 32) that the rows' tokens see
                const int first_col = wk * KW;
                const uint32_t there = valid_of[at][first_col / 32] >> (first_col % 32);
                const uint32_t see0 = tok0 >= 0 ? there & see_bits(mask0, g.mask_words, tok0, j0 + first_col - old) : 0u;
                const uint32_t see1 = tok1 >= 0 ? there & see_bits(mask1, g.mask_words, tok1, j0 + first_col - old) : 0u;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t see = e < 2 ? see0 : see1;
                        s[nb][e] = (see >> (nb * 8 + 2 * cq + (e & 1))) & 1u ? s[nb][e] * scale2 : -INFINITY;
                    }
                }
            }
            float n0 = m0, n1 = m1;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                n0 = fmaxf(n0, fmaxf(s[nb][0], s[nb][1]));
                n1 = fmaxf(n1, fmaxf(s[nb][2], s[nb][3]));
            }
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 1));
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 1));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2));
            const float ref0 = n0 == -INFINITY ? 0.0f : n0, ref1 = n1 == -INFINITY ? 0.0f : n1;
            const float keep0 = exp2_fast(m0 - ref0), keep1 = exp2_fast(m1 - ref1);
            m0 = n0;
            m1 = n1;
            z0 *= keep0;
            z1 *= keep1;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                s[nb][0] = exp2_fast(s[nb][0] - ref0);
                s[nb][1] = exp2_fast(s[nb][1] - ref0);
                s[nb][2] = exp2_fast(s[nb][2] - ref1);
                s[nb][3] = exp2_fast(s[nb][3] - ref1);
                z0 += s[nb][0] + s[nb][1];
                z1 += s[nb][2] + s[nb][3];
            }
            if constexpr (!S::kF32Type) {
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    o[i][0] *= keep0;
                    o[i][1] *= keep0;
                    o[i][2] *= keep1;
                    o[i][3] *= keep1;
                }
            }
            // ---- O += P V
            if constexpr (S::kF32Type) {
                float ph[NB][4], pl[NB][4];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    // k index c and c + 4 are places 2c and 2c + 1: the layout the scores already have
                    const float p[4] = {s[nb][0], s[nb][2], s[nb][1], s[nb][3]};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        split_tf32(p[e], ph[nb][e], pl[nb][e]);
                    }
                }
                const uint8_t* vr = vt + (wk * KW + 2 * cq) * S::kRow + gq * 4;
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const float x = *reinterpret_cast<const float*>(vr + nb * 8 * S::kRow + i * 32);
                        const float y = *reinterpret_cast<const float*>(vr + (nb * 8 + 1) * S::kRow + i * 32);
                        float xh, yh, xl, yl;
                        split_tf32(x, xh, xl);
                        split_tf32(y, yh, yl);
                        mma_tf32_8(t, pl[nb], xh, yh);
                        mma_tf32_8(t, ph[nb], xl, yl);
                        mma_tf32_8(t, ph[nb], xh, yh);
                    }
                    o[i][0] = fmaf(o[i][0], keep0, t[0]);
                    o[i][1] = fmaf(o[i][1], keep0, t[1]);
                    o[i][2] = fmaf(o[i][2], keep1, t[2]);
                    o[i][3] = fmaf(o[i][3], keep1, t[3]);
                }
            } else {
                const uint32_t vb = smem_u32(vt);
#pragma unroll
                for (int nb = 0; nb < NB; nb += 2) {
                    // weights to the cache's type: at most u off each, which the sum over places averages; the
                    // sum z keeps all their bits
                    const uint32_t p[4] = {pack2<T>(s[nb][0], s[nb][1]), pack2<T>(s[nb][2], s[nb][3]),
                                           pack2<T>(s[nb + 1][0], s[nb + 1][1]), pack2<T>(s[nb + 1][2], s[nb + 1][3])};
                    const int row = wk * KW + nb * 8 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) {
                        uint32_t b[4];
                        ldsm4_t(b, vb + row * S::kRow + (((2 * i + (lane >> 4)) ^ (row & 7)) << 4));
                        mma16<T>(o[2 * i], p, b[0], b[1]);
                        mma16<T>(o[2 * i + 1], p, b[2], b[3]);
                    }
                }
            }
            // values that are not finite, for the rows that see them
            uint64_t mine = (odd >> (wk * KW)) & ((uint64_t{1} << KW) - 1);
#pragma unroll 1
            for (; mine != 0; mine &= mine - 1) { // the same for the whole warp
                const int col = __ffsll(static_cast<long long>(mine)) - 1, holder = (lane & 28) | ((col & 7) >> 1);
                float p0 = 0.0f, p1 = 0.0f;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    if (nb == col >> 3) {
                        p0 = (col & 1) != 0 ? s[nb][1] : s[nb][0];
                        p1 = (col & 1) != 0 ? s[nb][3] : s[nb][2];
                    }
                }
                p0 = __shfl_sync(0xffffffffu, p0, holder);
                p1 = __shfl_sync(0xffffffffu, p1, holder);
                const T* v = static_cast<const T*>(a.vc) + v_at[at][wk * KW + col] + 2 * cq;
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    if (i * 8 < D) {
                        const float x0 = to_f32(v[i * 8]), x1 = to_f32(v[i * 8 + 1]);
                        o[i][0] += p0 > 0.0f ? p0 * x0 : 0.0f;
                        o[i][1] += p0 > 0.0f ? p0 * x1 : 0.0f;
                        o[i][2] += p1 > 0.0f ? p1 * x0 : 0.0f;
                        o[i][3] += p1 > 0.0f ? p1 * x1 : 0.0f;
                    }
                }
            }
        }
        cp_wait<0>();
        __syncthreads();

        // ---- join the warps of each row group: sums over the ring's memory
        z0 += __shfl_xor_sync(0xffffffffu, z0, 1);
        z0 += __shfl_xor_sync(0xffffffffu, z0, 2);
        z1 += __shfl_xor_sync(0xffffffffu, z1, 1);
        z1 += __shfl_xor_sync(0xffffffffu, z1, 2);
        float* join = reinterpret_cast<float*>(ring); // [WK][RT][DP]
        {
            const int l0 = wr * 16 + gq;
            if (cq == 0) {
                warp_ml[wk][l0] = make_float2(m0, z0);
                warp_ml[wk][l0 + 8] = make_float2(m1, z1);
            }
            float* d0 = join + (wk * RT + l0) * DP + 2 * cq;
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) {
                *reinterpret_cast<float2*>(d0 + i * 8) = make_float2(o[i][0], o[i][1]);
                *reinterpret_cast<float2*>(d0 + 8 * DP + i * 8) = make_float2(o[i][2], o[i][3]);
            }
        }
        __syncthreads();
        const bool whole = t_begin == 0 && t_end == rq.tiles;
        const int my_slot = static_cast<int>(2 * cta) + (t_begin == 0 ? 1 : 0);
        for (int i = tid; i < rows * (DP / 4); i += NT) {
            const int row = i / (DP / 4), d = (i - row * (DP / 4)) * 4;
            if (d >= D) {
                continue;
            }
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                m = fmaxf(m, warp_ml[k][row].x);
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            float z = 0.0f;
            float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float2 ml = warp_ml[k][row];
                const float f = exp2_fast(ml.x - ref);
                const float4 y = *reinterpret_cast<const float4*>(join + (k * RT + row) * DP + d);
                z += f * ml.y;
                if (f != 0.0f) { // a part that saw nothing adds nothing
                    x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
                }
            }
            if (whole) {
                store_row4<T>(a, rq.first, kvh, group, rb * RT + row, d, x, m, z);
            } else {
                *reinterpret_cast<float4*>(part_o + (static_cast<int64_t>(my_slot) * RT + row) * DP + d) = x;
                if (d == 0) {
                    part_ml[static_cast<int64_t>(my_slot) * RT + row] = make_float2(m, z);
                }
            }
        }
        if (!whole && tickets != nullptr) { // null: a launch of its own joins
            const int c0 = cta_of(item_w0, W, grid), c1 = cta_of(item_w1 - 1, W, grid);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const uint32_t n = atomicAdd(&tickets[c0], 1u);
                is_last = n == static_cast<uint32_t>(c1 - c0);
                if (is_last) {
                    tickets[c0] = 0; // for the next launch
                }
            }
            __syncthreads();
            if (is_last) {
                __threadfence();
                join_pieces<T, DP, RT, NT>(a, part_o, part_ml, c0, c1, rq.first, kvh, group, rb * RT, rows, tid);
            }
        }
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    }
}

template <typename T, int DP, int WR, int WK>
void launch_attn(nb2_device* dev, const TreeAttnArgs& a) {
    using S = Shape<T, DP, WR, WK>;
    auto kernel = tree_attn_kernel<T, DP, WR, WK>;
    static int per_sm[64] = {};
    if (per_sm[dev->ordinal] == 0) {
        check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem),
                   "cudaFuncSetAttribute(tree attention)");
        int n = 0;
        check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, S::kThreads, S::kSmem),
                   "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
        per_sm[dev->ordinal] = std::max(1, n);
    }
    const int grid = dev->num_sms * per_sm[dev->ordinal];
    const size_t o_bytes = static_cast<size_t>(grid) * 2 * S::RT * DP * 4;
    uint8_t* ws = static_cast<uint8_t*>(dev->scratch(o_bytes + static_cast<size_t>(grid) * 2 * S::RT * 8));
    const int group = static_cast<int>(a.g.q_heads / a.g.kv_heads);
    float* part_o = reinterpret_cast<float*>(ws);
    float2* part_ml = reinterpret_cast<float2*>(ws + o_bytes);
    dim3 join;
    const bool apart = join_apart(a, grid, S::RT, DP, join);
    kernel<<<grid, S::kThreads, S::kSmem, dev->stream>>>(a, group, dev->num_sms, part_o, part_ml,
                                                         apart ? nullptr : dev->tickets(grid));
    check_cuda(cudaGetLastError(), "tree attention launch");
    if (apart) {
        join_kernel<T, DP, S::RT, S::KT, false>
            <<<join, kJoinThreads, 0, dev->stream>>>(a, group, grid, dev->num_sms, part_o, part_ml);
    }
    check_cuda(cudaGetLastError(), "tree attention join");
}

template <typename T, int DP>
void pick_rows(nb2_device* dev, const TreeAttnArgs& a) {
    const int64_t rows = std::min(a.g.max_new, a.g.tokens) * (a.g.q_heads / a.g.kv_heads);
    if (rows <= 16) {
        launch_attn<T, DP, 1, 4>(dev, a);
    } else if (rows <= 32 || DP * sizeof(T) > 512) { // 64 rows of 256 float32 in two parts do not fit
        launch_attn<T, DP, 2, 4>(dev, a);
    } else if constexpr (DP * sizeof(T) <= 512) {
        launch_attn<T, DP, 4, 2>(dev, a);
    }
}

template <typename T>
void pick_dim(nb2_device* dev, const TreeAttnArgs& a) {
    if (a.g.head_dim <= 64) {
        pick_rows<T, 64>(dev, a);
    } else if (a.g.head_dim <= 128) {
        pick_rows<T, 128>(dev, a);
    } else {
        pick_rows<T, 256>(dev, a);
    }
}

} // namespace

void tree_attention(nb2_device* dev, TreeAttnArgs a) {
    if (a.g.tokens == 0) {
        return;
    }
    a.err = dev->error_word();
    if (tree_attention_tc_takes(a, dev->num_sms)) {
        tree_attention_tc(dev, a);
    } else if (a.g.dtype == kF32) {
        pick_dim<float>(dev, a);
    } else if (a.g.dtype == kF16) {
        pick_dim<__half>(dev, a);
    } else {
        pick_dim<__nv_bfloat16>(dev, a);
    }
}

} // namespace nb2
