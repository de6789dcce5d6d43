// Tree attention for many rows a key/value head (wide trees, large groups), on
// the tcgen05 tensor cores: 16-bit types, head dimensions 64 to 128, pages of a
// power of two. The split of the work, the masks and the join are those of
// serving_attn.cu; with 33 rows and more that kernel is bound by its mma.sync and
// shared-memory rate.
//
// One CTA an SM: two softmax groups of four warps, a TMA warp, an MMA thread for each group. K and V
// tiles of 128 places come page by page as 4-D TMA boxes (64 elements x page) into 128-byte
// swizzled slabs, through rings of their own. Tensor memory holds two score tiles S (128 rows x 128
// places, fp32) and two accumulators O; group s owns S and O number s, one row a thread, so a row's
// maximum and sum need no exchange between threads. It takes S in halves of 64 places: reads a half, writes
// its weights P as packed 16-bit over the half's first 32 columns, and the MMA thread multiplies P from there with V (whose
// keys are the contraction: V is the MN-major operand as it lies in the cache) and puts the next tile's scores
// in the half's place, beside the softmax of the other half.
//   kTiles = 2: the groups are two blocks of 128 rows and share every tile of places.
//   kTiles = 1: up to 128 rows; the groups take alternate tiles of the same rows, and join at the end.
// O is rescaled in place, by its own group, only when a row's maximum has grown by more than 2^8 since its reference
// was set (the weights and sums stay far inside the range of their types; the final division takes the reference out).
//
// Measured, bfloat16, head dimension 128: 16 trees of 33-64 tokens, 32/8 heads, over 300-6,000 places (216 MB) 90 us, 2.4 TB/s
// and 470 TFLOP/s; 8 of 7-16 tokens, 40/8 heads, over 9,000-60,000 places (1.1 GB, float16) 235 us among other passes
// (4.7 TB/s; 207 us and 5.4 TB/s with an idle GPU before it), bound by HBM but for item ends. The first is bound by a tile's chain of copy, scores, softmax and products (4,450 clocks, where HBM alone takes 2,800) and
// by what a CTA does before its first tile (20,000 clocks) and after its last (16,000, with a join). Whole tiles
// of scores in place of halves 98 us; both slabs of a page as one 5-D box 2 us more on the first, 4 less on the second.
// ptxas spills 194-202 bytes a thread in each instance (what lives across the items, under the launch's 168 registers).
//
// Values that are not finite, and rows past the end of a page list, would reach rows that do not see them
// as 0 * inf: in the tiles that hold new tokens (or holes) the group clears such rows of V in shared
// memory before its P is released, and adds p * v itself for the rows that see the place.
//
// Every wait is bounded; a thread that gives up raises the CTA's abort flag, after which all loops run
// out without waiting: no product or copy is issued any more and no result is stored (the softmax threads
// still read and write their own tensor memory, which is held until the CTA ends).

#include "serving_attn.cuh"

#include <type_traits>

namespace nb2 {

namespace {

constexpr int kTcThreads = 384; // two softmax groups; a TMA warp, two MMA warps and one that only makes up the third group
constexpr int kSoftmax = 256; // threads of the two softmax groups
constexpr int kTile = 128;    // places of a tile, rows of a block
constexpr int kHalf = 64;     // places of a score product
constexpr uint32_t kColO = 256;
constexpr int kTcRows = 32; // rows a key/value head above which this kernel is taken

// ---- instructions -------------------------------------------------------------

// Shared-memory matrix descriptor, 128-byte swizzle (see sdesc_k128), with its leading byte offset: for an MN-major
// operand the distance of the next 64 elements of N.
__device__ __forceinline__ uint64_t sdesc_128(uint32_t saddr, uint32_t lbo) {
    return static_cast<uint64_t>((saddr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) | (64ull << 32) |
           (1ull << 46) | (2ull << 61);
}

// kind::f16, fp32 accumulator, M = 128: operand type, N, and whether B is MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, int n, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
           (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}

// D[tmem] += A[tmem] * B[smem]; A is 16-bit, two elements a column
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(1u)
                 : "memory");
}

// 32 lanes x 32 columns to registers, complete: the wait is part of the statement, so that nothing that uses them can
// come before it.
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
                 "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                   "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
                   "=r"(r[30]), "=r"(r[31])
                 : "r"(t));
}
// 32 lanes x 64 columns to registers, complete.
__device__ __forceinline__ void tmem_ld64(uint32_t t, uint32_t (&r)[64]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
                 "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,"
                 "%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,"
                 "%60,%61,%62,%63}, [%64];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                   "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                   "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                   "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(t)
                 : "memory");
}

__device__ __forceinline__ void tmem_ld1(uint32_t t, uint32_t& r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(t) : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t t, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
                 "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
                 "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
                 "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

__device__ __forceinline__ void tmem_st16u(uint32_t t, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
                     t),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// A page's 64 elements x box rows; coordinates element, head, place, block (out of range reads zeros). No multicast.
__device__ __forceinline__ void tma_load_page(void* dst, const CUtensorMap* map, int e, int head, int place, int block,
                                              uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(e), "r"(head), "r"(place), "r"(block)
                 : "memory");
}

// Registers of a warp group: the launch's 168 x 384 go as 208 to each softmax group (half a row's scores, 64, stay in
// registers) and 88 to the third.
template <int N>
__device__ __forceinline__ void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
static_assert((2 * 208 + 88) * 128 <= 168 * 384, "the groups share what the launch has");

__device__ __forceinline__ void bar_named(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
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

struct TcArgs {
    TreeAttnArgs a;
    int group;
    int box; // places of a TMA box: min(block_size, 128)
    float* part_o;
    float2* part_ml;
    uint32_t* tickets;
    long long bound;
};

template <int DP, int kTiles>
struct TcShape {
    static constexpr int RT = kTile * kTiles;
    static constexpr int kSlabs = DP / 64;
    static constexpr int kSlab = kTile * 128;         // bytes of 64 elements x 128 places
    static constexpr int kKV = kSlabs * kSlab;        // a K or a V tile
    static constexpr int kQ = kTiles * kKV;
    static constexpr int NS = DP == 64 ? 4 : kTiles == 2 ? 2 : 3;
    // Barriers of landed tiles, taken in turn. A wait by parity is right only where the barrier's phase before is known to be
    // over, and a group knows that of its own tiles: with alternate tiles a group and an odd ring, a stage's
    // tile before is the other group's, so that there are barriers for two rounds of the ring.
    static constexpr int NF = kTiles == 1 && NS % 2 == 1 ? 2 * NS : NS;
    static constexpr int kSmem = 1024 + kQ + 2 * NS * kKV;
};

template <typename T, int DP, int kTiles>
__global__ void __launch_bounds__(kTcThreads, 1)
    tree_attn_tc_kernel(const __grid_constant__ TcArgs args, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map) {
    using S = TcShape<DP, kTiles>;
    constexpr int NS = S::NS, NF = S::NF, RT = S::RT;
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
    const TreeAttnArgs& a = args.a;
    const nb2_tree_attn_geom& g = a.g;
    extern __shared__ uint8_t tc_dyn[];
    uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_dyn) + 1023) & ~uintptr_t(1023));
    uint8_t* ks = qs + S::kQ;
    uint8_t* vs = ks + NS * S::kKV;
    __shared__ uint64_t k_full[NF], k_empty[NS], v_full[NF], v_empty[NS], s_full[2][2], p_full[2][2], o_done[2][2], q_full,
        q_taken, drain;
    __shared__ int64_t red[kTcThreads / 32], found[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word, is_last, hole_word;
    // of a tile that is prepared (two of them: a thread can be one tile ahead): places that are there, by group, and
    // places whose values are not finite, by group (0 where both share the tile) and slab
    __shared__ uint32_t valid_of[2][2][4], odd[2][2][2][4];
    __shared__ float2 other_ml[kTile];
    volatile int* abort_flag = &abort_word;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = args.group;
    bool bad = false;
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(&k_empty[i], kTiles);
            mbar_init(&v_empty[i], kTiles);
        }
        for (int i = 0; i < NF; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&v_full[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            for (int h = 0; h < 2; ++h) {
                mbar_init(&s_full[i][h], 1);
                mbar_init(&p_full[i][h], kTile);
                mbar_init(&o_done[i][h], 1);
            }
        }
        mbar_init(&q_full, kSoftmax);
        mbar_init(&q_taken, 2);
        mbar_init(&drain, 2);
        abort_word = 0;
        hole_word = 0;
        fence_mbar_init();
    }
    if (warp == 9) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == 8 && lane == 0) {
        prefetch_tmap(&k_map);
        prefetch_tmap(&v_map);
    }
    const Span span = find_span<RT, kTile, kTcThreads>(a, group, 1, red, found, bad);
    spare_tokens<T>(a, tid, kTcThreads);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    // every role walks the same items
    auto items = [&](auto&& body) {
        int r = span.request;
        int64_t r_unit = span.request_unit;
        Request rq{};
        if (span.w0 < span.w1) {
            rq = request_at<RT, kTile>(a, r, group);
        }
        for (int64_t w = span.w0; w < span.w1;) {
            while (w >= r_unit + rq.units(g.kv_heads)) {
                r_unit += rq.units(g.kv_heads);
                rq = request_at<RT, kTile>(a, ++r, group);
            }
            const int64_t item = (w - r_unit) / rq.per_item();
            const int64_t item_w0 = r_unit + item * rq.per_item() + rq.extra; // its first tile
            const int64_t from = max(w, item_w0);
            w = min(span.w1, item_w0 + rq.tiles);
            if (from < w) {
                const int kvh = static_cast<int>(item / rq.row_blocks);
                const int rb = static_cast<int>(item - static_cast<int64_t>(kvh) * rq.row_blocks);
                body(r, rq, item_w0, kvh, rb, static_cast<int>(from - item_w0), static_cast<int>(w - item_w0));
            }
        }
    };

    if (warp >= 8) {
        regs_down<88>();
        if (warp == 8) {
            // ---- TMA: a lane a box
            uint32_t n = 0; // tiles so far
            const int size = static_cast<int>(g.block_size), boxes = kTile / args.box;
            items([&](int r, const Request& rq, int64_t, int kvh, int, int t0, int t1) {
                const int32_t* table = a.table + r * g.table_stride;
                for (int t = t0; t < t1; ++t, ++n) {
                    const int st = n % NS;
                    const uint32_t phase = (n / NS + 1) & 1;
                    // 128 places are at most 16 boxes of a slab; lane = box + 16 * slab
                    const int box = lane & 15, slab = lane >> 4;
                    const bool mine = box < boxes && slab < S::kSlabs;
                    const int j = t * kTile + box * args.box;
                    int block = -1; // out of range: zeros
                    if (mine && j < rq.total) {
                        block = table[j / size];
                        block = block < 0 || block >= g.num_blocks ? -1 : block;
                    }
                    bool ok = mbar_wait(&k_empty[st], phase, abort_flag, a.err, args.bound);
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok) {
                        if (lane == 0) {
                            mbar_arrive_expect_tx(&k_full[n % NF], S::kKV);
                        }
                        __syncwarp();
                        if (mine) {
                            tma_load_page(ks + st * S::kKV + slab * S::kSlab + box * args.box * 128, &k_map, slab * 64, kvh,
                                          j % size, block, &k_full[n % NF]);
                        }
                    }
                    ok = mbar_wait(&v_empty[st], phase, abort_flag, a.err, args.bound);
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok) {
                        if (lane == 0) {
                            mbar_arrive_expect_tx(&v_full[n % NF], S::kKV);
                        }
                        __syncwarp();
                        if (mine) {
                            tma_load_page(vs + st * S::kKV + slab * S::kSlab + box * args.box * 128, &v_map, slab * 64, kvh,
                                          j % size, block, &v_full[n % NF]);
                        }
                    }
                }
            });
            // copies in flight land before the CTA may go: their barriers complete on their own
            for (uint32_t i = n > NS ? n - NS : 0; i < n; ++i) {
                const long long c0 = clock64();
                while (!mbar_try_wait(&k_full[i % NF], (i / NF) & 1) && clock64() - c0 < kWaitBoundCycles && !*abort_flag) {
                }
                while (!mbar_try_wait(&v_full[i % NF], (i / NF) & 1) && clock64() - c0 < kWaitBoundCycles && !*abort_flag) {
                }
            }
            if (*abort_flag) { // some barriers will not complete: give the copies the time they take
                const long long c0 = clock64();
                while (clock64() - c0 < 2000000) {
                }
            }
        } else if (warp < 11 && lane == 0) {
            // ---- MMA: a thread a group. An MMA holds its issuing thread about as long as it runs, so one thread for both
            // groups left the tensor cores idle while it looked for the next work (700 clocks to issue eight, 250 to 600
            // between).
            const int s = warp - 9;
            uint32_t n = 0, items_done = 0, uses = 0; // tiles of all items so far, items, this group's tiles
            const uint32_t idesc_s = idesc_f16(kBf16, kHalf, false), idesc_o = idesc_f16(kBf16, DP, true);
            const uint32_t q = smem_u32(qs + (kTiles == 2 ? s * S::kKV : 0)), t_s = tmem + s * kTile,
                           t_o = tmem + kColO + s * kTile;
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                const bool ok = mbar_wait(bar, parity, abort_flag, a.err, args.bound);
                tc_fence_after();
                return ok;
            };
            items([&](int, const Request&, int64_t, int, int, int t0, int t1) {
                bool ok = wait(&q_full, items_done & 1);
                ++items_done;
                mbar_arrive(&q_taken);
                constexpr int kStep = kTiles == 2 ? 1 : 2;
                const int i0 = kTiles == 2 ? 0 : s, nt = t1 - t0;
                // S = Q K^T of half h of a tile; the last half's commit gives K back
                auto scores = [&](int i, int h) {
                    const uint32_t st = (n + i) % NS;
                    ok = ok && wait(&k_full[(n + i) % NF], ((n + i) / NF) & 1);
                    if (ok) {
                        const uint32_t k = smem_u32(ks + st * S::kKV) + h * kHalf * 128;
#pragma unroll
                        for (int c = 0; c < DP / 16; ++c) {
                            const uint32_t at = (c / 4) * S::kSlab + (c % 4) * 32;
                            mma_f16(t_s + h * kHalf, sdesc_128(q + at, 16), sdesc_128(k + at, 16), idesc_s, c > 0);
                        }
                        mma_commit(&s_full[s][h]);
                        if (h == 1) {
                            mma_commit(&k_empty[st]);
                        }
                    }
                };
                if (i0 < nt) {
                    scores(i0, 0);
                    scores(i0, 1);
                }
                for (int i = i0; i < nt; i += kStep, ++uses) {
                    const uint32_t st = (n + i) % NS;
                    ok = ok && wait(&v_full[(n + i) % NF], ((n + i) / NF) & 1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // O += P V of the half, then the half's next scores where its weights were
                        ok = ok && wait(&p_full[s][h], uses & 1);
                        if (ok) {
                            const uint32_t v = smem_u32(vs + st * S::kKV) + h * kHalf * 128;
#pragma unroll
                            for (int c = 0; c < kHalf / 16; ++c) {
                                mma_f16_ta(t_o, t_s + h * kHalf + c * 8, sdesc_128(v + c * 2048, S::kSlab), idesc_o);
                            }
                            mma_commit(&o_done[s][h]);
                            if (h == 1) {
                                mma_commit(&v_empty[st]);
                            }
                        }
                        if (i + kStep < nt) {
                            ok = ok && wait(&o_done[s][h], uses & 1);
                            scores(i + kStep, h);
                        }
                    }
                }
                n += t1 - t0;
            });
            // what was issued completes before tensor memory is freed
            mma_commit(&drain);
            const long long c0 = clock64();
            while (!mbar_try_wait(&drain, 0) && clock64() - c0 < kWaitBoundCycles) {
            }
        }
        __syncwarp();
    } else {
        regs_up<208>();
        // ---- softmax: group s, one row a thread
        const int s = warp >> 2, wt = tid & 127;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + lanes + s * kTile, t_o = tmem + lanes + kColO + s * kTile;
        const float scale2 = fmaxf(fabsf(g.scale) * kLog2e, 1e-30f); // not 0: -inf * 0 is no weight
        const bool flip = g.scale < 0.0f; // Q is negated instead, so that a row's largest product is its maximum
        const int size = static_cast<int>(g.block_size);
        const int share = kTiles == 2 ? kSoftmax : kTile; // threads that prepare a tile together
        uint32_t s_uses = 0, n = 0, items_begun = 0;
        uint32_t zeros[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            zeros[i] = 0;
        }
        items([&](int r, const Request& rq, int64_t item_w0, int kvh, int rb, int t0, int t1) {
            const int rows = min(RT, rq.n * group - rb * RT);
            const int old = rq.total - rq.n;
            const int32_t* table = a.table + r * g.table_stride;
            const int row = (kTiles == 2 ? s * kTile : 0) + wt;
            const int tok = row < rows ? (rb * RT + row) / group : -1;
            const uint32_t* mask = a.mask != nullptr ? a.mask + (rq.first + max(tok, 0)) * g.mask_words : nullptr;
            // What runs once an item is kept small (rolled loops): unrolled, its instructions came from L2 each time and an item
            // cost as much as nine tiles.
            // the 16-byte chunks of the item's rows, in q and in out, shared by the 256 threads
            constexpr int kRowChunks = DP / 8, kRowStep = kSoftmax / kRowChunks, kRowSteps = RT / kRowStep;
            auto for_rows = [&](auto&& f) {
                const int ch = tid % kRowChunks;
                int qr = tid / kRowChunks;
                int qt = (rb * RT + qr) / group, hq = rb * RT + qr - qt * group;
                const int dt = kRowStep / group, dh = kRowStep - dt * group;
#pragma unroll 4
                for (int u = 0; u < kRowSteps; ++u) {
                    const int64_t t = rq.first + qt, h = static_cast<int64_t>(kvh) * group + hq;
                    f(qr, ch, static_cast<const T*>(a.q) + t * g.q_stride + h * g.q_head_stride + ch * 8,
                      static_cast<T*>(a.out) + t * g.o_stride + h * g.o_head_stride + ch * 8);
                    qr += kRowStep;
                    qt += dt;
                    hq += dh;
                    if (hq >= group) {
                        hq -= group;
                        ++qt;
                    }
                }
            };
            // ---- Q into shared memory (K-major slabs of 64), zero past the rows and head_dim
            for_rows([&](int qr, int ch, const T* src, T*) {
                const bool in = qr < rows && ch * 8 < g.head_dim;
                const int lr = qr % kTile, to = (qr / kTile) * S::kKV + (ch / 8) * S::kSlab + lr * 128 +
                                                (((ch & 7) ^ (lr & 7)) << 4);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(qs + to)),
                             "l"(in ? src : static_cast<const T*>(a.q)), "r"(in ? 16 : 0)
                             : "memory");
            });
            asm volatile("cp.async.commit_group;" ::: "memory");
            // places of this CTA's tiles without a block: then every tile looks its places up
            bool hole = false;
            for (int j = t0 * kTile / size + tid; j * static_cast<int64_t>(size) < min(rq.total, t1 * kTile); j += kSoftmax) {
                hole |= table[j] < 0 || table[j] >= g.num_blocks;
            }
            if (hole) {
                hole_word = 1;
                bad = true;
            }
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                tmem_st32(t_o + c, zeros);
            }
            tmem_wait_st();
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (flip) { // a thread's own chunks
                for_rows([&](int qr, int ch, const T*, T*) {
                    const int lr = qr % kTile;
                    uint4* x = reinterpret_cast<uint4*>(qs + (qr / kTile) * S::kKV + (ch / 8) * S::kSlab + lr * 128 +
                                                        (((ch & 7) ^ (lr & 7)) << 4));
                    *x = make_uint4(x->x ^ 0x80008000u, x->y ^ 0x80008000u, x->z ^ 0x80008000u, x->w ^ 0x80008000u);
                });
            }
            fence_proxy_async_smem();
            // Not before both MMA threads have seen the item before: one that has no tile of it is awaited by nothing else, and
            // two items behind it would take this one's phase for one that is still to come.
            bool ok = items_begun == 0 || mbar_wait(&q_taken, (items_begun - 1) & 1, abort_flag, a.err, args.bound);
            ++items_begun;
            mbar_arrive(&q_full);
            bar_named(1, kSoftmax);
            const bool holes = *const_cast<volatile int*>(&hole_word) != 0;

            float m = -INFINITY, z = 0.0f; // reference and sum of this row
            ok = ok && !*abort_flag;
            uint32_t halves = 0; // of this item, whose weights this thread has given
            // After the product of the last weights that this thread has given. (A barrier for each half: the phase before the one
            // awaited is then always over, its half's next scores having been made after it.)
            auto rest = [&] {
                if (halves > 0) {
                    const uint32_t h = (halves - 1) & 1;
                    ok = mbar_wait(&o_done[s][h], (s_uses - (h == 1 ? 1 : 0)) & 1, abort_flag, a.err, args.bound) && ok;
                    __syncwarp();
                    tc_fence_after();
                }
            };
            // The reference for scores whose largest is `raw`: O and the sum move to a new one where it is too far below,
            // after the last product.
            auto refer = [&](float raw) {
                const float now = raw == -INFINITY ? -INFINITY : raw * scale2;
                if (!__any_sync(0xffffffffu, now > m + 8.0f)) {
                    return;
                }
                rest();
                const float to = fmaxf(m, now), keep = to == -INFINITY ? 1.0f : exp2_fast(m - to);
                if (__any_sync(0xffffffffu, m > -INFINITY)) {
#pragma unroll 1
                    for (int c = 0; c < DP; c += 16) {
                        float v[16];
                        tmem_ld16(t_o + c, v);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            v[i] *= keep;
                        }
                        tmem_st16(t_o + c, v);
                    }
                    tmem_wait_st();
                }
                z *= keep;
                m = to;
            };
            auto at_rest = [&] { return m == -INFINITY ? 0.0f : m; };
            for (int t = t0 + (kTiles == 2 ? 0 : s); t < t1; t += kTiles == 2 ? 1 : 2) {
                const uint32_t tile = n + (t - t0);
                const int j0 = t * kTile;
                const bool plain = j0 + kTile <= old && !holes;
                // bits of the tile's places that this row's token sees, if they are there
                uint32_t sees[4] = {0, 0, 0, 0};
                auto seen = [&](int w) { // of places 32 w .. 32 w + 31
                    return (w == 0 ? sees[0] : w == 1 ? sees[1] : w == 2 ? sees[2] : sees[3]) & valid_of[s_uses & 1][s][w];
                };
                const int mine = kTiles == 2 ? 0 : s; // whose odd[] the tile uses
                if (!plain) {
                    // ---- V's rows that may not be multiplied: no such place, or not finite
                    uint8_t* vt = vs + (tile % NS) * S::kKV;
                    const int j = j0 + wt; // the place of this thread
                    bool there = j < rq.total;
                    if (there && holes) {
                        const int b = table[j / size];
                        there = b >= 0 && b < g.num_blocks;
                    }
                    const uint32_t valid = __ballot_sync(0xffffffffu, there);
                    if (tok >= 0) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            sees[w] = see_bits(mask, g.mask_words, tok, j0 + 32 * w - old);
                        }
                    }
                    ok = mbar_wait(&v_full[tile % NF], (tile / NF) & 1, abort_flag, a.err, args.bound) && ok;
#pragma unroll 1
                    for (int sl = 0; sl < S::kSlabs; ++sl) {
                        if (kTiles == 2 && S::kSlabs == 2 && sl != s) {
                            continue; // the groups share the slabs
                        }
                        if (kTiles == 2 && S::kSlabs == 1 && s != 0) {
                            continue;
                        }
                        uint8_t* vr = vt + sl * S::kSlab + wt * 128;
                        bool odd_here = false;
#pragma unroll 2
                        for (int c = 0; c < 8; ++c) {
                            const uint4 x = *reinterpret_cast<const uint4*>(vr + ((c ^ (wt & 7)) << 4)); // no bank twice
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t u = e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w;
                                constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
                                odd_here |= (u & kExp) == kExp || ((u >> 16) & kExp) == kExp;
                            }
                        }
                        if (!there || odd_here) {
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                *reinterpret_cast<uint4*>(vr + ((c ^ (wt & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        const uint32_t o = __ballot_sync(0xffffffffu, there && odd_here);
                        if (lane == 0) {
                            odd[s_uses & 1][mine][sl][warp & 3] = o;
                        }
                    }
                    fence_proxy_async_smem();
                    if (lane == 0) {
                        valid_of[s_uses & 1][s][warp & 3] = valid;
                    }
                    bar_named(kTiles == 2 ? 1 : 2 + s, share);
                }
#pragma unroll 1
                for (int h = 0; h < 2; ++h, ++halves) {
                    // ---- the row's scores of a half
                    const uint32_t t_h = t_s + h * kHalf;
                    ok = mbar_wait(&s_full[s][h], s_uses & 1, abort_flag, a.err, args.bound) && ok;
                    __syncwarp();
                    tc_fence_after();
                    float zz[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    // 32 scores to weights, packed over the scores. They are rounded to the cache's type, as both operands of
                    // the product must have it: each at most u off, which the sum over places averages (the error against
                    // 64 bits is 1.1 to 1.4 times that of unrounded weights; a second product of their rest would double
                    // the tensor cores' work). The sum z keeps all their bits.
                    auto weights = [&](int c, const float* x, float ref) {
                        uint32_t pk[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float p0 = exp2_fast(fmaf(x[2 * i], scale2, -ref));
                            const float p1 = exp2_fast(fmaf(x[2 * i + 1], scale2, -ref));
                            zz[(2 * i) & 3] += p0;
                            zz[(2 * i + 1) & 3] += p1;
                            pk[i] = pack2<T>(p0, p1);
                        }
                        tmem_st16u(t_h + c * 16, pk);
                    };
                    if (plain) { // the row stays in registers
                        float x[kHalf];
                        uint32_t v[kHalf];
                        tmem_ld64(t_h, v);
#pragma unroll
                        for (int i = 0; i < kHalf; ++i) {
                            x[i] = __uint_as_float(v[i]);
                        }
                        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                        for (int i = 4; i < kHalf; ++i) {
                            top[i & 3] = fmaxf(top[i & 3], x[i]);
                        }
                        refer(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                        const float ref = at_rest();
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            weights(c, x + c * 32, ref);
                        }
                    } else {
                        auto chunk = [&](int c, float (&x)[32]) {
                            const uint32_t see = seen(2 * h + c);
                            uint32_t v[32];
                            tmem_ld32(t_h + c * 32, v);
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                x[i] = (see >> i) & 1u ? __uint_as_float(v[i]) : -INFINITY;
                            }
                        };
                        float top = -INFINITY;
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            float x[32];
                            chunk(c, x);
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                top = fmaxf(top, x[i]);
                            }
                        }
                        refer(top);
                        // ---- places whose values are not finite, for the rows that see them
#pragma unroll 1
                        for (int sw = 0; sw < S::kSlabs * 2; ++sw) {
                            const int sl = sw >> 1, w = 2 * h + (sw & 1);
                            for (uint32_t left = odd[s_uses & 1][mine][sl][w]; left != 0; left &= left - 1) {
                                rest(); // O is changed
                                const int key = w * 32 + __ffs(left) - 1, j = j0 + key;
                                uint32_t raw_s;
                                tmem_ld1(t_s + key, raw_s);
                                const float p = (seen(w) >> (key & 31)) & 1u
                                                    ? exp2_fast(fmaf(__uint_as_float(raw_s), scale2, -at_rest()))
                                                    : 0.0f;
                                const int64_t b = table[j / size];
                                const T* v = static_cast<const T*>(a.vc) + b * g.vc_block_stride +
                                             (j % size) * g.vc_place_stride + kvh * g.vc_head_stride + sl * 64;
#pragma unroll 1
                                for (int c = 0; c < 64; c += 16) {
                                    float o[16];
                                    tmem_ld16(t_o + sl * 64 + c, o);
#pragma unroll
                                    for (int i = 0; i < 16; ++i) {
                                        const bool in = p > 0.0f && sl * 64 + c + i < g.head_dim;
                                        o[i] += in ? p * to_f32(v[in ? c + i : 0]) : 0.0f;
                                    }
                                    tmem_st16(t_o + sl * 64 + c, o);
                                    tmem_wait_st();
                                }
                            }
                        }
                        const float ref = at_rest();
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            float x[32];
                            chunk(c, x);
                            weights(c, x, ref);
                        }
                    }
                    z += (zz[0] + zz[1]) + (zz[2] + zz[3]);
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&p_full[s][h]);
                }
                ++s_uses;
            }
            // ---- the item's end: O at rest, joined where the groups share rows, stored
            const int my_tiles = kTiles == 2 ? t1 - t0 : (t1 - t0 + 1 - s) / 2;
            if (my_tiles > 0) {
                for (int h = 0; h < 2; ++h) {
                    ok = mbar_wait(&o_done[s][h], (s_uses - 1) & 1, abort_flag, a.err, args.bound) && ok;
                }
            }
            __syncwarp();
            tc_fence_after();
            const bool whole = t0 == 0 && t1 == rq.tiles;
            const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0);
            float mm = m, ff = 1.0f, f_other = 0.0f, zs = z;
            if (kTiles == 1) {
                // both groups hold all rows' sums over half of the tiles: each joins half of the elements
                if (s == 1) {
                    other_ml[wt] = make_float2(m, z);
                }
                tc_fence_before();
                bar_named(1, kSoftmax);
                tc_fence_after();
                const float2 o1 = other_ml[wt];
                bar_named(1, kSoftmax);
                if (s == 0) {
                    other_ml[wt] = make_float2(m, z);
                }
                bar_named(1, kSoftmax);
                const float2 o2 = other_ml[wt];
                const float2 ot = s == 0 ? o1 : o2;
                mm = fmaxf(m, ot.x);
                const float ref = mm == -INFINITY ? 0.0f : mm;
                ff = exp2_fast(m - ref);
                f_other = exp2_fast(ot.x - ref);
                // the same order in both groups
                zs = s == 0 ? ff * z + f_other * ot.y : f_other * ot.y + ff * z;
            }
            const bool clean = ok && !*abort_flag, live = row < rows && clean;
            constexpr int kCols = kTiles == 2 ? DP : DP / 2;
            const int c0 = kTiles == 2 ? 0 : s * kCols;
            // finished values of a row's 32 elements from d on, through Q's shared memory (its products are
            // done) so that the stores to out are of whole rows: a row a thread, each store met 32 lines
            auto stage = [&](int d, const float* x, float sum) {
                const float inv = 1.0f / sum;
                const bool none = sum == 0.0f; // no place was seen
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = none ? 0u : pack2<T>(x[i + 2 * e] * inv, x[i + 2 * e + 1] * inv);
                    }
                    *reinterpret_cast<uint4*>(qs + row * DP * 2 + ((((d + i) >> 3) ^ (row & 7)) << 4)) =
                        make_uint4(y[0], y[1], y[2], y[3]);
                }
            };
            auto finish = [&](float top, float sum) { // after stage() of all elements
                bar_named(1, kSoftmax);
                if (clean) {
                    for_rows([&](int qr, int ch, const T*, T* dst) {
                        if (qr < rows && ch * 8 < g.head_dim) {
                            *reinterpret_cast<uint4*>(dst) =
                                *reinterpret_cast<const uint4*>(qs + qr * DP * 2 + ((ch ^ (qr & 7)) << 4));
                        }
                    });
                    if (row < rows && (kTiles == 2 || s == 0) && a.lse != nullptr) {
                        const int64_t h = static_cast<int64_t>(kvh) * group + (rb * RT + row - tok * group);
                        a.lse[(rq.first + tok) * g.q_heads + h] = sum == 0.0f ? -INFINITY : top * kLn2 + logf(sum);
                    }
                }
            };
            // a piece lies in its slot four elements by four, the rows together
            float4* piece = reinterpret_cast<float4*>(args.part_o) + slot * (DP / 4) * RT + row;
#pragma unroll 1
            for (int c = 0; c < kCols; c += 32) {
                uint32_t v[32];
                float x[32];
                __syncwarp();
                tmem_ld32(t_o + c0 + c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    x[i] = __uint_as_float(v[i]);
                }
                if (kTiles == 1) {
                    tmem_ld32(tmem + lanes + kColO + (1 - s) * kTile + c0 + c, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float p = ff != 0.0f ? ff * x[i] : 0.0f;
                        const float q = f_other != 0.0f ? f_other * __uint_as_float(v[i]) : 0.0f;
                        x[i] = p + q;
                    }
                }
                if (whole) {
                    stage(c0 + c, x, zs);
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        __stcg(piece + (c0 + c + i) / 4 * RT, make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]));
                    }
                }
            }
            if (whole) {
                finish(mm, zs);
            } else {
                if (live && (kTiles == 2 || s == 0)) {
                    __stcg(args.part_ml + slot * RT + row, make_float2(mm, zs));
                }
            }
            if (!whole && args.tickets != nullptr) { // null: a launch of its own joins
                const int p0 = cta_of(item_w0, span.W, span.grid), p1 = cta_of(item_w0 + rq.tiles - 1, span.W, span.grid);
                __threadfence();
                bar_named(1, kSoftmax);
                if (tid == 0) {
                    const uint32_t k = atomicAdd(&args.tickets[p0], 1u);
                    is_last = k == static_cast<uint32_t>(p1 - p0);
                    if (is_last) {
                        args.tickets[p0] = 0; // for the next launch
                    }
                }
                bar_named(1, kSoftmax);
                if (*const_cast<volatile int*>(&is_last)) {
                    // all pieces are there: added in the order of their CTAs
                    __threadfence();
                    float top = -INFINITY, sum = 0.0f;
                    constexpr int kJoin = kCols < 64 ? kCols : 64; // elements of a row at a time
#pragma unroll 1
                    for (int c = 0; c < kCols; c += kJoin) {
                        float x[kJoin];
#pragma unroll
                        for (int i = 0; i < kJoin; ++i) {
                            x[i] = 0.0f;
                        }
                        top = -INFINITY;
                        sum = 0.0f;
#pragma unroll 1
                        for (int p = p0; p <= p1; ++p) {
                            const int64_t at = 2 * static_cast<int64_t>(p) + (p == p0 ? 1 : 0);
                            const float4* src = reinterpret_cast<const float4*>(args.part_o) + (at * DP + c0 + c) / 4 * RT + row;
                            const float2 ml = live ? __ldcg(args.part_ml + at * RT + row) : make_float2(-INFINITY, 0.0f);
                            float4 y[kJoin / 4];
#pragma unroll
                            for (int i = 0; i < kJoin / 4; ++i) {
                                y[i] = live ? __ldcg(src + i * RT) : make_float4(0, 0, 0, 0);
                            }
                            const float to = fmaxf(top, ml.x), ref = to == -INFINITY ? 0.0f : to;
                            const float f = exp2_fast(top - ref), h = exp2_fast(ml.x - ref);
                            top = to;
                            sum = f * sum + h * ml.y;
#pragma unroll
                            for (int i = 0; i < kJoin / 4; ++i) {
                                const float* z4 = &y[i].x;
#pragma unroll
                                for (int k = 0; k < 4; ++k) { // a piece that saw nothing adds nothing
                                    x[4 * i + k] = h != 0.0f ? f * x[4 * i + k] + h * z4[k] : f * x[4 * i + k];
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < kJoin; i += 32) {
                            stage(c0 + c + i, x + i, sum);
                        }
                    }
                    finish(top, sum);
                }
            }
            tc_fence_before();
            bar_named(1, kSoftmax); // shared words and Q are free for the next item
            if (tid == 0) {
                hole_word = 0;
            }
            bar_named(1, kSoftmax);
            n += t1 - t0;
        });
    }
    if (bad) {
        record_error(a.err, kDevIndexOutOfRange);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

CUtensorMap page_map(const void* base, const nb2_tree_attn_geom& g, bool bf16, int64_t block_stride, int64_t place_stride,
                     int64_t head_stride, int box) {
    CUtensorMap m{};
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(g.head_dim), static_cast<cuuint64_t>(g.kv_heads),
                                static_cast<cuuint64_t>(g.block_size), static_cast<cuuint64_t>(g.num_blocks)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(head_stride * 2), static_cast<cuuint64_t>(place_stride * 2),
                                   static_cast<cuuint64_t>(block_stride * 2)};
    const cuuint32_t boxes[4] = {64, 1, static_cast<cuuint32_t>(box), 1}, ones[4] = {1, 1, 1, 1};
    const CUresult e = encode_tiled()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                                      const_cast<void*>(base), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) {
        fail(kStatusCuda, "tree attention: cuTensorMapEncodeTiled failed (" + std::to_string(static_cast<int>(e)) + ")");
    }
    return m;
}

template <typename T, int DP, int kTiles>
void launch_tc(nb2_device* dev, const TreeAttnArgs& a) {
    using S = TcShape<DP, kTiles>;
    auto kernel = tree_attn_tc_kernel<T, DP, kTiles>;
    static bool set[64] = {};
    if (!set[dev->ordinal]) {
        check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem),
                   "cudaFuncSetAttribute(tree attention)");
        set[dev->ordinal] = true;
    }
    const nb2_tree_attn_geom& g = a.g;
    constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
    const int box = static_cast<int>(std::min<int64_t>(g.block_size, kTile));
    const CUtensorMap km = page_map(a.kc, g, bf16, g.kc_block_stride, g.kc_place_stride, g.kc_head_stride, box);
    const CUtensorMap vm = page_map(a.vc, g, bf16, g.vc_block_stride, g.vc_place_stride, g.vc_head_stride, box);
    const int grid = dev->num_sms;
    const size_t o_bytes = static_cast<size_t>(grid) * 2 * S::RT * DP * 4;
    uint8_t* ws = static_cast<uint8_t*>(dev->scratch(o_bytes + static_cast<size_t>(grid) * 2 * S::RT * 8));
    const int group = static_cast<int>(g.q_heads / g.kv_heads);
    float* part_o = reinterpret_cast<float*>(ws);
    float2* part_ml = reinterpret_cast<float2*>(ws + o_bytes);
    dim3 join;
    const bool apart = join_apart(a, grid, S::RT, DP, join);
    const TcArgs args{a, group, box, part_o, part_ml, apart ? nullptr : dev->tickets(grid), dev->wait_bound};
    kernel<<<grid, kTcThreads, S::kSmem, dev->stream>>>(args, km, vm);
    check_cuda(cudaGetLastError(), "tree attention launch");
    if (apart) {
        join_kernel<T, DP, S::RT, kTile, true><<<join, kJoinThreads, 0, dev->stream>>>(a, group, grid, 1, part_o, part_ml);
    }
    check_cuda(cudaGetLastError(), "tree attention join");
}

template <typename T, int DP>
void pick_tiles(nb2_device* dev, const TreeAttnArgs& a) {
    const int64_t rows = std::min(a.g.max_new, a.g.tokens) * (a.g.q_heads / a.g.kv_heads);
    rows > kTile ? launch_tc<T, DP, 2>(dev, a) : launch_tc<T, DP, 1>(dev, a);
}

} // namespace

bool tree_attention_tc_takes(const TreeAttnArgs& a, int sms) {
    const nb2_tree_attn_geom& g = a.g;
    const int64_t rows = std::min(g.max_new, g.tokens) * (g.q_heads / g.kv_heads);
    const bool page = g.block_size >= 8 && (g.block_size & (g.block_size - 1)) == 0;
    const int64_t most = int64_t{1} << 39; // a map's stride, in elements here
    bool strides = true;
    for (int64_t s : {g.kc_block_stride, g.kc_place_stride, g.kc_head_stride, g.vc_block_stride, g.vc_place_stride,
                      g.vc_head_stride}) {
        strides = strides && s > 0 && s < most;
    }
    // Up to 64 rows with less than a tile a CTA: an item's beginning and end cost more than its products (48 rows, 2 key/value
    // heads: 2 requests over 3,400 places 34 us here and 26 there, 7 over 3,000 places 31 and 39; 8 heads 45 and 59).
    const int64_t tiles = g.batch * g.kv_heads * ((g.table_blocks * g.block_size + kTile - 1) / kTile);
    const bool enough = rows > 64 || (rows > kTcRows && tiles > sms);
    return g.dtype != kF32 && enough && g.head_dim >= 64 && g.head_dim <= 128 && page && strides && g.num_blocks > 0;
}

void tree_attention_tc(nb2_device* dev, const TreeAttnArgs& a) {
    if (a.g.dtype == kF16) {
        a.g.head_dim <= 64 ? pick_tiles<__half, 64>(dev, a) : pick_tiles<__half, 128>(dev, a);
    } else {
        a.g.head_dim <= 64 ? pick_tiles<__nv_bfloat16, 64>(dev, a) : pick_tiles<__nv_bfloat16, 128>(dev, a);
    }
}

} // namespace nb2
