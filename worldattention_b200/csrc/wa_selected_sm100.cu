// Gradient of attention over selected key blocks on the tensor cores of sm_100a: bf16, head_dim 128, blocks of 64 or 128 tokens.
//
// Two launches of one kernel.  Each owns a block of one side at a time -- the first of keys, for dK and dV, the second of queries, for dQ -- and
// meets the blocks of the other side that are listed with it.  For blocks of 64 tokens (128: further down) a step meets two blocks,
// which need not be neighbours (nor, with shared keys, of one query head).  With F1, F2 the owned rows and G1, G2 the met ones (keys: F = k, v and G = q, dout; queries: F = q, dout and G = k, v)
//     S = G1 F1^T   dP = G2 F2^T                      [128 met rows x 64 owned ones]
//     P = 2^(S c - lse)   dS = P (dP - delta)         (lse and delta of the query row: 128 of a step's, or 64 of an item's)
//     dV^T += G2^T P   dK^T (or dQ^T) += G1^T dS      [128 channels x 64 owned rows]
// so all four products have 128 rows and 64 columns, the met tile is the first operand of all of them as it lies (row-major for the
// scores, transposed for the sums), and P and dS, which a thread holds by rows, are second operands that go to shared memory the
// way they are.  The met rows' lists: bits per key block, or the clean ids of a query block.  Every sum is made in one CTA in
// the order of its list: no atomics, equal calls give equal bits; the price is that S and dP are computed in both launches.
//
// One persistent CTA of twenty warps per SM: sixteen turn scores into P and dS and sums into bf16, one walks the lists and issues the loads, one
// issues the scores' products, one the sums' and one stores finished sums.  Tensor memory holds two steps' scores and the sums of two owned
// tiles (2 x 128 + 2 x 128 columns).
//
// What bounds it: the tensor pipe, and how long a step takes from load to sum.  A product of 128 x 64 x 16 keeps the pipe for 48 cycles (32 would do, but both
// operands come from shared memory), a step's for 1536 (dQ: 1152) of the 2080 (1600) that it lasts: 72 % of the time.  Two steps are in flight, and each is
// a chain of a tile's arrival (1100), the scores (770), P and dS (1100) and the sums.
// 32 760 tokens over themselves, 32 of 512 blocks a row, 12 heads: dK/dV 805 us, dQ 610.  One issuing warp for both took 1323 and 986, eight workers 998
// and 819, five slots in turn and sums stored by the workers 920 and 708.  Tried since: a second loading warp 809 and 628, owned tiles loaded one by one 815
// and 643, the next item's list read ahead 843 and 602.
// Roundings: P and dS to bf16 as factors of products, as their other factors are; sums in float32; gradients once at the end.
//
// Every wait is bounded (about two seconds); on expiry a flag is raised, all roles leave, tensor memory is freed and the kernel returns.
#include "wa_selected.cuh"
#include "wa_sm100_ptx.cuh"

namespace wa {
namespace sm100 {

constexpr int SB_OWN = 64;                              // owned rows of an item
constexpr int SB_OWN_BYTES = SB_OWN * TILE * 2;         // 16 KB: [half of the channels][row][64 channels]
constexpr int SB_P_BYTES = TILE * SB_OWN * 2;           // 16 KB: [met row][64 owned rows]
constexpr int SB_DESCS = 4;
constexpr int SB_BARRIER_BYTES = 3 * 1024;
constexpr int SB_WORKERS = 16;                          // warps that make P and dS
constexpr int SB_THREADS = (SB_WORKERS + 4) * 32;

template <bool KEYS> struct SbRing {
    // met tiles (32 KB each): G1 and G2 of a step take one each, of slots of their own.  G2 goes first (dQ: with the scores; keys: its sum is issued first),
    // and two are enough to load the next while this one is read; three of G1's then keep the loads off the way from one step's sums to the next
    // but one's scores (five slots in turn, window: dQ 693 us)
    static constexpr int SLOTS1 = 3, SLOTS2 = 2, SLOTS = SLOTS1 + SLOTS2;
    static __device__ __forceinline__ uint32_t slot(int g, uint32_t step) { return g == 0 ? step % SLOTS1 : SLOTS1 + step % SLOTS2; }
    static __device__ __forceinline__ uint32_t parity(int g, uint32_t step) { return (g == 0 ? step / SLOTS1 : step / SLOTS2) & 1u; }
    static constexpr int FACTORS = 2;                   // P and dS of one step, or dS of two
    static constexpr int SMEM = 2 * SB_OWN_BYTES + SLOTS * TILE_BYTES + FACTORS * SB_P_BYTES + SB_BARRIER_BYTES;
};

enum { SB_FIRST = 1, SB_LAST = 2, SB_EMPTY = 4, SB_END = 8 };
struct SbDesc {
    int item, flags;
    int of[2];           // of the met rows 0..63 and 64..127: queries' launch: how many are tokens; keys': their place among the rows of `stats`
};

struct SbBarriers {
    // queries: 64 (-normaliser) and 64 (-delta) of the owned rows, [four items] -- when an item's are loaded, the warps may still be three items behind, but not
    // four: the scores of the item before needed a slot that the sums of that one gave back
    float stats[4 * TILE];
    uint64_t desc_full[SB_DESCS], desc_empty[SB_DESCS];
    uint64_t f_full, f_empty, stats_full[4];
    uint64_t full[5], empty[5];
    uint64_t s_full[2], s_free[2], p_full[2], p_free[2];
    uint64_t acc_full[2], acc_empty[2];
    uint64_t staged[4];                // of four items: one may be staged while the one three before it is being stored, whose slot the next would need
    uint64_t stored[2];                // queries: of each group
    uint32_t tmem_base;
    int abort_flag;
    SbDesc desc[SB_DESCS];
};
static_assert(sizeof(SbBarriers) <= SB_BARRIER_BYTES, "barrier block exceeds its shared-memory budget");
static_assert(SbRing<true>::SMEM <= 227 * 1024 && SbRing<false>::SMEM <= 227 * 1024, "shared memory budget exceeded");

struct SbParams {
    int H, Hkv, group, Lq, Lkv, Nq, Nkv;
    int owned, items;                 // owned tiles of a head; of all heads
    int list_stride, row_words;
    long long padded;                 // rows of `stats` of a head
    const int32_t *index, *num;       // queries
    const int32_t *q_order, *k_order; // blocks of the owned side, heaviest first, or null: as they come
    const uint32_t *rows;             // keys
    const float *stats;
    __nv_bfloat16 *d1, *d2;           // dV; dK or dQ
    long long d1b, d1l, d1h, d2b, d2l, d2h;
    float scale, scale_log2;
    int *work_counter, *error_flag, *status_mirror;
};

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}

// What an owned tile meets, one id at a time, by a whole warp: 32 words of bits or 32 ids in its lanes' registers.
template <bool KEYS>
struct SbList {
    const uint32_t *bits;
    const int32_t *ids;
    int n, at, words_per_head;
    uint32_t mine;
    unsigned left;
    __device__ void begin(const SbParams &p, long long list, int lane) {
        at = 0;
        if (KEYS) {
            words_per_head = p.row_words;
            n = p.group * p.row_words;
            bits = p.rows + list * n;
        } else {
            n = p.num[list];
            ids = p.index + list * p.list_stride;
        }
        fetch(lane);
    }
    __device__ void fetch(int lane) {
        if (KEYS) {
            mine = at + lane < n ? bits[at + lane] : 0u;
            left = __ballot_sync(0xffffffffu, mine != 0u);
        } else {
            mine = at + lane < n ? (uint32_t)ids[at + lane] : 0u;
            left = __ballot_sync(0xffffffffu, at + lane < n);
        }
    }
    // -1: no more.  keys: head within the group in the upper, query block in the lower 32 bits
    __device__ long long next(int lane) {
        while (left == 0u) {
            at += 32;
            if (at >= n) return -1;
            fetch(lane);
        }
        const int src = __ffs(left) - 1;
        const uint32_t word = __shfl_sync(0xffffffffu, mine, src);
        if (!KEYS) {
            left &= left - 1;
            return (long long)word;
        }
        if (lane == src) mine &= mine - 1;
        if ((word & (word - 1)) == 0u) left &= left - 1;
        const int w = at + src, head = w / words_per_head;
        return ((long long)head << 32) | (unsigned)((w - head * words_per_head) * 32 + __ffs(word) - 1);
    }
};

template <bool KEYS>
__global__ void __launch_bounds__(SB_THREADS, 1)
selected_grad_sm100_kernel(const __grid_constant__ CUtensorMap tm_f1, const __grid_constant__ CUtensorMap tm_f2, const __grid_constant__ CUtensorMap tm_g1,
                           const __grid_constant__ CUtensorMap tm_g2, const __grid_constant__ CUtensorMap tm_d1, const __grid_constant__ CUtensorMap tm_d2,
                           const SbParams p) {
    using Ring = SbRing<KEYS>;
    constexpr int SLOTS = Ring::SLOTS;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *f_s = smem, *g_s = f_s + 2 * SB_OWN_BYTES, *p_s = g_s + SLOTS * TILE_BYTES;      // p_s: [P, dS], or [two steps] dS
    SbBarriers *bar = reinterpret_cast<SbBarriers *>(p_s + Ring::FACTORS * SB_P_BYTES);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    volatile int *abort_flag = &bar->abort_flag;
    const FailSink sink{p.error_flag, p.status_mirror};

    if (threadIdx.x == 0) {
        bar->abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;
        if (bar->abort_flag) report_failure(sink, 498);
        for (int i = 0; i < SB_DESCS; ++i) {
            mbar_init(&bar->desc_full[i], 1);
            mbar_init(&bar->desc_empty[i], 3 + SB_WORKERS);       // the warps that issue products or store, and the workers
        }
        mbar_init(&bar->f_full, 1);
        mbar_init(&bar->f_empty, 1);
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar->stats_full[i], 1);
            mbar_init(&bar->staged[i], SB_WORKERS / 2);
        }
        for (int i = 0; i < SLOTS; ++i) {
            mbar_init(&bar->full[i], 1);
            mbar_init(&bar->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar->s_full[i], 1);
            mbar_init(&bar->s_free[i], SB_WORKERS / 2);
            mbar_init(&bar->p_full[i], SB_WORKERS / 2);
            mbar_init(&bar->p_free[i], 1);
            mbar_init(&bar->stored[i], 1);
            mbar_init(&bar->acc_full[i], 1);
            mbar_init(&bar->acc_empty[i], SB_WORKERS / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == SB_WORKERS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (KEYS) {        // (dQ waits at its end: see wa_selected_backward)
        pdl_wait();
        pdl_release_dependents();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar->tmem_base;
    // columns: S of two steps, dP of two steps, then the sums of two items (each dV^T, dK^T or dQ^T)
    const uint32_t tm_s = tmem, tm_dp = tmem + 2 * SB_OWN, tm_acc = tmem + 4 * SB_OWN;

    if (warp == SB_WORKERS) {
        // ================= lists and loads =================
        const bool leader = elect_one();
        uint32_t descs = 0, items = 0, steps = 0;       // so many so far
        bool ok = true;
        int at = blockIdx.x;
        auto wait = [&](uint64_t *b, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, sink, code)); };
        auto tell = [&](int item, int flags, int of0, int of1) {
            const uint32_t d = descs % SB_DESCS;
            if (!wait(&bar->desc_empty[d], ((descs / SB_DESCS) & 1u) ^ 1u, 401)) return false;
            if (leader) {
                bar->desc[d].item = item;
                bar->desc[d].flags = flags;
                bar->desc[d].of[0] = of0;
                bar->desc[d].of[1] = of1;
                mbar_arrive(&bar->desc_full[d]);
            }
            __syncwarp();
            ++descs;
            return true;
        };
        while (ok) {
            if (at >= p.items) {
                tell(0, SB_END, 0, 0);
                break;
            }
            const int32_t *order = KEYS ? p.k_order : p.q_order;
            const int item = order ? order[at] : at;
            int next_at = 0;
            if (lane == 0) next_at = (int)gridDim.x + atomicAdd(p.work_counter, 1);
            const int tile = item % p.owned, head = item / p.owned;      // head: (batch, head) of the owned side
            const int b = head / (KEYS ? p.Hkv : p.H), h = head - b * (KEYS ? p.Hkv : p.H);
            const int hk = KEYS ? h : h / p.group;
            SbList<KEYS> list;
            list.begin(p, item, lane);
            long long ahead = list.next(lane);
            if (ahead < 0) {
                ok = tell(item, SB_EMPTY, 0, 0);
            } else {
                // the owned tile: its last score products of the item before are done
                ok = wait(&bar->f_empty, (items & 1u) ^ 1u, 402);
                if (ok && leader) {
                    mbar_expect_tx(&bar->f_full, 2 * SB_OWN_BYTES);
                    tma_load_5d(f_s, &tm_f1, &bar->f_full, 0, tile * SB_OWN, 0, h, b);
                    tma_load_5d(f_s + SB_OWN_BYTES, &tm_f2, &bar->f_full, 0, tile * SB_OWN, 0, h, b);
                    if (!KEYS) {
                        mbar_expect_tx(&bar->stats_full[items & 3u], SB_OWN * 8);
                        bulk_load(bar->stats + (items & 3u) * TILE, p.stats + ((long long)head * p.padded + tile * SB_OWN) * 2, SB_OWN * 8, &bar->stats_full[items & 3u]);
                    }
                }
                __syncwarp();
                ++items;
                int flags = SB_FIRST;
                while (ok && ahead >= 0) {
                    const long long one = ahead, two = list.next(lane);
                    ahead = two < 0 ? -1 : list.next(lane);
                    if (ahead < 0) flags |= SB_LAST;
                    // rows and heads of the two halves; what is missing lies behind the last block and loads as zeros
                    const int blocks = KEYS ? p.Nq : p.Nkv;
                    const int i0 = (int)(one & 0xffffffff), i1 = two < 0 ? blocks : (int)(two & 0xffffffff);
                    const int h0 = KEYS ? h * p.group + (int)(one >> 32) : hk, h1 = KEYS ? (two < 0 ? h0 : h * p.group + (int)(two >> 32)) : hk;
                    if (KEYS) ok = tell(item, flags, (int)((b * p.H + h0) * p.padded) + i0 * SB_OWN, (int)((b * p.H + h1) * p.padded) + i1 * SB_OWN);
                    else ok = tell(item, flags, min(p.Lkv - i0 * SB_OWN, SB_OWN), two < 0 ? 0 : min(p.Lkv - i1 * SB_OWN, SB_OWN));
                    flags = 0;
#pragma unroll
                    for (int g = 0; g < 2 && ok; ++g) {
                        const uint32_t slot = Ring::slot(g, steps);
                        ok = wait(&bar->empty[slot], Ring::parity(g, steps) ^ 1u, 403);
                        if (ok && leader) {
                            uint8_t *dst = g_s + slot * TILE_BYTES;
                            uint64_t *full = &bar->full[slot];
                            const CUtensorMap *map = g == 0 ? &tm_g1 : &tm_g2;
                            mbar_expect_tx(full, TILE_BYTES);
                            tma_load_5d(dst, map, full, 0, i0 * SB_OWN, 0, h0, b);
                            tma_load_5d(dst + HALF_BYTES / 2, map, full, 0, i1 * SB_OWN, 0, h1, b);
                            tma_load_5d(dst + HALF_BYTES, map, full, 0, i0 * SB_OWN, 1, h0, b);
                            tma_load_5d(dst + HALF_BYTES + HALF_BYTES / 2, map, full, 0, i1 * SB_OWN, 1, h1, b);
                        }
                        __syncwarp();
                    }
                    ++steps;
                }
            }
            at = __shfl_sync(0xffffffffu, next_at, 0);
        }
        if (*abort_flag) {      // given up: copies on their way land within microseconds, the block's shared memory is kept for a millisecond
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) { }
        }
    } else if (warp == SB_WORKERS + 1) {
        // ================= scores =================
        // One thread blocks for about as long as its products run, so that its waits and commits are time in which the tensor pipe idles; the scores
        // and the sums are issued by warps of their own, and each covers the other's.
        const bool leader = elect_one();
        constexpr uint32_t SCORE = instr_desc(false, SB_OWN);
        uint32_t descs = 0, items = 0, steps = 0;
        bool ok = true;
        auto wait = [&](uint64_t *b, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, sink, code)); };
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 411);
            if (!ok) break;
            const int flags = bar->desc[d].flags;
            __syncwarp();
            if (leader) mbar_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
            if (flags & SB_EMPTY) continue;
            if (flags & SB_FIRST) {
                ok = wait(&bar->f_full, items & 1u, 412);
                ++items;
            }
            const uint32_t buf = steps & 1u;
#pragma unroll
            for (int g = 0; g < 2 && ok; ++g) {
                const uint32_t slot = Ring::slot(g, steps);
                ok = wait(&bar->full[slot], Ring::parity(g, steps), 413);
                if (ok && g == 0) ok = wait(&bar->s_free[buf], ((steps >> 1) & 1u) ^ 1u, 414);      // the scores of step u - 2 have been read
                if (!ok) break;
                tc_fence_after();
                if (leader) {
                    const uint64_t a = smem_desc(smem_u32(g_s + slot * TILE_BYTES), 16, 1024), f = smem_desc(smem_u32(f_s + g * SB_OWN_BYTES), 16, 1024);
                    const uint32_t to = (g == 0 ? tm_s : tm_dp) + buf * SB_OWN;
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        mma_ss(to, a + (uint64_t)(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4), f + (uint64_t)(((kk >> 2) * (SB_OWN_BYTES / 2) + (kk & 3) * 32) >> 4), SCORE, kk > 0);
                    if (g == 1) tc_commit(&bar->s_full[buf]);
                    if (!KEYS && g == 1) tc_commit(&bar->empty[slot]);       // values take no part in dQ's sum
                    if (g == 1 && (flags & SB_LAST)) tc_commit(&bar->f_empty);
                }
                __syncwarp();
            }
            ++steps;
        }
    } else if (warp == SB_WORKERS + 2) {
        // ================= sums =================
        const bool leader = elect_one();
        constexpr uint32_t SUM = instr_desc(true, SB_OWN) | (1u << 15);      // both operands transposed
        uint32_t descs = 0, items = 0, steps = 0;
        bool ok = true;
        auto wait = [&](uint64_t *b, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, sink, code)); };
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 415);
            if (!ok) break;
            const int flags = bar->desc[d].flags;
            __syncwarp();
            if (leader) mbar_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
            if (flags & SB_EMPTY) continue;
            const bool fresh = flags & SB_FIRST;
            if (fresh) {
                ok = wait(&bar->acc_empty[items & 1u], ((items >> 1) & 1u) ^ 1u, 416);
                ++items;
            }
            const uint32_t buf = steps & 1u, s1 = Ring::slot(0, steps), s2 = Ring::slot(1, steps), last = (items - 1) & 1u;
            const uint32_t acc = tm_acc + last * 2 * SB_OWN;
            const uint8_t *factors = p_s + (KEYS ? 0 : buf * SB_P_BYTES);
            auto add = [&](uint32_t to, uint32_t slot, const uint8_t *factor) {
                const uint64_t a = smem_desc(smem_u32(g_s + slot * TILE_BYTES), HALF_BYTES, 1024), f = smem_desc(smem_u32(factor), HALF_BYTES, 1024);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) mma_ss(to, a + (uint64_t)((kk * 2048) >> 4), f + (uint64_t)((kk * 2048) >> 4), SUM, !(fresh && kk == 0));
            };
            if (ok) ok = wait(&bar->p_full[buf], (steps >> 1) & 1u, 417);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
                // (the factors were made from both scores: those have read their tiles too)
                if (KEYS) {
                    add(acc, s2, factors);
                    tc_commit(&bar->empty[s2]);
                }
                add(acc + SB_OWN, s1, factors + (KEYS ? SB_P_BYTES : 0));
                if (!KEYS || !(flags & SB_LAST)) tc_commit(&bar->empty[s1]);       // (keys: the item's sums are left in its last slot, free when they are stored)
                tc_commit(&bar->p_free[buf]);
                if (flags & SB_LAST) tc_commit(&bar->acc_full[last]);
            }
            __syncwarp();
            ++steps;
        }
    } else if (warp == SB_WORKERS + 3) {
        // ================= stores =================
        uint32_t descs = 0, steps = 0, items = 0;
        bool ok = true;
        auto wait = [&](uint64_t *b, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, sink, code)); };
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 427);
            if (!ok) break;
            const int item = bar->desc[d].item, flags = bar->desc[d].flags;
            warp_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
            if (flags & SB_EMPTY) continue;
            const uint32_t buf = steps & 1u, slot = Ring::slot(0, steps);
            ++steps;
            if (!(flags & SB_LAST)) continue;
            ok = wait(&bar->staged[items & 3u], (items >> 2) & 1u, 428);
            if (!ok) break;
            ++items;
            if (lane == 0) {
                const int tile = item % p.owned, head = item / p.owned, heads = KEYS ? p.Hkv : p.H, b = head / heads, h = head - b * heads;
                const uint8_t *from = KEYS ? g_s + slot * TILE_BYTES : p_s + buf * SB_P_BYTES;
                // (rows behind the last one are clipped by the map)
                if (KEYS) tma_store_5d(&tm_d1, from, 0, tile * SB_OWN, 0, h, b);
                tma_store_5d(&tm_d2, from + (KEYS ? SB_OWN_BYTES : 0), 0, tile * SB_OWN, 0, h, b);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                mbar_arrive(KEYS ? &bar->empty[slot] : &bar->stored[buf]);
            }
            __syncwarp();
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");      // all stores have landed before the block exits
        __syncwarp();
    } else {
        // ================= P, dS and the finished sums =================
        // Two groups of eight warps take the steps in turn: a step is a chain of waits, tensor-memory reads, exponentials and fences, longer than
        // its products take, and two of them overlap.  A thread has one met row (tensor-memory lane) and 32 of its 64 columns, 16 at a time.
        // The group that took an item's last step leaves the finished sums, as bf16, in that step's slot, or where its dS was, and a warp of its own stores
        // them: it would only wait otherwise.  (dQ's in the slot, too, one of three: window 614 -> 632 us.  Stored by all workers from registers, 64 bytes of
        // a row at a time, the sums of an item held either group up for 3900 cycles, dQ's for 2100: one and a half steps.)
        const int quarter = warp & 3, half = (warp >> 2) & 1, group = warp >> 3, part = warp >> 2, row = quarter * 32 + lane;
        const uint32_t lane_addr = ((uint32_t)(quarter * 32)) << 16;
        uint32_t descs = 0, steps = 0, items = 0, staged = 0;       // staged: by this group
        bool ok = true;
        auto wait = [&](uint64_t *b, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, sink, code)); };
        // zeros for channel `row` of 16 owned rows
        auto clear = [&](int item, __nv_bfloat16 *to, long long sb, long long sl, long long sh) {
            const int tile = item % p.owned, head = item / p.owned, heads = KEYS ? p.Hkv : p.H;
            const int b = head / heads, h = head - b * heads, first = tile * SB_OWN + part * 16;
            const int n = min(16, (KEYS ? p.Lkv : p.Lq) - first);
            __nv_bfloat16 *at = to + b * sb + (long long)first * sl + h * sh + row;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < n) at[j * sl] = __float2bfloat16_rn(0.f);
        };
        // the sums of the item that ends with this group's step: [half of the channels][owned row][64 channels], pieces of 16 bytes swizzled by row
        auto finish = [&](uint8_t *to) {
            const uint32_t it = items - 1, a = it & 1u;
            if (!wait(&bar->acc_full[a], (it >> 1) & 1u, 421)) return false;       // (the sums of this step have read its tiles and factors, too)
            tc_fence_after();
            to += (row >> 6) * (SB_OWN_BYTES / 2) + (row & 7) * 2;
            const int piece = (row & 63) >> 3;
#pragma unroll 1
            for (int g = 0; g < (KEYS ? 4 : 2); ++g) {
                const int col = half * 32 + (g & 1) * 16, of = KEYS ? g >> 1 : 1;       // dV, then dK; or dQ
                uint32_t v[16];
                TMEM_LD16(tm_acc + (a * 2 + of) * SB_OWN + col + lane_addr, v);
                tmem_wait_ld16(v);
                if (g + 1 == (KEYS ? 4 : 2)) {
                    tc_fence_before();
                    warp_arrive(&bar->acc_empty[a]);
                }
                const float scale = of ? p.scale : 1.0f;
                uint8_t *at = to + (KEYS ? of * SB_OWN_BYTES : 0) + col * 128;
#pragma unroll
                for (int j = 0; j < 16; ++j) *reinterpret_cast<__nv_bfloat16 *>(at + j * 128 + ((piece ^ (j & 7)) << 4)) = __float2bfloat16_rn(__uint_as_float(v[j]) * scale);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(&bar->staged[it & 3u]);
            ++staged;
            return true;
        };
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 422);
            if (!ok) break;
            const SbDesc desc = bar->desc[d];
            warp_arrive(&bar->desc_empty[d]);
            ++descs;
            if (desc.flags & SB_END) break;
            if (desc.flags & SB_EMPTY) {
                if (KEYS) clear(desc.item, p.d1, p.d1b, p.d1l, p.d1h);
                clear(desc.item, p.d2, p.d2b, p.d2l, p.d2h);
                continue;
            }
            if (desc.flags & SB_FIRST) {
                if (!KEYS) ok = wait(&bar->stats_full[items & 3u], (items >> 2) & 1u, 423);
                ++items;
            }
            if ((steps & 1u) == (uint32_t)group && ok) {
                const uint32_t buf = steps & 1u;
                // (-normaliser, -delta) of the met row, or of the owned rows: 64 of one, 64 of the other
                const float *st = bar->stats + ((items - 1) & 3u) * TILE;
                const int of = row < SB_OWN ? desc.of[0] : desc.of[1];
                float2 norm = make_float2(0.f, 0.f), delta = norm;
                if (KEYS) {        // (on their way while the scores are)
                    const float *at = p.stats + (long long)of * 2 + (row & 63);
                    norm.x = norm.y = __ldg(at);
                    delta.x = delta.y = __ldg(at + SB_OWN);
                }
                // queries: rows that are no keys
                const bool real = KEYS || (row & 63) < of;
                if (!KEYS) {       // the sums of step u - 2 have read the factors that lie here, and a store what was left since
                    if (ok) ok = wait(&bar->p_free[buf], ((steps >> 1) & 1u) ^ 1u, 425);
                    if (ok) ok = wait(&bar->stored[buf], (staged & 1u) ^ 1u, 424);
                }
                if (ok) ok = wait(&bar->s_full[buf], (steps >> 1) & 1u, 426);
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_at = tm_s + buf * SB_OWN + lane_addr, dp_at = tm_dp + buf * SB_OWN + lane_addr;
                const float2 c = make_float2(p.scale_log2, p.scale_log2);
                uint32_t pw[2][8], dw[2][8];       // P (keys) and dS as pairs of bf16
                uint8_t *factors = p_s + (KEYS ? 0 : buf * SB_P_BYTES) + row * 128;
                auto leave = [&](int n) {          // 16 columns, 16-byte pieces swizzled by row
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint8_t *to = factors + (((half * 4 + 2 * n + q) ^ (row & 7)) << 4);
                        if (KEYS) *reinterpret_cast<uint4 *>(to) = make_uint4(pw[n][4 * q], pw[n][4 * q + 1], pw[n][4 * q + 2], pw[n][4 * q + 3]);
                        *reinterpret_cast<uint4 *>(to + (KEYS ? SB_P_BYTES : 0)) = make_uint4(dw[n][4 * q], dw[n][4 * q + 1], dw[n][4 * q + 2], dw[n][4 * q + 3]);
                    }
                };
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int col = half * 32 + n * 16;
                    uint32_t x[16], y[16];
                    TMEM_LD16(s_at + col, x);
                    TMEM_LD16(dp_at + col, y);
                    tmem_wait_ld16(x);
                    tmem_wait_ld16(y);
                    if (n == 1) {
                        tc_fence_before();
                        warp_arrive(&bar->s_free[buf]);
                    }
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        float4 n4 = make_float4(norm.x, norm.x, norm.x, norm.x), d4;
                        if (!KEYS) {
                            n4 = *reinterpret_cast<const float4 *>(st + col + j);
                            d4 = *reinterpret_cast<const float4 *>(st + SB_OWN + col + j);
                        }
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const float2 nn = e == 0 ? make_float2(n4.x, n4.y) : make_float2(n4.z, n4.w);
                            const float2 d = KEYS ? delta : e == 0 ? make_float2(d4.x, d4.y) : make_float2(d4.z, d4.w);
                            const float2 z = __ffma2_rn(make_float2(__uint_as_float(x[j + e]), __uint_as_float(x[j + e + 1])), c, nn);
                            float2 pr = make_float2(ex2(z.x), ex2(z.y));
                            float2 ds = __fmul2_rn(pr, __fadd2_rn(make_float2(__uint_as_float(y[j + e]), __uint_as_float(y[j + e + 1])), d));
                            if (!KEYS && !real) ds = make_float2(0.f, 0.f);
                            const __nv_bfloat162 hp = __floats2bfloat162_rn(pr.x, pr.y), hd = __floats2bfloat162_rn(ds.x, ds.y);
                            if (KEYS) pw[n][(j + e) >> 1] = *reinterpret_cast<const uint32_t *>(&hp);
                            dw[n][(j + e) >> 1] = *reinterpret_cast<const uint32_t *>(&hd);
                        }
                    }
                    if (!KEYS) leave(n);
                }
                if (KEYS) {
                    // the sums of the step before have read the factors that lie here.  (On a barrier for every other step, so that a group cannot mistake the
                    // end of the step before that for it: it has waited for the one before its last step.)
                    ok = wait(&bar->p_free[buf ^ 1u], ((steps - 1u) >> 1) & 1u, 425);
                    if (!ok) break;
                    if (__builtin_expect(norm.x == -INFINITY, 0)) {      // no query: its scores are no numbers where a key holds an infinity
#pragma unroll
                        for (int j = 0; j < 8; ++j) pw[0][j] = pw[1][j] = dw[0][j] = dw[1][j] = 0u;
                    }
                    leave(0);
                    leave(1);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&bar->p_full[buf]);
                if (desc.flags & SB_LAST) ok = finish(KEYS ? g_s + Ring::slot(0, steps) * TILE_BYTES : p_s + buf * SB_P_BYTES);
            }
            ++steps;
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == SB_WORKERS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    if (!KEYS) pdl_wait();
}

// ---- blocks of 128 tokens ---------------------------------------------------------------------------
// An item owns a whole block, and the roles of the operands change:
//     S = F1 G1^T   dP = F2 G2^T               [128 owned rows x 128 met ones]
//     dV += P G2   dK (or dQ) += dS G1         [128 owned rows x 128 channels]
// P and dS go back to tensor memory over the scores that they were made from and are first operands from there; shared memory holds nothing but
// tiles, its reads (two tiles for 128 columns of a score product, one for a sum) are half those of the kernel above for the same
// work, and a met tile is loaded half as often.  A warp writes its 32 columns of P as 16 words over the first half of its own 32 columns of S, so
// that no warp waits for another's reads; the products take each K step's address from there.
// Finished sums leave through the last step's slots, of which G1's and G2's are kept as above: the workers leave them there as bf16, and a warp of its own stores
// them and gives the slots back.  (Stored by the workers themselves, 32 rows of 16 or 32 bytes at a time, an item's end took
// 8000 cycles, three steps' time; lists of a chunk's keys are five steps long.)
// What bounds it: as above; the tensor pipe is busy 66 % of the time for dQ, and 50 % for dK/dV, whose items are short (five steps): each ends with a
// chain of sums, reads, stores and the next one's tiles.  4680 queries, 32 of 256 blocks a row, 12 heads: dK/dV 230 us, dQ 145 (131 behind the other; 299
// and 217 before the two changes above).  Tried: an item's sums left in the next item's first step 255 us.
// Tensor memory: S, dP, dV and dK; or S, two of dP, and dQ.  Scores of step u + 1 follow as soon as their columns are free: behind the sum that
// read P or dS, or, for dQ's S, behind the workers' reads.
template <bool KEYS>
struct SwBarriers {
    float stats[2][2 * TILE];         // keys: of the met rows, per step; 64 rows' (-normaliser), their (-delta), and the same of the others
    uint64_t desc_full[SB_DESCS], desc_empty[SB_DESCS];
    uint64_t f_full, f_empty, stats_full[2], stats_empty[2];
    uint64_t full[5], empty[5];
    uint64_t s_full, s_free, p_full;
    uint64_t dp_full[2], dp_free[2], ds_full[2];
    uint64_t acc_full[2], acc_empty[2], staged[2][SB_DESCS];   // of dK or dQ, and of dV
    uint32_t tmem_base;
    int abort_flag;
    SbDesc desc[SB_DESCS];
};
constexpr int SW_SMEM = (2 + SbRing<true>::SLOTS) * TILE_BYTES + SB_BARRIER_BYTES;
static_assert(sizeof(SwBarriers<true>) <= SB_BARRIER_BYTES && SW_SMEM <= 227 * 1024, "shared memory budget exceeded");

template <bool KEYS>
__global__ void __launch_bounds__(SB_THREADS, 1)
selected_grad_wide_kernel(const __grid_constant__ CUtensorMap tm_f1, const __grid_constant__ CUtensorMap tm_f2, const __grid_constant__ CUtensorMap tm_g1,
                          const __grid_constant__ CUtensorMap tm_g2, const __grid_constant__ CUtensorMap tm_d1, const __grid_constant__ CUtensorMap tm_d2,
                          const SbParams p) {
    constexpr int DPS = KEYS ? 1 : 2;                    // buffers of dP
    using Ring = SbRing<KEYS>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *f_s = smem, *g_s = f_s + 2 * TILE_BYTES;
    SwBarriers<KEYS> *bar = reinterpret_cast<SwBarriers<KEYS> *>(g_s + Ring::SLOTS * TILE_BYTES);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    volatile int *abort_flag = &bar->abort_flag;
    const FailSink sink{p.error_flag, p.status_mirror};

    if (threadIdx.x == 0) {
        bar->abort_flag = (smem_u32(smem) & 1023u) ? 1 : 0;
        if (bar->abort_flag) report_failure(sink, 498);
        for (int i = 0; i < SB_DESCS; ++i) {
            mbar_init(&bar->desc_full[i], 1);
            mbar_init(&bar->desc_empty[i], 3 + SB_WORKERS);
            mbar_init(&bar->staged[0][i], SB_WORKERS);
            mbar_init(&bar->staged[1][i], SB_WORKERS);
        }
        mbar_init(&bar->f_full, 1);
        mbar_init(&bar->f_empty, 1);
        for (int i = 0; i < Ring::SLOTS; ++i) {
            mbar_init(&bar->full[i], 1);
            mbar_init(&bar->empty[i], 1);
        }
        mbar_init(&bar->s_full, 1);
        mbar_init(&bar->s_free, KEYS ? 1 : SB_WORKERS);  // the sum that read P; the workers that read S
        mbar_init(&bar->p_full, SB_WORKERS);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar->stats_full[i], 1);
            mbar_init(&bar->stats_empty[i], SB_WORKERS);
            mbar_init(&bar->dp_full[i], 1);
            mbar_init(&bar->dp_free[i], 1);
            mbar_init(&bar->ds_full[i], SB_WORKERS);
            mbar_init(&bar->acc_full[i], 1);
            mbar_init(&bar->acc_empty[i], SB_WORKERS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == SB_WORKERS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem_base)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (KEYS) {        // (dQ waits at its end: see wa_selected_backward)
        pdl_wait();
        pdl_release_dependents();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar->tmem_base;
    const uint32_t tm_s = tmem, tm_dp = tmem + TILE, tm_sum1 = tmem + 2 * TILE, tm_sum2 = tmem + 3 * TILE;       // (dQ: the second dP lies at tm_sum1)
    auto wait = [&](uint64_t *b, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, sink, code)); };

    if (warp == SB_WORKERS) {
        // ================= lists and loads =================
        const bool leader = elect_one();
        uint32_t descs = 0, items = 0, steps = 0;
        bool ok = true;
        int at = blockIdx.x;
        auto tell = [&](int item, int flags, int real) {
            const uint32_t d = descs % SB_DESCS;
            if (!wait(&bar->desc_empty[d], ((descs / SB_DESCS) & 1u) ^ 1u, 431)) return false;
            if (leader) {
                bar->desc[d].item = item;
                bar->desc[d].flags = flags;
                bar->desc[d].of[0] = real;
                mbar_arrive(&bar->desc_full[d]);
            }
            __syncwarp();
            ++descs;
            return true;
        };
        while (ok) {
            if (at >= p.items) {
                tell(0, SB_END, 0);
                break;
            }
            const int32_t *order = KEYS ? p.k_order : p.q_order;
            const int item = order ? order[at] : at;
            int next_at = 0;
            if (lane == 0) next_at = (int)gridDim.x + atomicAdd(p.work_counter, 1);
            const int tile = item % p.owned, head = item / p.owned;
            const int b = head / (KEYS ? p.Hkv : p.H), h = head - b * (KEYS ? p.Hkv : p.H);
            const int hk = KEYS ? h : h / p.group;
            SbList<KEYS> list;
            list.begin(p, item, lane);
            long long ahead = list.next(lane);
            if (ahead < 0) {
                ok = tell(item, SB_EMPTY, 0);
            } else {
                ok = wait(&bar->f_empty, (items & 1u) ^ 1u, 432);
                if (ok && leader) {
                    mbar_expect_tx(&bar->f_full, 2 * TILE_BYTES);
                    tma_load_5d(f_s, &tm_f1, &bar->f_full, 0, tile * TILE, 0, h, b);
                    tma_load_5d(f_s + TILE_BYTES, &tm_f2, &bar->f_full, 0, tile * TILE, 0, h, b);
                }
                __syncwarp();
                ++items;
                int flags = SB_FIRST;
                while (ok && ahead >= 0) {
                    const int i0 = (int)(ahead & 0xffffffff), h0 = KEYS ? h * p.group + (int)(ahead >> 32) : hk;
                    ahead = list.next(lane);
                    if (ahead < 0) flags |= SB_LAST;
                    ok = tell(item, flags, min((KEYS ? p.Lq : p.Lkv) - i0 * TILE, TILE));
                    flags = 0;
#pragma unroll
                    for (int g = 0; g < 2 && ok; ++g) {
                        const uint32_t slot = Ring::slot(g, steps);
                        ok = wait(&bar->empty[slot], Ring::parity(g, steps) ^ 1u, 433);
                        if (ok && leader) {
                            mbar_expect_tx(&bar->full[slot], TILE_BYTES);
                            tma_load_5d(g_s + slot * TILE_BYTES, g == 0 ? &tm_g1 : &tm_g2, &bar->full[slot], 0, i0 * TILE, 0, h0, b);
                        }
                        __syncwarp();
                    }
                    if (KEYS && ok) {      // (behind the tiles: it waits for the workers to be through with step u - 2, which the next tiles would as well)
                        const uint32_t s = steps & 1u;
                        ok = wait(&bar->stats_empty[s], ((steps >> 1) & 1u) ^ 1u, 434);
                        if (ok && leader) {
                            mbar_expect_tx(&bar->stats_full[s], TILE * 8);
                            bulk_load(bar->stats[s], p.stats + (((long long)b * p.H + h0) * p.padded + (long long)i0 * TILE) * 2, TILE * 8, &bar->stats_full[s]);
                        }
                        __syncwarp();
                    }
                    ++steps;
                }
            }
            at = __shfl_sync(0xffffffffu, next_at, 0);
        }
        if (*abort_flag) {      // given up: copies on their way land within microseconds, the block's shared memory is kept for a millisecond
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) { }
        }
    } else if (warp == SB_WORKERS + 1) {
        // ================= scores =================
        const bool leader = elect_one();
        constexpr uint32_t SCORE = instr_desc(false, TILE);
        uint32_t descs = 0, items = 0, steps = 0;
        bool ok = true;
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 441);
            if (!ok) break;
            const int flags = bar->desc[d].flags;
            __syncwarp();
            if (leader) mbar_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
            if (flags & SB_EMPTY) continue;
            if (flags & SB_FIRST) {
                ok = wait(&bar->f_full, items & 1u, 442);
                ++items;
            }
            const uint32_t buf = steps % DPS;
#pragma unroll
            for (int g = 0; g < 2 && ok; ++g) {
                const uint32_t slot = Ring::slot(g, steps);
                ok = wait(&bar->full[slot], Ring::parity(g, steps), 443);
                if (ok) ok = g == 0 ? wait(&bar->s_free, (steps & 1u) ^ 1u, 444) : wait(&bar->dp_free[buf], ((steps / DPS) & 1u) ^ 1u, 445);
                if (!ok) break;
                tc_fence_after();
                if (leader) {
                    const uint64_t f = smem_desc(smem_u32(f_s + g * TILE_BYTES), 16, 1024), m = smem_desc(smem_u32(g_s + slot * TILE_BYTES), 16, 1024);
                    const uint32_t to = g == 0 ? tm_s : tm_dp + buf * TILE;
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint64_t off = (uint64_t)(((kk >> 2) * HALF_BYTES + (kk & 3) * 32) >> 4);
                        mma_ss(to, f + off, m + off, SCORE, kk > 0);
                    }
                    tc_commit(g == 0 ? &bar->s_full : &bar->dp_full[buf]);
                    if (!KEYS && g == 1) tc_commit(&bar->empty[slot]);       // values take no part in dQ's sum
                    if (g == 1 && (flags & SB_LAST)) tc_commit(&bar->f_empty);
                }
                __syncwarp();
            }
            ++steps;
        }
    } else if (warp == SB_WORKERS + 2) {
        // ================= sums =================
        const bool leader = elect_one();
        constexpr uint32_t SUM = instr_desc(true, TILE);
        uint32_t descs = 0, items = 0, steps = 0;
        bool ok = true;
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 451);
            if (!ok) break;
            const int flags = bar->desc[d].flags;
            __syncwarp();
            if (leader) mbar_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
            if (flags & SB_EMPTY) continue;
            const bool fresh = flags & SB_FIRST;
            if (fresh) ++items;
            const uint32_t buf = steps % DPS, s1 = Ring::slot(0, steps), s2 = Ring::slot(1, steps);
            auto add = [&](uint32_t to, uint32_t factor, uint32_t slot) {       // factor: 8 words a K step, two steps of each 32 columns
                const uint64_t m = smem_desc(smem_u32(g_s + slot * TILE_BYTES), HALF_BYTES, 1024);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    mma_ts(to, factor + (kk >> 1) * 32 + (kk & 1) * 8, m + (uint64_t)((kk * 2048) >> 4), SUM, !(fresh && kk == 0));
            };
            if (KEYS) {
                if (fresh) ok = wait(&bar->acc_empty[1], items & 1u, 452);
                if (ok) ok = wait(&bar->p_full, steps & 1u, 453);
                if (ok) ok = wait(&bar->full[s2], Ring::parity(1, steps), 455);       // (P needs its query rows only, not yet those of dout)
                if (!ok) break;
                tc_fence_after();
                if (leader) {
                    add(tm_sum1, tm_s, s2);
                    tc_commit(&bar->s_free);
                    if (flags & SB_LAST) tc_commit(&bar->acc_full[1]);
                }
                __syncwarp();
            }
            if (fresh && ok) ok = wait(&bar->acc_empty[0], items & 1u, 452);
            if (ok) ok = wait(&bar->ds_full[buf], (steps / DPS) & 1u, 454);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
                // (An item's sums are left in its last step's slots: those are free when they are stored.)
                if (KEYS && !(flags & SB_LAST)) tc_commit(&bar->empty[s2]);      // free with dV's sum: dS was made from dP, which has read it too
                add(tm_sum2, tm_dp + buf * TILE, s1);
                tc_commit(&bar->dp_free[buf]);
                if (!(flags & SB_LAST)) tc_commit(&bar->empty[s1]);
                else tc_commit(&bar->acc_full[0]);
            }
            __syncwarp();
            ++steps;
        }
    } else if (warp == SB_WORKERS + 3) {
        // ================= stores =================
        uint32_t descs = 0, steps = 0, items = 0;
        bool ok = true;
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 456);
            if (!ok) break;
            const int item = bar->desc[d].item, flags = bar->desc[d].flags;
            if (flags & SB_LAST) {
                const int tile = item % p.owned, head = item / p.owned, b = head / (KEYS ? p.Hkv : p.H), h = head - b * (KEYS ? p.Hkv : p.H);
#pragma unroll
                for (int g = KEYS ? 1 : 0; g >= 0 && ok; --g) {
                    ok = wait(&bar->staged[g][items % SB_DESCS], (items / SB_DESCS) & 1u, 457);
                    if (ok && lane == 0) {
                        const uint32_t slot = Ring::slot(g, steps);
                        tma_store_5d(g == 1 ? &tm_d1 : &tm_d2, g_s + slot * TILE_BYTES, 0, tile * TILE, 0, h, b);       // (rows behind the last one are clipped by the map)
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        mbar_arrive(&bar->empty[slot]);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                ++items;
            }
            if (!(flags & (SB_EMPTY | SB_END))) ++steps;
            // only now: a ring of descriptions is then also a bound on the items that are staged and not yet stored
            warp_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");      // all stores have landed before the block exits
        __syncwarp();
    } else {
        // ================= P, dS and the finished sums =================
        // a thread has one owned row (tensor-memory lane) and 32 met ones (columns)
        const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;
        const uint32_t at = (((uint32_t)(quarter * 32)) << 16) + part * 32;
        uint32_t descs = 0, steps = 0, items = 0;
        bool ok = true;
        float2 norm = make_float2(0.f, 0.f), delta = norm;        // queries: of the row
        const float2 c = make_float2(p.scale_log2, p.scale_log2);
        // an item's sums to its last step's slots: [half of the channels][row][64 channels], pieces of 16 bytes swizzled by row
        auto finish = [&]() {
#pragma unroll 1
            for (int g = KEYS ? 1 : 0; g >= 0; --g) {      // dV to G2's slot, while dK's products run; dK or dQ to G1's
                if (!wait(&bar->acc_full[g], items & 1u, 465)) return false;
                tc_fence_after();
                uint32_t v[32];
                TMEM_LD32((g == 0 ? tm_sum2 : tm_sum1) + at, v);
                tmem_wait_ld32(v);
                tc_fence_before();
                warp_arrive(&bar->acc_empty[g]);
                const float scale = g == 0 ? p.scale : 1.0f;
                uint8_t *to = g_s + Ring::slot(g, steps) * TILE_BYTES + (part >> 1) * HALF_BYTES + row * 128;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(v[8 * q + 2 * e]) * scale, __uint_as_float(v[8 * q + 2 * e + 1]) * scale);
                        w[e] = *reinterpret_cast<const uint32_t *>(&x);
                    }
                    *reinterpret_cast<uint4 *>(to + ((((part & 1) * 4 + q) ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                warp_arrive(&bar->staged[g][items % SB_DESCS]);
            }
            ++items;
            return true;
        };
        // zeros for a quarter of the channels of 32 of an item's rows
        auto clear = [&](int item, __nv_bfloat16 *to, long long sb, long long sl, long long sh) {
            const int tile = item % p.owned, head = item / p.owned, heads = KEYS ? p.Hkv : p.H, b = head / heads, l = tile * TILE + row;
            if (l >= (KEYS ? p.Lkv : p.Lq)) return;
            uint4 *out = reinterpret_cast<uint4 *>(to + b * sb + (long long)l * sl + (head - b * heads) * sh + part * 32);
#pragma unroll
            for (int q = 0; q < 4; ++q) out[q] = make_uint4(0u, 0u, 0u, 0u);
        };
        while (ok) {
            const uint32_t d = descs % SB_DESCS;
            ok = wait(&bar->desc_full[d], (descs / SB_DESCS) & 1u, 461);
            if (!ok) break;
            const int item = bar->desc[d].item, flags = bar->desc[d].flags, real = bar->desc[d].of[0];
            warp_arrive(&bar->desc_empty[d]);
            ++descs;
            if (flags & SB_END) break;
            if (flags & SB_EMPTY) {
                if (KEYS) clear(item, p.d1, p.d1b, p.d1l, p.d1h);
                clear(item, p.d2, p.d2b, p.d2l, p.d2h);
                continue;
            }
            if (!KEYS && (flags & SB_FIRST)) {
                const int head = item / p.owned;
                const float *st = p.stats + (long long)head * p.padded * 2 + selected_stat((item - head * p.owned) * TILE + row);
                norm = make_float2(st[0], st[0]);
                delta = make_float2(st[64], st[64]);
            }
            uint32_t v[32];
            const uint32_t s2 = steps & 1u, buf = steps % DPS;
            const float *st = bar->stats[s2] + (part >> 1) * TILE + (part & 1) * 32;       // keys: of the 32 met rows
            if (KEYS) ok = wait(&bar->stats_full[s2], (steps >> 1) & 1u, 462);
            if (ok) ok = wait(&bar->s_full, steps & 1u, 463);
            if (!ok) break;
            tc_fence_after();
            float2 pr[16];
            TMEM_LD32(tm_s + at, v);
            tmem_wait_ld32(v);
            if (!KEYS) {
                tc_fence_before();
                warp_arrive(&bar->s_free);
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float4 n4 = KEYS ? *reinterpret_cast<const float4 *>(st + 2 * j) : make_float4(norm.x, norm.x, norm.x, norm.x);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 z = __ffma2_rn(make_float2(__uint_as_float(v[2 * (j + e)]), __uint_as_float(v[2 * (j + e) + 1])), c,
                                                e == 0 ? make_float2(n4.x, n4.y) : make_float2(n4.z, n4.w));
                    pr[j + e] = make_float2(ex2(z.x), ex2(z.y));
                }
            }
            uint32_t w[16];
            auto pack = [&]() {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const __nv_bfloat162 x = __floats2bfloat162_rn(pr[j].x, pr[j].y);
                    w[j] = *reinterpret_cast<const uint32_t *>(&x);
                }
            };
            if (real < TILE) {      // tokens that are none (the last block): a score of theirs is no number where the owned row holds an infinity
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (part * 32 + 2 * j >= real) pr[j].x = 0.f;
                    if (part * 32 + 2 * j + 1 >= real) pr[j].y = 0.f;
                }
            }
            if (KEYS) {
                pack();
                TMEM_ST16(tm_s + at, w);
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(&bar->p_full);
            }
            ok = wait(&bar->dp_full[buf], (steps / DPS) & 1u, 464);
            if (!ok) break;
            tc_fence_after();
            TMEM_LD32(tm_dp + buf * TILE + at, v);
            tmem_wait_ld32(v);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float4 d4 = KEYS ? *reinterpret_cast<const float4 *>(st + SB_OWN + 2 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 x = make_float2(__uint_as_float(v[2 * (j + e)]), __uint_as_float(v[2 * (j + e) + 1]));
                    const float2 dl = KEYS ? (e == 0 ? make_float2(d4.x, d4.y) : make_float2(d4.z, d4.w)) : delta;
                    pr[j + e] = __fmul2_rn(pr[j + e], __fadd2_rn(x, dl));
                }
            }
            pack();
            TMEM_ST16(tm_dp + buf * TILE + at, w);
            tmem_wait_st();
            tc_fence_before();
            if (KEYS) warp_arrive(&bar->stats_empty[s2]);
            warp_arrive(&bar->ds_full[buf]);
            if (flags & SB_LAST) ok = finish();
            ++steps;
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == SB_WORKERS) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    if (!KEYS) pdl_wait();
}

static bool aligned_view(const wa_tensor4 *t) {
    return t->ptr && (uintptr_t)t->ptr % 16 == 0 && t->stride_h % 8 == 0 && t->stride_l % 8 == 0 && t->stride_b % 8 == 0 && t->stride_h > 0 && t->stride_l > 0;
}

template <bool KEYS, int BLK>      // BLK: 64, or 128 for the kernel that owns whole blocks of 128
static int launch_owned(const wa_selected_params *p, SbParams kp, cudaStream_t stream) {
    const char *what = "wa_selected_backward(tcgen05)";
    constexpr int OWN = BLK == TILE ? TILE : SB_OWN, SMEM = BLK == TILE ? SW_SMEM : SbRing<KEYS>::SMEM;
    const wa_tensor4 &f1 = KEYS ? p->k : p->q, &f2 = KEYS ? p->v : p->dout, &g1 = KEYS ? p->q : p->k, &g2 = KEYS ? p->dout : p->v;
    const int Lf = KEYS ? p->Lkv : p->Lq, Hf = KEYS ? p->Hkv : p->H, Lg = KEYS ? p->Lq : p->Lkv, Hg = KEYS ? p->H : p->Hkv;
    CUtensorMap maps[4];
    int rc;
    if ((rc = selected_sm100_map(&maps[0], &f1, p->B, Lf, Hf, "the owned rows", OWN, 2))) return rc;
    if ((rc = selected_sm100_map(&maps[1], &f2, p->B, Lf, Hf, "the owned rows", OWN, 2))) return rc;
    if ((rc = selected_sm100_map(&maps[2], &g1, p->B, Lg, Hg, "the met rows", BLK, BLK == TILE ? 2 : 1))) return rc;
    if ((rc = selected_sm100_map(&maps[3], &g2, p->B, Lg, Hg, "the met rows", BLK, BLK == TILE ? 2 : 1))) return rc;
    static PerDeviceOnce attr_set;
    if (!attr_set.done()) {
        cudaError_t e;
        if constexpr (BLK == TILE) e = cudaFuncSetAttribute(selected_grad_wide_kernel<KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        else e = cudaFuncSetAttribute(selected_grad_sm100_kernel<KEYS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
        attr_set.mark();
    }
    kp.owned = ceil_div(Lf, OWN);
    kp.items = p->B * Hf * kp.owned;
    const wa_tensor4 &d2 = KEYS ? p->dk : p->dq;
    kp.d1 = (__nv_bfloat16 *)p->dv.ptr; kp.d1b = p->dv.stride_b; kp.d1l = p->dv.stride_l; kp.d1h = p->dv.stride_h;
    kp.d2 = (__nv_bfloat16 *)d2.ptr; kp.d2b = d2.stride_b; kp.d2l = d2.stride_l; kp.d2h = d2.stride_h;
    kp.work_counter += KEYS ? 0 : 1;
    const int sms = sm_count();
    const dim3 grid(kp.items < sms ? kp.items : sms);
    cudaError_t e;
    CUtensorMap outs[2];
    if ((rc = selected_sm100_map(&outs[0], KEYS ? &p->dv : &p->dq, p->B, Lf, Hf, "a gradient", OWN, 2))) return rc;
    if ((rc = selected_sm100_map(&outs[1], KEYS ? &p->dk : &p->dq, p->B, Lf, Hf, "a gradient", OWN, 2))) return rc;
    if constexpr (BLK == TILE) {
        e = launch_dependent(selected_grad_wide_kernel<KEYS>, grid, dim3(SB_THREADS), SMEM, stream, maps[0], maps[1], maps[2], maps[3], outs[0], outs[1], kp);
    } else {
        e = launch_dependent(selected_grad_sm100_kernel<KEYS>, grid, dim3(SB_THREADS), SMEM, stream, maps[0], maps[1], maps[2], maps[3], outs[0], outs[1], kp);
    }
    if (e != cudaSuccess) return fail((int)e, "%s: %s", what, cudaGetErrorString(e));
    return check_launch(what);
}

}  // namespace sm100

bool selected_sm100_backward_supported(const wa_selected_params *p) {
    using namespace sm100;
    return selected_sm100_tensors(p) && aligned_view(&p->dout) && aligned_view(&p->dq) && aligned_view(&p->dk) && aligned_view(&p->dv) &&
           (long long)p->B * p->H * (ceil_div(p->Lq, SB_OWN) + 1ll) <= (1 << 24) &&
           (long long)p->B * p->Hkv * (ceil_div(p->Lkv, SB_OWN) + 1ll) <= (1 << 24);
}

int selected_sm100_backward(const wa_selected_params *p, const int32_t *index, const int32_t *num, const uint32_t *rows, const float *stats,
                            const int32_t *q_order, const int32_t *k_order, int *counters, cudaStream_t stream) {
    using namespace sm100;
    SbParams kp{};
    kp.H = p->H; kp.Hkv = p->Hkv; kp.group = p->H / p->Hkv; kp.Lq = p->Lq; kp.Lkv = p->Lkv;
    kp.Nq = ceil_div(p->Lq, p->block_size); kp.Nkv = ceil_div(p->Lkv, p->block_size);
    kp.list_stride = p->index_stride; kp.row_words = ceil_div(kp.Nq, 32);
    kp.padded = (long long)selected_stats_rows(p, kp.Nq);
    kp.index = index; kp.num = num; kp.rows = rows; kp.stats = stats; kp.q_order = q_order; kp.k_order = k_order;
    kp.scale = (float)pow((double)TILE, -0.5);
    kp.scale_log2 = (float)(pow((double)TILE, -0.5) * 1.4426950408889634);
    kp.work_counter = counters;
    kp.error_flag = kp.work_counter + 2;
    kp.status_mirror = p->status_mirror;
    int rc;
    if (p->block_size == TILE) return (rc = launch_owned<true, TILE>(p, kp, stream)) ? rc : launch_owned<false, TILE>(p, kp, stream);
    return (rc = launch_owned<true, HALF>(p, kp, stream)) ? rc : launch_owned<false, HALF>(p, kp, stream);
}

}  // namespace wa
