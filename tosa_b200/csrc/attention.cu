// Attention over packed prompts on the tensor cores, one pass over the keys.
//
//   out_i = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q_i.k_j),  j over the keys that row i sees
//
// With t_j = scale * log2(e) * q_i.k_j the kernel keeps, per row, a reference m and
// l = sum 2^(t_j - m), o = sum 2^(t_j - m) v_j. m follows the running maximum only when that has
// grown by more than 8: l and o are then multiplied by 2^(m - m'). Between such steps a weight is at
// most 2^8, far inside the range of both types, and since weights and their sum share m the result
// does not depend on it. lse = (m + log2 l) ln 2.
//
// An item is two tiles of 128 rows (two heads of one key head's group, or two row tiles of one head) that
// walk the same blocks of 128 keys. One CTA an SM takes item after item: the grid has a block for each,
// and a running CTA takes over blocks that have not begun, heaviest first within a sequence. 12 warps:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one row a thread: read the scores from tensor memory, write
//                   the weights back to it as f16 / bf16, rescale o there when m moves, and store the
//                   result at the item's end
//   warp 8          issues the MMAs: S = Q K^T (both from shared memory), O += P V (P from tensor memory)
//   warp 9          finds the items and loads by TMA: the Q tiles, then K and V blocks through a ring,
//                   running ahead into the next item
//   warps 10-11     look through the V blocks that some row sees only in part (see guard_block)
// While one tile's softmax runs, the tensor cores work on the other tile. Tensor memory: S of both
// tiles (128 columns each; P takes the first 64 of its S once the scores have been read) and O.
//
// Per tile and block the MMAs take 2 * 128 * 128 * head_dim multiply-adds (1024 cycles at head_dim 128)
// and the 128 * 128 exponentials 1024 cycles of the special-function units. A tile's chain is softmax,
// then O += P V, then the next S, so what counts is the softmax's length beside the other tile's MMAs:
// part of the exponentials is computed as a polynomial on the otherwise idle FMA units, and the
// first half of the weights is handed over while the second half is computed.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "attention.cuh"
#include "ptx.cuh"
#include "quant.cuh"

namespace tb {

constexpr int kRows = 128;      // rows of a tile
constexpr int kKeys = 128;      // keys of a block
constexpr int kThreads = 384;
// Registers: launched with 168 a thread (64,512); the softmax warpgroups take 208, the other one keeps 88.
constexpr int kLaunchRegs = 168;
constexpr int kSoftmaxRegs = 208;
constexpr int kOtherRegs = 88;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "register split above the launch total");
constexpr float kGrowth = 8.f;  // m follows the maximum when it has grown by more than this (powers of two)
constexpr long long kDrainCycles = 2000000000ll;  // bound on a CTA's waits for its own copies and MMAs at its end
constexpr int kGuards = 4;
constexpr int kItems = 2;       // items announced at a time
constexpr int kItemReaders = 11;  // warps that read an item: softmax, MMA, guards
// Of every 8 pairs of exponentials this many are polynomials (see the kernel's head).
constexpr int kPolyPairs = 3;

// DCH: 64-element chunks of head_dim.
template <int DCH>
struct PromptCfg {
    static constexpr int kChunk = kRows * 128;        // one chunk of a tile: 128 rows of 128 bytes, swizzled
    static constexpr int kTile = DCH * kChunk;
    static constexpr int kStages = DCH == 2 ? 4 : 6;  // ring of K and V blocks
    static constexpr int kStaging = 8 * 4096;         // each softmax warp's 32 result rows of 64 elements, swizzled
    static constexpr int kTiles = (2 + kStages) * kTile + kStaging;
};

// A guarded value that is not finite is noted by its key, counted from the item's first guarded block.
constexpr uint32_t kNoKey = 0xFFFFu;

struct Item {
    int valid, q0, k0, lq, lk, sub, kv_head;  // sub: the first tile's number among (row tile, head of the group)
};

struct PromptShared {
    alignas(16) uint4 response;  // of cancel_next_block
    uint64_t q_full[2], q_empty[2], full[8], empty[8], guard[kGuards], s_full[2], p_half[2], p_full[2], o_full[2], drain;
    uint64_t item_full[kItems], item_empty[kItems], guard_done[kItems], next;
    uint32_t tmem;
    int abort;
    Item item[kItems];
    int odd[kItems];                          // some guarded value of the item is not finite
    uint32_t first[kItems][3][kKeys / 2];     // per dimension (16 bits): the first key with NaN, +inf, -inf
};
static_assert(sizeof(PromptShared) + PromptCfg<2>::kTiles <= 232448 && sizeof(PromptShared) + PromptCfg<1>::kTiles <= 232448,
              "shared memory above 227 KB");

struct PromptArgs {
    void* out;
    float* lse;
    const int32_t *cu_q, *cu_k;
    long long o_token, o_head;
    long long total_q, total_k;
    int batch, group, kv_heads, head_dim, causal;
    float scale_log2;
    uint32_t* err;
    long long timeout_cycles;
};

// One tile's place: rows row0 .. row0 + rows - 1 of its sequence, of one head.
struct Tile {
    int row0, rows, head;
    int blocks;     // blocks of keys that some row sees
    int seen_by_all;  // keys that every row sees (the first row's)
};

__device__ __forceinline__ int visible(int causal, int row, int lq, int lk) {
    return causal ? max(0, min(lk, row + lk - lq + 1)) : lk;
}

__device__ __forceinline__ Tile tile_of(const PromptArgs& a, const Item& it, int t) {
    Tile x{0, 0, 0, 0, INT32_MAX};
    const int sub = it.sub + t, rt = sub / a.group;
    x.row0 = rt * kRows;
    x.rows = min(kRows, it.lq - x.row0);
    if (x.rows <= 0) {
        x.rows = 0;
        return x;
    }
    x.head = it.kv_head * a.group + (sub - rt * a.group);
    x.blocks = (visible(a.causal, x.row0 + x.rows - 1, it.lq, it.lk) + kKeys - 1) / kKeys;
    x.seen_by_all = visible(a.causal, x.row0, it.lq, it.lk);
    return x;
}

// The first block of keys that some row of a tile that takes it does not see whole.
__device__ __forceinline__ int first_guarded(const Tile& x, const Tile& y) {
    return min(x.blocks > 0 ? x.seen_by_all / kKeys : INT32_MAX, y.blocks > 0 ? y.seen_by_all / kKeys : INT32_MAX);
}

// A weight of 0 does not take a key out of a product when the value is NaN or infinite. In a block
// that some row sees only in part, V is therefore put in order before the MMA reads it: rows past the
// sequence's end become zero, and values that are not finite become zero with their place noted
// (first[]), to be added by the rows that do see them when they store their result. 64 threads, a few
// hundred cycles that the ring's depth hides. `rel`: the block's first key counted from first_guarded.
template <bool BF16, int DCH>
__device__ void guard_block(PromptShared& sh, int slot, uint8_t* v, int live, int rel, int t) {
    constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u;   // exponent of both halves
    constexpr uint32_t kOne = BF16 ? 0x00800080u : 0x04000400u;   // all ones + 1: a carry into bit 15
    constexpr uint32_t kFrac = BF16 ? 0x7Fu : 0x3FFu;
#pragma unroll 4
    for (int i = t; i < DCH * kKeys * 8; i += 64) {
        const int row = (i >> 3) & (kKeys - 1);
        uint4* p = reinterpret_cast<uint4*>(v) + i;
        if (row >= live) {
            *p = make_uint4(0, 0, 0, 0);
            continue;
        }
        const uint4 x = *p;
        const uint32_t odd = (((x.x & kExp) + kOne) | ((x.y & kExp) + kOne) | ((x.z & kExp) + kOne) | ((x.w & kExp) + kOne)) & 0x80008000u;
        if (odd == 0) continue;
        // swizzled place: 16-byte vector (i & 7) of the row holds vector (i & 7) ^ (row & 7)
        const int d0 = (i >> 10) * 64 + (((i & 7) ^ (row & 7)) << 3);
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = (w[e >> 1] >> ((e & 1) * 16)) & 0xFFFFu;
            if ((h & (kExp & 0xFFFFu)) != (kExp & 0xFFFFu)) continue;
            const int kind = (h & kFrac) ? 0 : ((h >> 15) ? 2 : 1);
            const uint32_t key = min(static_cast<uint32_t>(rel + row), kNoKey - 1), shift = (e & 1) * 16;
            uint32_t* word = &sh.first[slot][kind][(d0 + e) >> 1];
            uint32_t old = *word;
            while (((old >> shift) & 0xFFFFu) > key) {  // ends: the half only gets smaller
                const uint32_t seen = atomicCAS(word, old, (old & ~(0xFFFFu << shift)) | (key << shift));
                if (seen == old) break;
                old = seen;
            }
            w[e >> 1] &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
            sh.odd[slot] = 1;
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct RingPos {
    int s = 0;
    uint32_t ph = 0;
    template <int S>
    __device__ __forceinline__ void step() {
        if (++s == S) {
            s = 0;
            ph ^= 1;
        }
    }
};

// Weights 2^(t - base) of 64 scores as 32 packed pairs, and their sum.
template <bool BF16, int POLY>
__device__ __forceinline__ void weights(const float* x, uint64_t scale, uint64_t neg_base, uint64_t (&sum)[2], uint32_t (&p)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const uint64_t t = fma_pair(pair_of(x[2 * i], x[2 * i + 1]), scale, neg_base);
        float u, w;
        if ((i & 7) >= 8 - POLY) {
            exp2_poly(t, u, w);
        } else {
            split_pair(t, u, w);
            u = exp2_fast(u);
            w = exp2_fast(w);
        }
        sum[i & 1] = add_pair(sum[i & 1], pair_of(u, w));
        p[i] = pack2<BF16>(u, w);
    }
}

template <bool BF16, int DCH>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const PromptArgs a) {
    using Cfg = PromptCfg<DCH>;
    constexpr int S = Cfg::kStages;
    extern __shared__ __align__(1024) uint8_t sq[];  // Q tiles, ring, staging, PromptShared
    uint8_t* ring = sq + 2 * Cfg::kTile;
    uint8_t* staging = ring + S * Cfg::kTile;
    PromptShared& sh = *reinterpret_cast<PromptShared*>(sq + Cfg::kTiles);
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    volatile int* abort_flag = &sh.abort;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_half[i], 4);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
        }
        for (int i = 0; i < S; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < kGuards; ++i) mbar_init(&sh.guard[i], 2);
        for (int i = 0; i < kItems; ++i) {
            mbar_init(&sh.item_full[i], 1);
            mbar_init(&sh.item_empty[i], kItemReaders);
            mbar_init(&sh.guard_done[i], 2);
            sh.odd[i] = 1;  // first[] is cleared before the first use
        }
        mbar_init(&sh.next, 1);
        mbar_init(&sh.drain, 1);
        fence_mbar_init();
        sh.abort = 0;
    }
    if (warp == 8) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    } else if (warp == 9 && lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        tma_prefetch_desc(&tmO);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const long long limit = a.timeout_cycles;
    const long long drain_limit = limit > kDrainCycles ? limit : kDrainCycles;
    // A wait by a whole warp; its lanes agree on whether it gave up.
    auto wait = [&](uint64_t* bar, uint32_t ph) {
        return __all_sync(0xffffffffu, mbar_wait_bounded(bar, ph, abort_flag, limit)) != 0;
    };
    auto gave_up = [&]() {
        if (lane == 0) {
            atomicOr(a.err, DEV_ERR_TIMEOUT);
            *abort_flag = 1;
        }
    };
    // The k-th item, false at the end or when a wait gave up.
    auto read_item = [&](int k, Item& it, bool& ok) {
        ok = wait(&sh.item_full[k % kItems], (k / kItems) & 1);
        if (!ok) return false;
        it = sh.item[k % kItems];
        return it.valid != 0;
    };
    auto done_with_item = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.item_empty[k % kItems]);
    };

    if (warp >= 8) {
        setmaxnreg_dec<kOtherRegs>();
        if (warp == 9) {
            // ---------------------------------------------------------------- items and loads
            grid_dependency_wait();
            RingPos r;
            uint32_t loads = 0, qn[2] = {0, 0};
            bool ok = true;
            int b0 = 0;            // sequences before b0 have `before` items (items come in rising order, as a rule)
            long long before = 0;
            int block = blockIdx.x;
            for (int k = 0;; ++k) {
                // items lie sequence behind sequence, ceil(row tiles * group / 2) for each
                Item it{};
                const long long want = block < 0 ? 0 : block / a.kv_heads;
                if (want < before) before = b0 = 0;
                while (block >= 0 && b0 < a.batch) {
                    const int b = b0 + lane;
                    int items = 0;
                    long long q0 = 0, q1 = 0, k0 = 0, k1 = 0;
                    if (b < a.batch) {
                        q0 = a.cu_q[b];
                        q1 = a.cu_q[b + 1];
                        k0 = a.cu_k[b];
                        k1 = a.cu_k[b + 1];
                        // (sequences out of range are reported by the first block's warp 10)
                        if (!(q0 < 0 || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k))
                            items = static_cast<int>(((q1 - q0 + kRows - 1) / kRows * a.group + 1) >> 1);
                    }
                    int x = items;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int y = __shfl_up_sync(0xffffffffu, x, o);
                        if (lane >= o) x += y;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, before + x > want);
                    if (over) {
                        const int l = __ffs(over) - 1;
                        it.valid = 1;
                        it.q0 = __shfl_sync(0xffffffffu, static_cast<int>(q0), l);
                        it.k0 = __shfl_sync(0xffffffffu, static_cast<int>(k0), l);
                        it.lq = __shfl_sync(0xffffffffu, static_cast<int>(q1), l) - it.q0;
                        it.lk = __shfl_sync(0xffffffffu, static_cast<int>(k1), l) - it.k0;
                        // the last rows, which see the most keys, first
                        it.sub = 2 * static_cast<int>(before + __shfl_sync(0xffffffffu, x, l) - 1 - want);
                        it.kv_head = block - static_cast<int>(want) * a.kv_heads;
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, x, 31);
                    b0 += 32;
                }
                const int slot = k % kItems;
                ok = wait(&sh.item_empty[slot], ((k / kItems) & 1) ^ 1);
                if (!ok) break;
                if (sh.odd[slot]) {  // the slot's last item noted keys: cleared now that its readers are done
                    for (int i = lane; i < 3 * kKeys / 2; i += 32) (&sh.first[slot][0][0])[i] = 0xFFFFFFFFu;
                    __syncwarp();
                    if (lane == 0) sh.odd[slot] = 0;
                }
                if (lane == 0) sh.item[slot] = it;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.item_full[slot]);
                if (!it.valid) break;
                if (lane == 0) {  // the next item's block, while this one loads
                    fence_proxy_async_smem();
                    mbar_arrive_expect_tx(&sh.next, 16);
                    cancel_next_block(&sh.response, &sh.next);
                }
                const Tile tile[2] = {tile_of(a, it, 0), tile_of(a, it, 1)};
                const int blocks = max(tile[0].blocks, tile[1].blocks);
                auto load_block = [&](const CUtensorMap* m, int j) {
                    ok = wait(&sh.empty[r.s], r.ph ^ 1);
                    if (!ok) return;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.full[r.s], Cfg::kTile);
#pragma unroll
                        for (int c = 0; c < DCH; ++c)
                            tma_load_3d(ring + r.s * Cfg::kTile + c * Cfg::kChunk, m, &sh.full[r.s], 64 * c, it.kv_head, it.k0 + j * kKeys);
                    }
                    __syncwarp();
                    ++loads;
                    r.step<S>();
                };
                for (int t = 0; t < 2 && ok; ++t) {
                    if (tile[t].blocks == 0) continue;
                    ok = wait(&sh.q_empty[t], (qn[t] & 1) ^ 1);
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.q_full[t], Cfg::kTile);
#pragma unroll
                        for (int c = 0; c < DCH; ++c)
                            tma_load_3d(sq + t * Cfg::kTile + c * Cfg::kChunk, &tmQ, &sh.q_full[t], 64 * c, tile[t].head, it.q0 + tile[t].row0);
                    }
                    __syncwarp();
                    ++qn[t];
                    if (t == 0) load_block(&tmK, 0);
                }
                if (ok && tile[0].blocks == 0 && blocks > 0) load_block(&tmK, 0);
                for (int j = 0; j < blocks && ok; ++j) {
                    load_block(&tmV, j);
                    if (ok && j + 1 < blocks) load_block(&tmK, j + 1);
                }
                // the answer is read even when a wait gave up: it must not arrive after the CTA's end
                const bool got = __all_sync(0xffffffffu, mbar_wait_bounded(&sh.next, k & 1, nullptr, drain_limit));
                if (!ok || !got) {
                    ok = false;
                    break;
                }
                block = cancelled_block(&sh.response);
                __syncwarp();
            }
            if (!ok) gave_up();
            // every issued load lands before the CTA may exit
            for (int t = 0; t < 2; ++t)
                if (qn[t]) mbar_wait_bounded(&sh.q_full[t], (qn[t] - 1) & 1, nullptr, drain_limit);
            for (uint32_t i = loads > S ? loads - S : 0; i < loads; ++i)
                mbar_wait_bounded(&sh.full[i % S], (i / S) & 1, nullptr, drain_limit);
        } else if (warp == 8) {
            // ---------------------------------------------------------------- MMAs
            // The whole warp walks along and one lane issues: descriptors then stay in uniform
            // registers, and a run of MMAs is issued faster than the tensor cores take them.
            const uint32_t idesc_s = idesc_f16(kRows, kKeys, BF16, false);
            const uint32_t idesc_o = idesc_f16(kRows, a.head_dim, BF16, true);
            const uint64_t dq = smem_desc(smem_u32(sq), 16, 1024, 2);             // K-major: Q, K
            const uint64_t dk = smem_desc(smem_u32(ring), 16, 1024, 2);
            const uint64_t dv = smem_desc(smem_u32(ring), Cfg::kChunk, 1024, 2);  // dimension-major: V
            const int ksteps = a.head_dim / 16;
            const bool leader = elect_one();
            auto scores = [&](int t, int stage) {
                const uint64_t qa = dq + ((t * Cfg::kTile) >> 4), kb = dk + ((stage * Cfg::kTile) >> 4);
                if (leader) {
#pragma unroll
                    for (int k = 0; k < 4 * DCH; ++k) {
                        const uint32_t o = ((k >> 2) * Cfg::kChunk + (k & 3) * 32) >> 4;
                        if (k < ksteps) tc_mma<1>(tmem + t * 128, qa + o, kb + o, idesc_s, k > 0);
                    }
                    tc_commit(&sh.s_full[t]);
                }
                __syncwarp();
            };
            auto product = [&](int t, int stage, int half, bool first) {
                const uint64_t vb = dv + ((stage * Cfg::kTile) >> 4);
                if (leader) {
#pragma unroll
                    for (int i = 0; i < kKeys / 32; ++i) {
                        const int k = half * (kKeys / 32) + i;
                        tc_mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, vb + ((k * 2048) >> 4), idesc_o, !first || k > 0);
                    }
                }
                __syncwarp();
            };
            auto commit = [&](uint64_t* bar) {
                if (leader) tc_commit(bar);
                __syncwarp();
            };
            RingPos r;                     // the K block at hand, then its V block, ...
            uint32_t n[2] = {0, 0};        // blocks of each tile so far
            uint32_t qn[2] = {0, 0}, vn = 0;
            bool ok = true;
            Item it;
            for (int k = 0; read_item(k, it, ok); ++k) {
                done_with_item(k);
                const Tile tile[2] = {tile_of(a, it, 0), tile_of(a, it, 1)};
                const int blocks = max(tile[0].blocks, tile[1].blocks);
                if (blocks == 0) continue;
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (ok && tile[t].blocks) {
                        ok = wait(&sh.q_full[t], qn[t]++ & 1) && wait(&sh.full[r.s], r.ph);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, r.s);
                        if (tile[t].blocks == 1) commit(&sh.q_empty[t]);
                    }
                if (!ok) break;
                commit(&sh.empty[r.s]);
                r.step<S>();
                for (int j = 0; j < blocks && ok; ++j, ++vn) {
                    const RingPos v = r;
                    r.step<S>();
                    ok = wait(&sh.full[v.s], v.ph) && wait(&sh.guard[vn % kGuards], (vn / kGuards) & 1);
                    if (!ok) break;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j < tile[t].blocks) {
                            ok = ok && wait(&sh.p_half[t], n[t] & 1);
                            if (!ok) break;
                            tc_fence_after();
                            //TR(40+t)
                            product(t, v.s, 0, j == 0);
                            ok = wait(&sh.p_full[t], n[t]++ & 1);
                            if (!ok) break;
                            tc_fence_after();
                            product(t, v.s, 1, false);
                            //TR(42+t)
                            if (j + 1 == tile[t].blocks) commit(&sh.o_full[t]);
                        }
                        if (t == 1) commit(&sh.empty[v.s]);
                        if (j + 1 < tile[t].blocks) {
                            ok = wait(&sh.full[r.s], r.ph);
                            if (!ok) break;
                            tc_fence_after();
                            scores(t, r.s);
                            //TR(44+t)
                            if (j + 2 == tile[t].blocks) commit(&sh.q_empty[t]);
                        }
                    }
                    if (!ok) break;
                    if (j + 1 < blocks) {
                        commit(&sh.empty[r.s]);
                        r.step<S>();
                    }
                }
                if (!ok) break;
            }
            if (!ok) gave_up();
            commit(&sh.drain);
            mbar_wait_bounded(&sh.drain, 0, nullptr, drain_limit);
            __syncwarp();
        } else {
            // ---------------------------------------------------------------- V blocks seen in part
            grid_dependency_wait();
            if (blockIdx.x == 0 && warp == 10)
                for (int b = lane; b < a.batch; b += 32) {
                    const long long q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
                    if (q0 < 0 || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) atomicOr(a.err, DEV_ERR_INDEX);
                }
            RingPos r;
            uint32_t vn = 0;
            bool ok = true;
            Item it;
            for (int k = 0; read_item(k, it, ok); ++k) {
                const Tile tile[2] = {tile_of(a, it, 0), tile_of(a, it, 1)};
                const int blocks = max(tile[0].blocks, tile[1].blocks);
                const int from = first_guarded(tile[0], tile[1]);
                for (int j = 0; j < blocks; ++j, ++vn) {
                    r.step<S>();  // past the K block
                    ok = wait(&sh.full[r.s], r.ph);
                    if (!ok) break;
                    // a tile that does not reach this block has no say in it
                    const int seen = min(j < tile[0].blocks ? tile[0].seen_by_all : INT32_MAX,
                                         j < tile[1].blocks ? tile[1].seen_by_all : INT32_MAX);
                    if (seen < (j + 1) * kKeys) {
                        guard_block<BF16, DCH>(sh, k % kItems, ring + r.s * Cfg::kTile, it.lk - j * kKeys, (j - from) * kKeys, threadIdx.x - 320);
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.guard[vn % kGuards]);
                    r.step<S>();
                }
                if (!ok) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.guard_done[k % kItems]);
                done_with_item(k);
            }
            if (!ok) gave_up();
        }
    } else {
        // -------------------------------------------------------------------- softmax
        setmaxnreg_inc<kSoftmaxRegs>();
        grid_dependency_wait();
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t ts = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * 128;
        const uint32_t to = ts + 256;  // O
        const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2);
        uint32_t n = 0, outs = 0;  // blocks and results so far
        bool ok = true;
        Item it;
        for (int k = 0; read_item(k, it, ok); ++k) {
            const Tile my = tile_of(a, it, t);
            const int row = my.row0 + r;
            const int sees = r < my.rows ? visible(a.causal, row, it.lq, it.lk) : it.lk;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < my.blocks; ++j, ++n) {
                ok = wait(&sh.s_full[t], n & 1);
                if (!ok) break;
                //TR(warp)
                tc_fence_after();
                uint32_t s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                tmem_ld_wait();
                float x[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) {
                    asm volatile("" : "+r"(s[i]));
                    x[i] = __uint_as_float(s[i]);
                }
                const bool part = my.seen_by_all < (j + 1) * kKeys;  // some row does not see the whole block
                if (part) {
                    const int seen = sees - j * kKeys;
#pragma unroll
                    for (int i = 0; i < 128; ++i) x[i] = i < seen ? x[i] : -INFINITY;
                }
                //TR(8+warp)
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = x[32 * c];
#pragma unroll
                    for (int i = 1; i < 31; i += 2) top[c] = max3_nan(top[c], x[32 * c + i], x[32 * c + i + 1]);
                    top[c] = max_nan(top[c], x[32 * c + 31]);
                }
                // a NaN among the scores becomes the row's reference and with it the whole row
                const float m1 = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])) * a.scale_log2;
                const bool grow = !(m1 <= m + kGrowth);
                if (__any_sync(0xffffffffu, grow)) {
                    const float mm = grow ? m1 : m;
                    if (j > 0) {
                        const float f = grow ? exp2_fast(m - mm) : 1.f;
                        l *= f;
                        for (int c = 0; c < a.head_dim; c += 16) {
                            uint32_t o[16];
                            tmem_ld_32x32b_x16(to + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                asm volatile("" : "+r"(o[i]));
                                o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            }
                            tmem_st_32x32b_x16(to + c, o);
                        }
                    }
                    m = mm;
                }
                const float base = m == -INFINITY ? 0.f : m;
                //TR(16+warp)
                const uint64_t neg = pair_of(-base, -base);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t p[32];
                    // keys that are not seen get a weight of exactly 0 from the special-function unit
                    if (part) weights<BF16, 0>(x + 64 * c, scale2, neg, sum, p);
                    else weights<BF16, kPolyPairs>(x + 64 * c, scale2, neg, sum, p);
                    tmem_st_32x32b_x32(ts + 32 * c, p);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(c == 0 ? &sh.p_half[t] : &sh.p_full[t]);
                }
                //TR(24+warp)
                float s0, s1;
                split_pair(add_pair(sum[0], sum[1]), s0, s1);
                l += s0 + s1;
                //TR(32+warp)
            }
            if (!ok) break;
            ok = wait(&sh.guard_done[k % kItems], (k / kItems) & 1);
            if (ok && my.blocks > 0) ok = wait(&sh.o_full[t], outs++ & 1);
            if (!ok) break;
            tc_fence_after();
            const bool live = r < my.rows, any = sees > 0;
            // (a reference that is not finite: a score of NaN or +inf, or every score -inf)
            const float inv = any ? (isfinite(m) ? __fdividef(1.f, l) : NAN) : 0.f;
            const int odd = sh.odd[k % kItems];
            const uint16_t* first = reinterpret_cast<const uint16_t*>(&sh.first[k % kItems][0][0]);
            const int rel = odd ? sees - first_guarded(tile_of(a, it, 0), tile_of(a, it, 1)) * kKeys : 0;
            // Each thread has a row, but the result leaves by TMA, 64 elements of the warp's 32 rows at a
            // time through its staging buffer (stores straight from the row's thread touch 32 lines an
            // instruction and took 6,300 cycles an item). A warp whose rows end inside the 32 stores its
            // rows itself, so that nothing past the sequence's end is written.
            const int warp_row = r & ~31;
            uint4* st = reinterpret_cast<uint4*>(staging + warp * 4096);
            const bool whole = warp_row + 32 <= my.rows;
#pragma unroll 1
            for (int c0 = 0; c0 < a.head_dim; c0 += 64) {
                uint32_t o[64];
                if (my.blocks > 0) {
                    tmem_ld_32x32b_x32(to + c0, *reinterpret_cast<uint32_t(*)[32]>(o));
                    tmem_ld_32x32b_x32(to + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 64; ++i) asm volatile("" : "+r"(o[i]));
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] = 0;
                }
                if (odd) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        float y = __uint_as_float(o[i]);
                        if (first[c0 + i] < rel) y = NAN;
                        if (first[kKeys + c0 + i] < rel) y += INFINITY;
                        if (first[2 * kKeys + c0 + i] < rel) y -= INFINITY;
                        o[i] = __float_as_uint(y);
                    }
                }
                uint32_t h[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) h[i] = pack2<BF16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                if (lane == 0) bulk_wait_read0();  // the buffer's last store has left
                __syncwarp();
#pragma unroll
                for (int v = 0; v < 8; ++v) st[lane * 8 + (v ^ (lane & 7))] = make_uint4(h[4 * v], h[4 * v + 1], h[4 * v + 2], h[4 * v + 3]);
                if (whole) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_3d(&tmO, st, c0, my.head, it.q0 + my.row0 + warp_row);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<long long>(it.q0 + my.row0 + warp_row) * a.o_token + my.head * a.o_head + c0;
                    const int v = lane & 7;
                    for (int rr = lane >> 3; warp_row + rr < my.rows && rr < 32; rr += 4)
                        if (c0 + 8 * v < a.head_dim) *reinterpret_cast<uint4*>(out + rr * a.o_token + 8 * v) = st[rr * 8 + (v ^ (rr & 7))];
                }
            }
            if (a.lse != nullptr && live)
                a.lse[static_cast<long long>(my.head) * a.total_q + it.q0 + row] =
                    any && m != -INFINITY ? (m + __log2f(l)) * kLn2 : -INFINITY;
            tc_fence_before();
            done_with_item(k);
        }
        if (!ok) gave_up();
        if (lane == 0) bulk_wait0();  // the warp's TMA stores are done before the CTA exits
        __syncwarp();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

tb_status attention_check(const char* op, int dtype, int q_heads, int kv_heads, int head_dim, float scale) {
    if (dtype != TB_DT_BF16 && dtype != TB_DT_FP16)
        return fail(TB_ERR_DTYPE_MISMATCH, "%s: unsupported type %d (FP16 or BF16)", op, dtype);
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads)
        return fail(TB_ERR_SHAPE_MISMATCH, "%s: %d query heads are no multiple of %d key heads", op, q_heads, kv_heads);
    if (head_dim < 16 || head_dim > 128 || head_dim % 16)
        return fail(TB_ERR_NOT_ACCELERATED, "%s: head_dim %d is not a multiple of 16 up to 128", op, head_dim);
    if (!(scale > 0.f) || !std::isfinite(scale) || !std::isfinite(scale * kLog2e))
        return fail(TB_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", op);
    return TB_OK;
}

// [tokens][heads][head_dim] as {head_dim, heads, tokens}, boxes of some tokens by 64 elements of one head.
static tb_status tile_map(CUtensorMap* m, const tb_attention_desc* d, const void* p, int64_t heads, int64_t tokens,
                          int64_t token_stride, int64_t head_stride, int box_tokens = kRows) {
    // the stride of a dimension of one element says nothing; the map wants a valid one
    const uint64_t head = heads > 1 ? head_stride : d->head_dim, token = tokens > 1 ? token_stride : d->head_dim;
    const uint64_t dims[3] = {static_cast<uint64_t>(d->head_dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
    const uint64_t strides[2] = {head * 2, token * 2};
    const uint32_t box[3] = {64, 1, static_cast<uint32_t>(box_tokens)};
    return encode_tiled(m, d->dtype == TB_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p,
                        dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool BF16, int DCH>
static tb_status launch_prompt(tb_context* ctx, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                               const CUtensorMap& o, const PromptArgs& a, long long grid, cudaStream_t st) {
    auto* kernel = prompt_kernel<BF16, DCH>;
    constexpr int kSmem = PromptCfg<DCH>::kTiles + static_cast<int>(sizeof(PromptShared));
    static bool ready = false;  // the attribute is per function and process-wide
    if (!ready) {
        // the warpgroups re-split the registers of the launch (setmaxnreg), which needs all of them
        cudaFuncAttributes fa;
        TB_CUDA(cudaFuncGetAttributes(&fa, kernel));
        if (fa.numRegs < kLaunchRegs)
            return fail(TB_ERR_CUDA, "attention built with %d registers a thread; its register split needs %d", fa.numRegs, kLaunchRegs);
        TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        ready = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA(cudaLaunchKernelEx(&cfg, kernel, q, k, v, o, a));
    ctx->launches++;
    return TB_OK;
}

}  // namespace tb

using namespace tb;

extern "C" {

TB_API tb_status tb_attention(tb_context* ctx, const tb_attention_desc* d, const void* q, const void* k, const void* v,
                              const int32_t* cu_q, const int32_t* cu_k, void* out, float* lse, void* stream) {
    if (!ctx || !d) return fail(TB_ERR_INVALID_ARGUMENT, "attention: null argument");
    TB_TRY(attention_check("attention", d->dtype, d->q_heads, d->kv_heads, d->head_dim, d->scale));
    if (d->batch < 0 || d->total_q < 0 || d->total_k < 0)
        return fail(TB_ERR_SHAPE_MISMATCH, "attention: negative dimension");
    if (d->total_q > (1ll << 30) || d->total_k > (1ll << 30) || d->batch > (1 << 20) || d->q_heads > 4096)
        return fail(TB_ERR_NOT_ACCELERATED, "attention: more than 2^30 rows, 2^20 sequences or 4096 heads");
    if (d->batch == 0 || d->total_q == 0) return TB_OK;
    if (!q || !cu_q || !cu_k || !out || (d->total_k > 0 && (!k || !v)))
        return fail(TB_ERR_INVALID_ARGUMENT, "attention: null pointer");
    long long strides = 0;
    for (int64_t s : {d->q_token_stride, d->q_head_stride, d->k_token_stride, d->k_head_stride, d->v_token_stride,
                      d->v_head_stride, d->out_token_stride, d->out_head_stride}) {
        if (s < 0) return fail(TB_ERR_SHAPE_MISMATCH, "attention: negative stride");
        strides |= s;
    }
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || (strides & 7))
        return fail(TB_ERR_INVALID_ARGUMENT, "attention: tensors must be 16-byte aligned with strides that are multiples of 8");
    // without keys nothing is loaded; the maps are made of q's first row
    const bool keys = d->total_k > 0;
    CUtensorMap mq, mk, mv, mo;
    TB_TRY(tile_map(&mq, d, q, d->q_heads, d->total_q, d->q_token_stride, d->q_head_stride));
    TB_TRY(tile_map(&mk, d, keys ? k : q, keys ? d->kv_heads : 1, keys ? d->total_k : 1, d->k_token_stride, d->k_head_stride));
    TB_TRY(tile_map(&mv, d, keys ? v : q, keys ? d->kv_heads : 1, keys ? d->total_k : 1, d->v_token_stride, d->v_head_stride));
    TB_TRY(tile_map(&mo, d, out, d->q_heads, d->total_q, d->out_token_stride, d->out_head_stride, 32));
    const int group = d->q_heads / d->kv_heads;
    PromptArgs a{out, lse, cu_q, cu_k, d->out_token_stride, d->out_head_stride, d->total_q, d->total_k, d->batch, group,
                 d->kv_heads, d->head_dim, d->causal, d->scale * kLog2e, ctx->dev_err, ctx->timeout_cycles};
    // most items that lengths summing to total_q can have: the lengths themselves are on the device
    const long long seqs = d->batch < d->total_q ? d->batch : d->total_q;
    const long long grid = ((d->total_q / kRows + seqs) * group / 2 + seqs) * d->kv_heads;
    if (grid > INT32_MAX) return fail(TB_ERR_NOT_ACCELERATED, "attention: more than 2^31 tiles");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = d->head_dim > 64;
    if (d->dtype == TB_DT_BF16)
        return wide ? launch_prompt<true, 2>(ctx, mq, mk, mv, mo, a, grid, st) : launch_prompt<true, 1>(ctx, mq, mk, mv, mo, a, grid, st);
    return wide ? launch_prompt<false, 2>(ctx, mq, mk, mv, mo, a, grid, st) : launch_prompt<false, 1>(ctx, mq, mk, mv, mo, a, grid, st);
}

}  // extern "C"
