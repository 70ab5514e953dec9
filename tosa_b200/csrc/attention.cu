// Attention over packed prompts on the tensor cores, one pass over the keys.
//
//   out_i = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q_i.k_j),  j over the keys that row i sees
//
// With t_j = scale * log2(e) * q_i.k_j the kernel keeps, per row, a reference m and
// l = sum 2^(t_j - m), o = sum 2^(t_j - m) v_j. m is the maximum of the first 32 keys (of the first
// block, where the row does not see all of it) and stays while the weights it gives are small enough: a
// block's maximum is not looked for, the sums of its weights (which are needed anyway) tell when it has run
// away, and then the block is done again with its maximum and l and o are multiplied by 2^(m - m'). Weights stay below 2^13, far inside the range of both types, and
// since weights and their sum share m the result does not depend on it. lse = (m + log2 l) ln 2.
//
// A tile is 128 rows: 128 tokens of one head, or where the group of a key head is a power of two up to 32,
// 128 / group tokens of all its heads (row = token * group + head), so that short sequences fill their
// tiles (one token of 8 heads takes 8 rows of one tile instead of one row of 8). An item is two tiles of
// one key head that walk the same blocks of 128 keys. One CTA an SM takes item after item: the grid has a
// block for each, and a running CTA takes over blocks that have not begun, sequences with many keys first
// and the heaviest first within a sequence. 16 warps:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one row a thread: read the scores from tensor memory, write
//                   the weights back to it as f16 / bf16, and rescale o there when m moves
//   warp 8          issues the MMAs: S = Q K^T (both from shared memory), O += P V (P from tensor memory)
//   warp 9          finds the items and loads by TMA: the Q tiles, then K and V blocks through a ring,
//                   running ahead into the next item
//   warps 10-11     look through the V blocks that some row sees only in part (see guard_block)
//   warps 12-15     divide o by l and store it, while the softmax goes on with the next item
// While one tile's softmax runs, the tensor cores work on the other tile. Tensor memory: S of both
// tiles (128 columns each; P takes the first 64 of its S once the scores have been read) and O.
//
// Per tile and block the MMAs take 2 * 128 * 128 * head_dim multiply-adds (1024 cycles at head_dim 128)
// and the 128 * 128 exponentials 1024 cycles of the special-function units. A tile's chain is softmax,
// then O += P V, then the next S, so what counts is the softmax's length beside the other tile's MMAs:
// scores are handled in pairs where the instruction set allows, no maximum is formed (see above), and
// the first half of the weights is handed over while the second half is computed. (Computing 3 of 8
// exponentials as polynomials on the FMA units, which are idle, made 8192 causal rows 458 us instead of
// 456 in short runs and 524 instead of 518 in sustained ones: the softmax is bound by the instructions
// that one warp can issue, and in sustained runs by power.)
//
// Measured at head_dim 128, bf16: 8192 causal rows of 32 heads in 476 to 490 us by the machine, 1122 to 1155
// TFLOP/s, in sustained runs at the power cap (1.46 GHz), 410 to 421 us, 1306 to 1341 TFLOP/s, in short ones;
// tensor pipe 68 % and special-function units 67 % of the active cycles. A block of both tiles takes some 2850 cycles, 2048 of them MMAs.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "attention.cuh"
#include "ptx.cuh"
#include "quant.cuh"

namespace tb {

constexpr int kRowsLog = 7;
constexpr int kRows = 1 << kRowsLog;  // rows of a tile
constexpr int kKeys = 128;      // keys of a block
constexpr int kThreads = 512;
// Registers: launched with 128 a thread (65,536); the two softmax warpgroups take 192, the others keep 64.
constexpr int kLaunchRegs = 128;
constexpr int kSoftmaxRegs = 192;
constexpr int kOtherRegs = 64;
static_assert(256 * kSoftmaxRegs + 256 * kOtherRegs <= kThreads * kLaunchRegs, "register split above the launch total");
constexpr float kGrowth = 8.f;      // where the maximum is known, m follows it when it has grown by 2^8
constexpr float kMostSum = 8192.f;  // 64 weights with a smaller sum are all below 2^13
constexpr long long kDrainCycles = 2000000000ll;  // bound on a CTA's waits for its own copies and MMAs at its end
constexpr int kGuards = 4;
constexpr int kItems = 2;       // items announced at a time
constexpr int kItemReaders = 15;  // warps that read an item: softmax, MMA, guards, results

// DCH: 64-element chunks of head_dim.
template <int DCH>
struct PromptCfg {
    static constexpr int kChunk = kRows * 128;        // one chunk of a tile: 128 rows of 128 bytes, swizzled
    static constexpr int kTile = DCH * kChunk;
    // Ring of K and V blocks; even, so that V blocks always use the same stages: the guards wait for V blocks
    // only, and a wait on a stage whose K block they had not waited for could take the phase before it for
    // the one it means (copies may land out of order; a ring of 3 timed out).
    static constexpr int kStages = DCH == 2 ? 4 : 6;
    static_assert(kStages % 2 == 0, "V blocks must keep to their stages");
    static constexpr int kStaging = 4 * 4096;         // each result warp's 32 rows of 64 elements, swizzled
    static constexpr int kTiles = (2 + kStages) * kTile + kStaging;
};

// A guarded value that is not finite is noted by its key, counted from the item's first guarded block.
constexpr uint32_t kNoKey = 0xFFFFu;

// One tile's place: its rows are the tokens from token0 on, each of the packed heads from `head` on.
struct Tile {
    int token0, rows, head;
    int blocks;       // blocks of keys that some row sees
    int seen_by_all;  // keys that every row sees (the first row's)
};

struct Item {
    int valid, q0, k0, lq, lk, kv_head;
    int blocks;         // the larger of the tiles' blocks
    int first_guarded;  // the first block of keys that some row of a tile that takes it does not see whole
    Tile tile[2];
};

struct PromptShared {
    alignas(16) uint4 response;  // of cancel_next_block
    uint64_t q_full[2], q_empty[2], full[8], empty[8], guard[kGuards], s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2], ml_full[2], half_done[2], drain;
    uint64_t item_full[kItems], item_empty[kItems], guard_done[kItems], next;
    uint32_t tmem;
    int abort;
    Item item[kItems];
    int odd[kItems];                          // some guarded value of the item is not finite
    uint32_t first[kItems][3][kKeys / 2];     // per dimension (16 bits): the first key with NaN, +inf, -inf
    float2 ml[2][kRows];                      // m and l of each row
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
    int pack_log;             // log2 of the heads that share a tile
    float scale_log2;
    unsigned early_next;  // grids up to this size let the next kernel start early
    uint32_t* err;
    long long timeout_cycles;
};

__device__ __forceinline__ int visible(int causal, int row, int lq, int lk) {
    return causal ? max(0, min(lk, row + lk - lq + 1)) : lk;
}

// Tiles of a key head's group for lq tokens, and tile `sub` of them in the order (token, head).
__device__ __forceinline__ int tiles_of(const PromptArgs& a, int lq) {
    const int tokens_log = kRowsLog - a.pack_log;
    return ((lq + (1 << tokens_log) - 1) >> tokens_log) * (a.group >> a.pack_log);
}
__device__ __forceinline__ Tile tile_of(const PromptArgs& a, int sub, int kv_head, int lq, int lk) {
    Tile x{0, 0, 0, 0, INT32_MAX};
    const int heads = a.group >> a.pack_log;  // 1 where all of the group is packed
    const int st = heads == 1 ? sub : sub / heads;
    x.token0 = st << (kRowsLog - a.pack_log);
    const int tokens = min(kRows >> a.pack_log, lq - x.token0);
    if (tokens <= 0) return x;
    x.rows = tokens << a.pack_log;
    x.head = kv_head * a.group + ((sub - st * heads) << a.pack_log);
    x.blocks = (visible(a.causal, x.token0 + tokens - 1, lq, lk) + kKeys - 1) / kKeys;
    x.seen_by_all = visible(a.causal, x.token0, lq, lk);
    return x;
}

// A weight of 0 does not take a key out of a product when the value is NaN or infinite. In a block
// that some row sees only in part, V is therefore put in order before the MMA reads it: rows past the
// sequence's end become zero, and values that are not finite become zero with their place noted
// (first[]), to be added by the rows that do see them when they are stored. 64 threads, some 400 cycles
// that the ring's depth hides: x * 0 + acc in the type's own arithmetic is NaN from the first value on
// that is not finite, so a block without one costs an instruction for two values. `rel`: the block's
// first key counted from first_guarded.
template <bool BF16>
__device__ __forceinline__ uint32_t sticky(uint32_t x, uint32_t acc) {
    uint32_t r;
    if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
    return r;
}

template <bool BF16, int DCH>
__device__ void note_odd(PromptShared& sh, int slot, uint8_t* v, int rel, int t) {
    constexpr uint32_t kExp = BF16 ? 0x7F80u : 0x7C00u, kFrac = BF16 ? 0x7Fu : 0x3FFu;
    for (int i = t; i < DCH * kKeys * 8; i += 64) {
        const int row = (i >> 3) & (kKeys - 1);
        uint4* p = reinterpret_cast<uint4*>(v) + i;
        const uint4 x = *p;
        // swizzled place: 16-byte vector (i & 7) of the row holds vector (i & 7) ^ (row & 7)
        const int d0 = (i >> 10) * 64 + (((i & 7) ^ (row & 7)) << 3);
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t shift = (e & 1) * 16, h = (w[e >> 1] >> shift) & 0xFFFFu;
            if ((h & kExp) != kExp) continue;
            const int kind = (h & kFrac) ? 0 : ((h >> 15) ? 2 : 1);
            const uint32_t key = min(static_cast<uint32_t>(rel + row), kNoKey - 1);
            uint32_t* word = &sh.first[slot][kind][(d0 + e) >> 1];
            uint32_t old = *word;
            while (((old >> shift) & 0xFFFFu) > key) {  // ends: the half only gets smaller
                const uint32_t seen = atomicCAS(word, old, (old & ~(0xFFFFu << shift)) | (key << shift));
                if (seen == old) break;
                old = seen;
            }
            w[e >> 1] &= ~(0xFFFFu << shift);
            sh.odd[slot] = 1;
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <bool BF16, int DCH>
__device__ __forceinline__ void guard_block(PromptShared& sh, int slot, uint8_t* v, int live, int rel, int t) {
    uint4* p = reinterpret_cast<uint4*>(v);
    if (live < kKeys) {  // rows past the sequence's end
        for (int i = t; i < DCH * kKeys * 8; i += 64)
            if (((i >> 3) & (kKeys - 1)) >= live) p[i] = make_uint4(0, 0, 0, 0);
    }
    uint32_t acc[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int i = t; i < DCH * kKeys * 8; i += 64) {
        const uint4 x = p[i];
        acc[0] = sticky<BF16>(x.x, acc[0]);
        acc[1] = sticky<BF16>(x.y, acc[1]);
        acc[2] = sticky<BF16>(x.z, acc[2]);
        acc[3] = sticky<BF16>(x.w, acc[3]);
    }
    // a sum of zeros is zero of either sign; anything else is NaN
    if (__any_sync(0xffffffffu, ((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7FFF7FFFu) != 0)) note_odd<BF16, DCH>(sh, slot, v, rel, t);
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

// Weights 2^(t - base) of 2 N scores as N packed pairs; returns their sum.
template <bool BF16, int N>
__device__ __forceinline__ float weights(const float* x, uint64_t scale, float base, uint32_t (&p)[N]) {
    const uint64_t neg = pair_of(-base, -base);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float u, w;
        split_pair(fma_pair(pair_of(x[2 * i], x[2 * i + 1]), scale, neg), u, w);
        u = exp2_fast(u);
        w = exp2_fast(w);
        sum[i & 1] = add_pair(sum[i & 1], pair_of(u, w));
        p[i] = pack2<BF16>(u, w);
    }
    float s0, s1;
    split_pair(add_pair(sum[0], sum[1]), s0, s1);
    return s0 + s1;
}

__device__ __forceinline__ float top32(const float* x) {
    float a = max3_nan(x[0], x[1], x[2]), b = max3_nan(x[3], x[4], x[5]);
#pragma unroll
    for (int i = 6; i < 30; i += 4) {
        a = max3_nan(a, x[i], x[i + 1]);
        b = max3_nan(b, x[i + 2], x[i + 3]);
    }
    return max3_nan(max_nan(a, b), x[30], x[31]);
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
            mbar_init(&sh.o_empty[i], 4);
            mbar_init(&sh.ml_full[i], 4);
            mbar_init(&sh.half_done[i], 1);
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
    // The next kernel may be placed on the SMs that are free; it waits for this one before it reads anything.
    if (gridDim.x <= a.early_next && threadIdx.x == 0) grid_launch_dependents();
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
    auto next_item = [&](int k, bool& ok) {
        ok = wait(&sh.item_full[k % kItems], (k / kItems) & 1);
        return ok && sh.item[k % kItems].valid != 0;
    };
    auto done_with_item = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.item_empty[k % kItems]);
    };

    if (warp >= 12) {
        // -------------------------------------------------------------------- results
        setmaxnreg_dec<kOtherRegs>();
        grid_dependency_wait();
        const int w = warp - 12, r = 32 * w + lane;
        // Each thread has a row, but the result leaves by TMA, 64 elements of the warp's 32 rows at a
        // time through its staging buffer (stores straight from the row's thread touch 32 lines an
        // instruction and took 6,300 cycles an item). A warp whose rows end inside the 32 stores its
        // rows itself, so that nothing past the sequence's end is written.
        uint4* st = reinterpret_cast<uint4*>(staging + w * 4096);
        uint32_t outs[2] = {0, 0}, prods[2] = {0, 0};
        bool ok = true;
        for (int k = 0; next_item(k, ok); ++k) {
            const Item& it = sh.item[k % kItems];
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                const Tile my = it.tile[t];
                if (my.rows == 0) continue;
                const int sees = visible(a.causal, my.token0 + (min(r, my.rows - 1) >> a.pack_log), it.lq, it.lk);
                const uint32_t to = tmem + (static_cast<uint32_t>(w * 32) << 16) + 256 + t * 128;
                ok = wait(&sh.ml_full[t], outs[t]++ & 1);
                if (ok && my.blocks > 0) ok = wait(&sh.guard_done[k % kItems], (k / kItems) & 1) && wait(&sh.o_full[t], prods[t]++ & 1);
                if (!ok) break;
                tc_fence_after();
                const float2 ml = sh.ml[t][r];
                const float m = ml.x, l = ml.y;
                const bool any = sees > 0;
                // (a reference that is not finite: a score of NaN or +inf, or every score -inf)
                const float inv = any ? (isfinite(m) ? __fdividef(1.f, l) : NAN) : 0.f;
                const int odd = sh.odd[k % kItems];
                const uint16_t* first = reinterpret_cast<const uint16_t*>(&sh.first[k % kItems][0][0]);
                const int rel = odd ? sees - it.first_guarded * kKeys : 0;
                const bool whole = 32 * w + 32 <= my.rows;
                const int token = it.q0 + my.token0 + ((32 * w) >> a.pack_log);  // the warp's first (pack <= 32)
#pragma unroll 1
                for (int c0 = 0; c0 < a.head_dim; c0 += 64) {
                    if (lane == 0) bulk_wait_read0();  // the buffer's last store has left
                    __syncwarp();
#pragma unroll 1
                    for (int c = 0; c < 64; c += 32) {
                        uint32_t o[32];
                        if (my.blocks > 0) {
                            tmem_ld_32x32b_x32(to + c0 + c, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(o[i]));
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0;
                        }
                        if (odd) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                float y = __uint_as_float(o[i]);
                                const int d = c0 + c + i;
                                if (first[d] < rel) y = NAN;
                                if (first[kKeys + d] < rel) y += INFINITY;
                                if (first[2 * kKeys + d] < rel) y -= INFINITY;
                                o[i] = __float_as_uint(y);
                            }
                        }
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            uint32_t h[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                h[i] = pack2<BF16>(__uint_as_float(o[8 * v + 2 * i]) * inv, __uint_as_float(o[8 * v + 2 * i + 1]) * inv);
                            st[lane * 8 + ((c / 8 + v) ^ (lane & 7))] = make_uint4(h[0], h[1], h[2], h[3]);
                        }
                    }
                    if (c0 + 64 >= a.head_dim) {  // O, m and l have been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.o_empty[t]);
                    }
                    if (whole) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_3d(&tmO, st, c0, my.head, token);
                            bulk_commit();
                        }
                    } else {
                        __syncwarp();
                        uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<long long>(token) * a.o_token + my.head * a.o_head + c0;
                        const int v = lane & 7, pack = (1 << a.pack_log) - 1;
                        for (int rr = lane >> 3; 32 * w + rr < my.rows && rr < 32; rr += 4)
                            if (c0 + 8 * v < a.head_dim)
                                *reinterpret_cast<uint4*>(out + (rr >> a.pack_log) * a.o_token + (rr & pack) * a.o_head + 8 * v) =
                                    st[rr * 8 + (v ^ (rr & 7))];
                        __syncwarp();
                    }
                }
                if (a.lse != nullptr && r < my.rows)
                    a.lse[static_cast<long long>(my.head + (lane & ((1 << a.pack_log) - 1))) * a.total_q + token + (lane >> a.pack_log)] =
                        any && m != -INFINITY ? (m + __log2f(l)) * kLn2 : -INFINITY;
            }
            if (!ok) break;
            done_with_item(k);
        }
        if (!ok) gave_up();
        if (lane == 0) bulk_wait0();  // the warp's TMA stores are done before the CTA exits
        __syncwarp();
    } else if (warp >= 8) {
        setmaxnreg_dec<kOtherRegs>();
        if (warp == 9) {
            // ---------------------------------------------------------------- items and loads
            grid_dependency_wait();
            RingPos r;
            uint32_t loads = 0, qn[2] = {0, 0};
            bool ok = true;
            // Items lie sequence behind sequence, ceil(tiles / 2) for each; sequences whose rows see
            // many keys first (by the power of two of their blocks), so that no long item begins late.
            int level = 32, b0 = a.batch;  // sequences of this level before b0, and of higher levels, have
            long long before = 0;          // `before` items (items come in rising order, as a rule)
            int block = blockIdx.x;
            uint32_t asked = 0;
            struct Seq { int q0, k0, lq, lk, level; };
            auto look_at = [&](int b) {
                Seq x{0, 0, 0, 0, -1};
                if (b < a.batch) {
                    const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
                    // (sequences out of range are reported by the first block's warp 10)
                    if (q0 >= 0 && q1 > q0 && q1 <= a.total_q && k0 >= 0 && k1 >= k0 && k1 <= a.total_k) {
                        x = Seq{q0, k0, q1 - q0, k1 - k0, 0};
                        x.level = 31 - __clz(visible(a.causal, x.lq - 1, x.lq, x.lk) / kKeys + 1);
                    }
                }
                return x;
            };
            const Seq first_window = look_at(lane);  // up to 32 sequences are looked at once
            for (int k = 0;; ++k) {
                int valid = 0, q0s = 0, k0s = 0, lq = 0, lk = 0, sub = 0, kv_head = 0;
                const long long want = block < 0 ? 0 : block / a.kv_heads;
                if (want < before) {
                    level = 32;
                    b0 = a.batch;
                    before = 0;
                }
                while (block >= 0) {
                    if (b0 >= a.batch) {  // the next lower level that occurs
                        int top = -1;
                        for (int b = lane; b < a.batch; b += 32) {
                            const int l = (b < 32 ? first_window : look_at(b)).level;
                            if (l < level) top = max(top, l);
                        }
                        level = __reduce_max_sync(0xffffffffu, top);
                        if (level < 0) break;
                        b0 = 0;
                    }
                    const Seq x = b0 == 0 ? first_window : look_at(b0 + lane);
                    int n = x.level == level ? (tiles_of(a, x.lq) + 1) >> 1 : 0;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int y = __shfl_up_sync(0xffffffffu, n, o);
                        if (lane >= o) n += y;
                    }
                    const unsigned over = __ballot_sync(0xffffffffu, before + n > want);
                    if (over) {
                        const int l = __ffs(over) - 1;
                        valid = 1;
                        q0s = __shfl_sync(0xffffffffu, x.q0, l);
                        k0s = __shfl_sync(0xffffffffu, x.k0, l);
                        lq = __shfl_sync(0xffffffffu, x.lq, l);
                        lk = __shfl_sync(0xffffffffu, x.lk, l);
                        // the last rows, which see the most keys, first
                        sub = 2 * static_cast<int>(before + __shfl_sync(0xffffffffu, n, l) - 1 - want);
                        kv_head = block - static_cast<int>(want) * a.kv_heads;
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, n, 31);
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
                Item& it = sh.item[slot];
                {
                    const Tile x = tile_of(a, sub + (lane & 1), kv_head, lq, lk);  // lanes 0 and 1 have the two tiles
                    const int guarded = x.blocks > 0 ? x.seen_by_all / kKeys : INT32_MAX;
                    const int blocks = max(x.blocks, __shfl_xor_sync(0xffffffffu, x.blocks, 1));
                    const int first = min(guarded, __shfl_xor_sync(0xffffffffu, guarded, 1));
                    if (lane < 2) it.tile[lane] = x;
                    if (lane == 0) {
                        it.valid = valid;
                        it.q0 = q0s;
                        it.k0 = k0s;
                        it.lq = lq;
                        it.lk = lk;
                        it.kv_head = kv_head;
                        it.blocks = blocks;
                        it.first_guarded = first;
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.item_full[slot]);
                // the next item's block, while this one loads
                auto ask = [&]() {
                    if (lane == 0) {
                        fence_proxy_async_smem();
                        mbar_arrive_expect_tx(&sh.next, 16);
                        cancel_next_block(&sh.response, &sh.next);
                    }
                    __syncwarp();
                };
                // (the answer is read even when a wait gave up: it must not arrive after the CTA's end)
                auto answer = [&]() {
                    if (!__all_sync(0xffffffffu, mbar_wait_bounded(&sh.next, asked++ & 1, nullptr, drain_limit))) return false;
                    block = cancelled_block(&sh.response);
                    __syncwarp();
                    return true;
                };
                if (!valid) {
                    // The grid has more blocks than there are items (the host does not know the lengths). Those
                    // past the last item are taken here, beside the end of the work; each left to run would
                    // hold an SM for 3 us.
                    while (block >= 0) {
                        ask();
                        if (!answer()) {
                            ok = false;
                            break;
                        }
                    }
                    break;
                }
                ask();
                const int blocks = it.blocks;
                auto load_block = [&](const CUtensorMap* m, int j) {
                    ok = wait(&sh.empty[r.s], r.ph ^ 1);
                    if (!ok) return;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.full[r.s], Cfg::kTile);
#pragma unroll
                        for (int c = 0; c < DCH; ++c)
                            tma_load_3d(ring + r.s * Cfg::kTile + c * Cfg::kChunk, m, &sh.full[r.s], 64 * c, kv_head, k0s + j * kKeys);
                    }
                    __syncwarp();
                    ++loads;
                    r.step<S>();
                };
                // Q's place is free only when the last item's last scores are through: until then its tiles come
                // as far as L2, and the first K block goes ahead
                if (lane < 2 * DCH && it.tile[lane / DCH].blocks)
                    tma_prefetch_3d(&tmQ, 64 * (lane % DCH), it.tile[lane / DCH].head, q0s + it.tile[lane / DCH].token0);
                __syncwarp();
                if (blocks > 0) load_block(&tmK, 0);
                for (int t = 0; t < 2 && ok; ++t) {
                    if (it.tile[t].blocks == 0) continue;
                    ok = wait(&sh.q_empty[t], (qn[t] & 1) ^ 1);
                    if (!ok) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&sh.q_full[t], Cfg::kTile);
#pragma unroll
                        for (int c = 0; c < DCH; ++c)
                            tma_load_3d(sq + t * Cfg::kTile + c * Cfg::kChunk, &tmQ, &sh.q_full[t], 64 * c, it.tile[t].head, q0s + it.tile[t].token0);
                    }
                    __syncwarp();
                    ++qn[t];
                }
                for (int j = 0; j < blocks && ok; ++j) {
                    load_block(&tmV, j);
                    if (ok && j + 1 < blocks) load_block(&tmK, j + 1);
                }
                if (!answer() || !ok) {
                    ok = false;
                    break;
                }
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
            uint32_t qn[2] = {0, 0}, on[2] = {0, 0}, vn = 0;  // Q tiles, results of each tile, V blocks so far
            bool ok = true;
            for (int k = 0; next_item(k, ok); ++k) {
                const Item& it = sh.item[k % kItems];
                const int nb[2] = {it.tile[0].blocks, it.tile[1].blocks}, blocks = it.blocks;
                const bool has[2] = {it.tile[0].rows > 0, it.tile[1].rows > 0};
                done_with_item(k);
                if (blocks > 0) {
                    ok = wait(&sh.full[r.s], r.ph);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (nb[t] == 0) continue;
                        ok = ok && wait(&sh.q_full[t], qn[t]++ & 1);
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, r.s);
                        if (nb[t] == 1) commit(&sh.q_empty[t]);
                    }
                    if (!ok) break;
                    commit(&sh.empty[r.s]);
                    r.step<S>();
                }
                for (int j = 0; j < blocks; ++j, ++vn) {
                    const RingPos v = r;
                    r.step<S>();
                    ok = wait(&sh.full[v.s], v.ph) && wait(&sh.guard[vn % kGuards], (vn / kGuards) & 1);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j < nb[t]) {
                            // the first product overwrites O, so the last result must have been read
                            if (j == 0 && on[t] > 0) ok = ok && wait(&sh.o_empty[t], (on[t] - 1) & 1);
                            ok = ok && wait(&sh.p_half[t], n[t] & 1);
                            if (!ok) break;
                            tc_fence_after();
                            product(t, v.s, 0, j == 0);
                            commit(&sh.half_done[t]);
                            ok = wait(&sh.p_full[t], n[t]++ & 1);
                            if (!ok) break;
                            tc_fence_after();
                            product(t, v.s, 1, false);
                            if (j + 1 == nb[t]) commit(&sh.o_full[t]);
                        }
                        if (t == 1) commit(&sh.empty[v.s]);
                        if (j + 1 < nb[t]) {
                            ok = wait(&sh.full[r.s], r.ph);
                            if (!ok) break;
                            tc_fence_after();
                            scores(t, r.s);
                            if (j + 2 == nb[t]) commit(&sh.q_empty[t]);
                        }
                    }
                    if (!ok) break;
                    if (j + 1 < blocks) {
                        commit(&sh.empty[r.s]);
                        r.step<S>();
                    }
                }
                if (!ok) break;
#pragma unroll
                for (int t = 0; t < 2; ++t) on[t] += has[t];
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
            for (int k = 0; next_item(k, ok); ++k) {
                const Item& it = sh.item[k % kItems];
                const int blocks = it.blocks, from = it.first_guarded, lk = it.lk;
                const int nb0 = it.tile[0].blocks, nb1 = it.tile[1].blocks, seen0 = it.tile[0].seen_by_all, seen1 = it.tile[1].seen_by_all;
                for (int j = 0; j < blocks; ++j, ++vn) {
                    r.step<S>();  // past the K block
                    ok = wait(&sh.full[r.s], r.ph);
                    if (!ok) break;
                    // a tile that does not reach this block has no say in it
                    const int seen = min(j < nb0 ? seen0 : INT32_MAX, j < nb1 ? seen1 : INT32_MAX);
                    if (seen < (j + 1) * kKeys) {
                        guard_block<BF16, DCH>(sh, k % kItems, ring + r.s * Cfg::kTile, lk - j * kKeys, (j - from) * kKeys, threadIdx.x - 320);
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
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t ts = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * 128;
        const uint32_t to = ts + 256;  // O
        const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2);
        uint32_t n = 0, outs = 0;  // blocks and results so far
        bool ok = true;
        for (int k = 0; next_item(k, ok); ++k) {
            const Item& it = sh.item[k % kItems];
            const Tile my = it.tile[t];
            // keys that this thread's row sees, and the first and the last row of the warp (rows past the
            // tile's end count as its last)
            const int last = (my.rows - 1) >> a.pack_log;
            const int sees = visible(a.causal, my.token0 + min(r >> a.pack_log, last), it.lq, it.lk);
            const int lo = __shfl_sync(0xffffffffu, sees, 0), hi = __shfl_sync(0xffffffffu, sees, 31);
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < my.blocks; ++j, ++n) {
                ok = wait(&sh.s_full[t], n & 1);
                if (!ok) break;
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
                const int lo_j = lo - j * kKeys, hi_j = hi - j * kKeys;
                // O and l to a new reference. (O holds every product so far: S was committed after them.)
                auto rescale = [&](float to_m) {
                    const float f = to_m == m ? 1.f : exp2_fast(m - to_m);
                    m = to_m;
                    l *= f;
#pragma unroll 1
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
                };
                auto hand_over = [&](uint64_t* bar) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                bool done = false;
                if (lo_j >= kKeys) {
                    if (j == 0) m = top32(x) * a.scale_log2;
                    uint32_t p[32];
                    const float s0 = weights<BF16, 32>(x, scale2, m, p);
                    // (also when m is not a number yet: -inf - -inf)
                    if (!__any_sync(0xffffffffu, !(s0 < kMostSum) || m == -INFINITY)) {
                        tmem_st_32x32b_x32(ts, p);
                        hand_over(&sh.p_half[t]);
                        l += s0;
                        float s1 = weights<BF16, 32>(x + 64, scale2, m, p);
                        const bool ran = !(s1 < kMostSum);
                        if (__any_sync(0xffffffffu, ran)) {
                            // the first half's product must be through before O is rescaled
                            ok = wait(&sh.half_done[t], n & 1);
                            if (!ok) break;
                            tc_fence_after();
                            rescale(ran ? max_nan(m, max_nan(top32(x + 64), top32(x + 96)) * a.scale_log2) : m);
                            s1 = weights<BF16, 32>(x + 64, scale2, m, p);
                        }
                        tmem_st_32x32b_x32(ts + 32, p);
                        hand_over(&sh.p_full[t]);
                        l += s1;
                        done = true;
                    }
                }
                if (!done) {
                    // Chunks of 32 keys: seen by all of the warp's rows, by some, or by none.
                    const int seen = sees - j * kKeys;
                    float top = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (32 * c >= hi_j) continue;
                        if (32 * (c + 1) > lo_j) {
#pragma unroll
                            for (int i = 32 * c; i < 32 * c + 32; ++i) x[i] = i < seen ? x[i] : -INFINITY;
                        }
                        top = max_nan(top, top32(x + 32 * c));
                    }
                    // a NaN among the scores becomes the row's reference and with it the whole row
                    top *= a.scale_log2;
                    const bool grow = !(top <= m + kGrowth);
                    if (j == 0) m = top;
                    else if (__any_sync(0xffffffffu, grow)) rescale(grow ? top : m);
                    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t p[16];
                        if (32 * c < hi_j) {
                            l += weights<BF16, 16>(x + 32 * c, scale2, base, p);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) p[i] = 0;
                        }
                        tmem_st_32x32b_x16(ts + 16 * c, p);
                        if (c == 1) hand_over(&sh.p_half[t]);
                    }
                    hand_over(&sh.p_full[t]);
                }
            }
            if (!ok) break;
            if (my.rows > 0) {
                if (outs > 0) ok = wait(&sh.o_empty[t], (outs - 1) & 1);  // the last m and l have been read
                if (!ok) break;
                ++outs;
                sh.ml[t][r] = make_float2(m, l);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.ml_full[t]);
            }
            done_with_item(k);
        }
        if (!ok) gave_up();
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

tb_status device_check(const char* op, const tb_context* ctx) {
    int current = 0;
    TB_CUDA(cudaGetDevice(&current));
    if (current != ctx->device)
        return fail(TB_ERR_INVALID_ARGUMENT, "%s: device %d is current, the context's is %d", op, current, ctx->device);
    return TB_OK;
}

// [tokens][heads][head_dim] as {head_dim, heads, tokens}, boxes of some tokens by some heads by 64 elements.
static tb_status tile_map(CUtensorMap* m, const tb_attention_desc* d, const void* p, int64_t heads, int64_t tokens,
                          int64_t token_stride, int64_t head_stride, int box_heads, int box_tokens) {
    // the stride of a dimension of one element says nothing; the map wants a valid one
    const uint64_t head = heads > 1 ? head_stride : d->head_dim, token = tokens > 1 ? token_stride : d->head_dim;
    const uint64_t dims[3] = {static_cast<uint64_t>(d->head_dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
    const uint64_t strides[2] = {head * 2, token * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(box_heads), static_cast<uint32_t>(box_tokens)};
    return encode_tiled(m, d->dtype == TB_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p,
                        dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool BF16, int DCH>
static tb_status launch_prompt(tb_context* ctx, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                               const CUtensorMap& o, const PromptArgs& a, long long grid, cudaStream_t st) {
    auto* kernel = prompt_kernel<BF16, DCH>;
    constexpr int kSmem = PromptCfg<DCH>::kTiles + static_cast<int>(sizeof(PromptShared));
    static OncePerDevice once;
    TB_TRY(once([&]() -> tb_status {
        // the warpgroups re-split the registers of the launch (setmaxnreg), which needs all of them
        cudaFuncAttributes fa;
        TB_CUDA(cudaFuncGetAttributes(&fa, kernel));
        if (fa.numRegs < kLaunchRegs)
            return fail(TB_ERR_CUDA, "attention built with %d registers a thread; its register split needs %d", fa.numRegs, kLaunchRegs);
        TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        return TB_OK;
    }));
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
    TB_TRY(device_check("attention", ctx));
    // without keys nothing is loaded; the maps are made of q's first row
    const bool keys = d->total_k > 0;
    CUtensorMap mq, mk, mv, mo;
    const int group = d->q_heads / d->kv_heads;
    int pack = 0;  // log2 of the heads of a tile
    if (group <= 32 && (group & (group - 1)) == 0)
        while ((1 << pack) < group) ++pack;
    TB_TRY(tile_map(&mq, d, q, d->q_heads, d->total_q, d->q_token_stride, d->q_head_stride, 1 << pack, kRows >> pack));
    TB_TRY(tile_map(&mk, d, keys ? k : q, keys ? d->kv_heads : 1, keys ? d->total_k : 1, d->k_token_stride, d->k_head_stride, 1, kKeys));
    TB_TRY(tile_map(&mv, d, keys ? v : q, keys ? d->kv_heads : 1, keys ? d->total_k : 1, d->v_token_stride, d->v_head_stride, 1, kKeys));
    TB_TRY(tile_map(&mo, d, out, d->q_heads, d->total_q, d->out_token_stride, d->out_head_stride, 1 << pack, 32 >> pack));
    // A grid that leaves SMs free lets the next kernel set itself up there (back to back, one chat turn 9.8 -> 8.9
    // us). With more items than SMs the next kernel's blocks would take SMs from this one's end (24 packed
    // prompts 126 -> 136 us).
    const unsigned early = static_cast<unsigned>(ctx->num_sms / 2);
    PromptArgs a{out, lse, cu_q, cu_k, d->out_token_stride, d->out_head_stride, d->total_q, d->total_k, d->batch, group,
                 d->kv_heads, d->head_dim, d->causal, pack, d->scale * kLog2e, early, ctx->dev_err, ctx->timeout_cycles};
    // most items that lengths summing to total_q can have: the lengths themselves are on the device
    const long long seqs = d->batch < d->total_q ? d->batch : d->total_q;
    const long long heads = group >> pack;
    const long long tiles = ((d->total_q - seqs) / (kRows >> pack) + seqs) * heads;
    const long long grid = (heads % 2 ? (tiles + seqs) / 2 : tiles / 2) * d->kv_heads;
    if (grid > INT32_MAX) return fail(TB_ERR_NOT_ACCELERATED, "attention: more than 2^31 tiles");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = d->head_dim > 64;
    if (d->dtype == TB_DT_BF16)
        return wide ? launch_prompt<true, 2>(ctx, mq, mk, mv, mo, a, grid, st) : launch_prompt<true, 1>(ctx, mq, mk, mv, mo, a, grid, st);
    return wide ? launch_prompt<false, 2>(ctx, mq, mk, mv, mo, a, grid, st) : launch_prompt<false, 1>(ctx, mq, mk, mv, mo, a, grid, st);
}

}  // extern "C"
