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
// A CTA takes two tiles of 128 rows (two heads of one key head's group, or two row tiles of one
// head) that walk the same blocks of 128 keys. 12 warps:
//   warps 0-3, 4-7  softmax of tile 0 / 1, one row a thread: read the scores from tensor memory, write
//                   the weights back to it as f16 / bf16, rescale o there when m moves, and store the
//                   result at the end
//   warp 8          issues the MMAs: S = Q K^T (both from shared memory), O += P V (P from tensor memory)
//   warp 9          TMA loads: the Q tiles, then K and V blocks through a ring
//   warps 10-11     look through the V blocks that some row sees only in part (see guard_block)
// While one tile's softmax runs, the tensor cores work on the other tile. Tensor memory: S of both
// tiles (128 columns each; P takes the first 64 of its S once the scores have been read) and O.
//
// Per tile and block the MMAs take 2 * 128 * 128 * head_dim multiply-adds (1024 cycles at head_dim 128)
// and the 128 * 128 exponentials 1024 cycles of the special-function units, so the two are level and
// neither may wait for the other.
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

// DCH: 64-element chunks of head_dim.
template <int DCH>
struct PromptCfg {
    static constexpr int kChunk = kRows * 128;        // one chunk of a tile: 128 rows of 128 bytes, swizzled
    static constexpr int kTile = DCH * kChunk;
    static constexpr int kStages = DCH == 2 ? 5 : 8;  // ring of K and V blocks
    static constexpr int kSmem = 1024 + (2 + kStages) * kTile;
};

struct PromptShared {
    uint64_t q_full[2], full[8], empty[8], guard[kGuards], guard_done, s_full[2], p_full[2], o_full[2], drain;
    uint32_t tmem;
    int abort;
    int seq, item;           // this CTA's sequence and item in it; seq < 0: none
    int scan[13];
    int odd;                 // some guarded value is not finite
    int first[3][kKeys];     // per dimension: the first guarded key with NaN, +inf, -inf
};

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

__device__ __forceinline__ int visible(const PromptArgs& a, int row, int lq, int lk) {
    if (!a.causal) return lk;
    return max(0, min(lk, row + lk - lq + 1));
}

__device__ __forceinline__ Tile tile_of(const PromptArgs& a, int sub, int kv_head, int lq, int lk) {
    Tile t{0, 0, 0, 0, 0};
    const int rt = sub / a.group;
    t.row0 = rt * kRows;
    t.rows = min(kRows, lq - t.row0);
    if (t.rows <= 0) {
        t.rows = 0;
        t.seen_by_all = INT32_MAX;
        return t;
    }
    t.head = kv_head * a.group + (sub - rt * a.group);
    t.blocks = (visible(a, t.row0 + t.rows - 1, lq, lk) + kKeys - 1) / kKeys;
    t.seen_by_all = visible(a, t.row0, lq, lk);
    return t;
}

// A weight of 0 does not take a key out of a product when the value is NaN or infinite. In a block
// that some row sees only in part, V is therefore put in order before the MMA reads it: rows past the
// sequence's end become zero, and values that are not finite become zero with their place noted
// (first[]), to be added by the rows that do see them when they store their result. 64 threads.
template <bool BF16, int DCH>
__device__ void guard_block(PromptShared& sh, uint8_t* v, int first_key, int lk, int head_dim, int t) {
    constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u;   // exponent of both halves
    constexpr uint32_t kOne = BF16 ? 0x00800080u : 0x04000400u;   // all ones + 1: a carry into bit 15
    constexpr uint32_t kFrac = BF16 ? 0x7Fu : 0x3FFu;
    const int live = lk - first_key;  // rows of the block inside the sequence
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
            atomicMin(&sh.first[kind][d0 + e], first_key + row);
            w[e >> 1] &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
            sh.odd = 1;
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ void tmem_ld_row(uint32_t taddr, uint32_t (&s)[128]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + 32 * c, r);
#pragma unroll
        for (int i = 0; i < 32; ++i) s[32 * c + i] = r[i];
    }
}

template <bool BF16, int DCH>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const PromptArgs a) {
    using Cfg = PromptCfg<DCH>;
    constexpr int S = Cfg::kStages;
    extern __shared__ uint8_t raw[];
    __shared__ PromptShared sh;
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sq = base;
    uint8_t* ring = base + 2 * Cfg::kTile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &sh.abort;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
        }
        for (int i = 0; i < S; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < kGuards; ++i) mbar_init(&sh.guard[i], 2);
        mbar_init(&sh.guard_done, 2);
        mbar_init(&sh.drain, 1);
        fence_mbar_init();
        sh.abort = 0;
        sh.seq = -1;
        sh.odd = 0;
    }
    for (int i = threadIdx.x; i < 3 * kKeys; i += kThreads) (&sh.first[0][0])[i] = INT32_MAX;
    if (warp == 8) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
        if (lane == 0) {
            tma_prefetch_desc(&tmQ);
            tma_prefetch_desc(&tmK);
            tma_prefetch_desc(&tmV);
        }
    }
    grid_dependency_wait();
    // This CTA's item: items lie sequence behind sequence, ceil(row tiles * group / 2) for each.
    const int kv_head = blockIdx.x % a.kv_heads;
    const long long want = blockIdx.x / a.kv_heads;
    {
        long long before = 0;
        for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
            const int b = b0 + threadIdx.x;
            int items = 0;
            if (b < a.batch) {
                const long long q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
                if (q0 < 0 || q1 < q0 || q1 > a.total_q || k0 < 0 || k1 < k0 || k1 > a.total_k) {
                    if (blockIdx.x == 0) atomicOr(a.err, DEV_ERR_INDEX);
                } else {
                    items = static_cast<int>(((q1 - q0 + kRows - 1) / kRows * a.group + 1) >> 1);
                }
            }
            int x = items;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) sh.scan[warp] = x;
            __syncthreads();
            int pre = 0, total = 0;
            for (int w = 0; w < kThreads / 32; ++w) {
                if (w < warp) pre += sh.scan[w];
                total += sh.scan[w];
            }
            const long long hi = before + pre + x, lo = hi - items;
            if (lo <= want && want < hi) {
                sh.seq = b;
                sh.item = static_cast<int>(hi - 1 - want);  // the last rows, which see the most keys, first
            }
            before += total;
            if (before > want) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int seq = sh.seq;
    const long long limit = a.timeout_cycles;
    const long long drain_limit = limit > kDrainCycles ? limit : kDrainCycles;

    if (seq >= 0) {
        const int q0 = a.cu_q[seq], k0 = a.cu_k[seq];
        const int lq = a.cu_q[seq + 1] - q0, lk = a.cu_k[seq + 1] - k0;
        const Tile tile[2] = {tile_of(a, 2 * sh.item, kv_head, lq, lk), tile_of(a, 2 * sh.item + 1, kv_head, lq, lk)};
        const int blocks = max(tile[0].blocks, tile[1].blocks);

        if (warp >= 8) {
            setmaxnreg_dec<kOtherRegs>();
            if (warp == 9 && lane == 0 && blocks > 0) {
                // ------------------------------------------------------------ loads
                for (int t = 0; t < 2; ++t) {
                    if (tile[t].blocks == 0) continue;
                    mbar_arrive_expect_tx(&sh.q_full[t], Cfg::kTile);
                    for (int c = 0; c < DCH; ++c)
                        tma_load_3d(sq + t * Cfg::kTile + c * Cfg::kChunk, &tmQ, &sh.q_full[t], 64 * c, tile[t].head,
                                    q0 + tile[t].row0);
                }
                int it = 0, s = 0;
                uint32_t ph = 0;
                bool ok = true;
                for (; it < 2 * blocks; ++it) {
                    if (!mbar_wait_bounded(&sh.empty[s], ph ^ 1, abort_flag, limit)) { ok = false; break; }
                    mbar_arrive_expect_tx(&sh.full[s], Cfg::kTile);
                    const CUtensorMap* m = (it & 1) ? &tmV : &tmK;
                    for (int c = 0; c < DCH; ++c)
                        tma_load_3d(ring + s * Cfg::kTile + c * Cfg::kChunk, m, &sh.full[s], 64 * c, kv_head,
                                    k0 + (it >> 1) * kKeys);
                    if (++s == S) { s = 0; ph ^= 1; }
                }
                if (!ok) { atomicOr(a.err, DEV_ERR_TIMEOUT); *abort_flag = 1; }
                // every issued load lands before the CTA may exit
                for (int t = 0; t < 2; ++t)
                    if (tile[t].blocks) mbar_wait_bounded(&sh.q_full[t], 0, nullptr, drain_limit);
                for (int i = it > S ? it - S : 0; i < it; ++i)
                    mbar_wait_bounded(&sh.full[i % S], (i / S) & 1, nullptr, drain_limit);
            } else if (warp == 8 && lane == 0 && blocks > 0) {
                // ------------------------------------------------------------ MMAs
                const uint32_t idesc_s = idesc_f16(kRows, kKeys, BF16, false);
                const uint32_t idesc_o = idesc_f16(kRows, a.head_dim, BF16, true);
                const int ksteps = a.head_dim / 16;
                bool ok = true;
                auto wait = [&](uint64_t* bar, uint32_t ph) {
                    if (ok && !mbar_wait_bounded(bar, ph, abort_flag, limit)) ok = false;
                    return ok;
                };
                auto scores = [&](int t, int stage) {
                    const uint32_t qa = smem_u32(sq + t * Cfg::kTile), kb = smem_u32(ring + stage * Cfg::kTile);
                    for (int k = 0; k < ksteps; ++k) {
                        const uint32_t o = (k >> 2) * Cfg::kChunk + (k & 3) * 32;
                        tc_mma<1>(tmem + t * 128, smem_desc(qa + o, 16, 1024, 2), smem_desc(kb + o, 16, 1024, 2), idesc_s, k > 0);
                    }
                    tc_commit(&sh.s_full[t]);
                };
                auto product = [&](int t, int stage, bool first) {
                    const uint32_t vb = smem_u32(ring + stage * Cfg::kTile);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        tc_mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8,
                                      smem_desc(vb + k * 2048, Cfg::kChunk, 1024, 2), idesc_o, !first || k > 0);
                };
                wait(&sh.full[0], 0);
                for (int t = 0; t < 2; ++t)
                    if (tile[t].blocks && wait(&sh.q_full[t], 0)) {
                        tc_fence_after();
                        scores(t, 0);
                    }
                tc_commit(&sh.empty[0]);
                int it = 1;  // V block j is ring entry 2 j + 1, the next K block 2 j + 2
                for (int j = 0; j < blocks && ok; ++j, it += 2) {
                    const int sv = it % S, sk = (it + 1) % S;
                    const uint32_t pv = (it / S) & 1, pk = ((it + 1) / S) & 1;
                    wait(&sh.full[sv], pv);
                    wait(&sh.guard[j % kGuards], (j / kGuards) & 1);
                    for (int t = 0; t < 2 && ok; ++t) {
                        if (j < tile[t].blocks && wait(&sh.p_full[t], j & 1)) {
                            tc_fence_after();
                            product(t, sv, j == 0);
                            if (j + 1 == tile[t].blocks) tc_commit(&sh.o_full[t]);
                        }
                        if (t == 1) tc_commit(&sh.empty[sv]);
                        if (j + 1 < tile[t].blocks && wait(&sh.full[sk], pk)) {
                            tc_fence_after();
                            scores(t, sk);
                        }
                    }
                    if (j + 1 < blocks) tc_commit(&sh.empty[sk]);
                }
                if (!ok) { atomicOr(a.err, DEV_ERR_TIMEOUT); *abort_flag = 1; }
                tc_commit(&sh.drain);
                mbar_wait_bounded(&sh.drain, 0, nullptr, drain_limit);
            } else if (warp >= 10) {
                // ------------------------------------------------------------ V blocks seen in part
                bool ok = true;
                for (int j = 0; j < blocks && ok; ++j) {
                    const int it = 2 * j + 1;
                    // a tile that does not reach this block has no say in it
                    const int seen = min(j < tile[0].blocks ? tile[0].seen_by_all : INT32_MAX,
                                         j < tile[1].blocks ? tile[1].seen_by_all : INT32_MAX);
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sh.full[it % S], (it / S) & 1, abort_flag, limit));
                    if (!ok) break;
                    if (seen < (j + 1) * kKeys) {
                        guard_block<BF16, DCH>(sh, ring + (it % S) * Cfg::kTile, j * kKeys, lk, a.head_dim, threadIdx.x - 320);
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.guard[j % kGuards]);
                }
                __syncwarp();
                if (lane == 0) {
                    if (!ok) { atomicOr(a.err, DEV_ERR_TIMEOUT); *abort_flag = 1; }
                    mbar_arrive(&sh.guard_done);
                }
            }
        } else {
            // ------------------------------------------------------------ softmax
            setmaxnreg_inc<kSoftmaxRegs>();
            const int t = warp >> 2;
            const Tile my = t ? tile[1] : tile[0];
            const int r = threadIdx.x & 127;
            const int row = my.row0 + r;
            const int sees = r < my.rows ? visible(a, row, lq, lk) : lk;
            const uint32_t ts = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * 128;
            const uint32_t to = ts + 256;  // O
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < my.blocks; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sh.s_full[t], j & 1, abort_flag, limit));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[128];
                tmem_ld_row(ts, s);
                tmem_ld_wait();
                float x[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) {
                    asm volatile("" : "+r"(s[i]));
                    x[i] = __uint_as_float(s[i]);
                }
                if (my.seen_by_all < (j + 1) * kKeys) {
                    const int n = sees - j * kKeys;
#pragma unroll
                    for (int i = 0; i < 128; ++i) x[i] = i < n ? x[i] : -INFINITY;
                }
                float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int i = 4; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], x[i]);
                const float m1 = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2;
                const bool grow = m1 > m + kGrowth;
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
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float u = exp2_fast(fmaf(x[64 * c + 2 * i], a.scale_log2, -base));
                        const float w = exp2_fast(fmaf(x[64 * c + 2 * i + 1], a.scale_log2, -base));
                        sum[(2 * i) & 3] += u;
                        sum[(2 * i + 1) & 3] += w;
                        p[i] = pack2<BF16>(u, w);
                    }
                    tmem_st_32x32b_x32(ts + 32 * c, p);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.p_full[t]);
            }
            if (my.blocks > 0 && ok)
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sh.o_full[t], 0, abort_flag, limit) &&
                                                 mbar_wait_bounded(&sh.guard_done, 0, abort_flag, limit));
            tc_fence_after();
            if (ok) {
                const bool live = r < my.rows, any = sees > 0;
                const float inv = any ? 1.f / l : 0.f;
                const int odd = sh.odd;
                uint16_t* out = static_cast<uint16_t*>(a.out) + static_cast<long long>(q0 + row) * a.o_token + my.head * a.o_head;
                for (int c = 0; c < a.head_dim; c += 16) {
                    uint32_t o[16];
                    if (my.blocks > 0) {
                        tmem_ld_32x32b_x16(to + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(o[i]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = 0;
                    }
                    if (odd) {
                        for (int i = 0; i < 16; ++i) {
                            float y = __uint_as_float(o[i]);
                            if (sh.first[0][c + i] < sees) y = NAN;
                            if (sh.first[1][c + i] < sees) y += INFINITY;
                            if (sh.first[2][c + i] < sees) y -= INFINITY;
                            o[i] = __float_as_uint(y);
                        }
                    }
                    uint32_t h[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        h[i] = any ? pack2<BF16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv) : 0u;
                    if (live) {
                        *reinterpret_cast<uint4*>(out + c) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                }
                if (a.lse != nullptr && live)
                    a.lse[static_cast<long long>(my.head) * a.total_q + q0 + row] =
                        any ? ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2 : -INFINITY;
            } else if (lane == 0) {
                atomicOr(a.err, DEV_ERR_TIMEOUT);
                *abort_flag = 1;
            }
            tc_fence_before();
        }
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

// [tokens][heads][head_dim] as {head_dim, heads, tokens}, boxes of 128 tokens by 64 elements of one head.
static tb_status tile_map(CUtensorMap* m, const tb_attention_desc* d, const void* p, int64_t heads, int64_t tokens,
                          const int64_t* stride) {
    // the stride of a dimension of one element says nothing; the map wants a valid one
    const uint64_t head = heads > 1 ? stride[1] : d->head_dim, token = tokens > 1 ? stride[0] : d->head_dim;
    const uint64_t dims[3] = {static_cast<uint64_t>(d->head_dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(tokens)};
    const uint64_t strides[2] = {head * 2, token * 2};
    const uint32_t box[3] = {64, 1, kRows};
    return encode_tiled(m, d->dtype == TB_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p,
                        dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool BF16, int DCH>
static tb_status launch_prompt(tb_context* ctx, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                               const PromptArgs& a, long long grid, cudaStream_t st) {
    auto* kernel = prompt_kernel<BF16, DCH>;
    static bool ready = false;  // the attribute is per function and process-wide
    if (!ready) {
        // the warpgroups re-split the registers of the launch (setmaxnreg), which needs all of them
        cudaFuncAttributes fa;
        TB_CUDA(cudaFuncGetAttributes(&fa, kernel));
        if (fa.numRegs < kLaunchRegs)
            return fail(TB_ERR_CUDA, "attention built with %d registers a thread; its register split needs %d", fa.numRegs, kLaunchRegs);
        TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptCfg<DCH>::kSmem));
        ready = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = PromptCfg<DCH>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA(cudaLaunchKernelEx(&cfg, kernel, q, k, v, a));
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
    for (const int64_t* s : {d->q_stride, d->k_stride, d->v_stride, d->out_stride}) {
        if (s[0] < 0 || s[1] < 0) return fail(TB_ERR_SHAPE_MISMATCH, "attention: negative stride");
        strides |= s[0] | s[1];
    }
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || (strides & 7))
        return fail(TB_ERR_INVALID_ARGUMENT, "attention: tensors must be 16-byte aligned with strides that are multiples of 8");
    // without keys nothing is loaded; the maps are made of q's first row
    const bool keys = d->total_k > 0;
    CUtensorMap mq, mk, mv;
    TB_TRY(tile_map(&mq, d, q, d->q_heads, d->total_q, d->q_stride));
    TB_TRY(tile_map(&mk, d, keys ? k : q, keys ? d->kv_heads : 1, keys ? d->total_k : 1, d->k_stride));
    TB_TRY(tile_map(&mv, d, keys ? v : q, keys ? d->kv_heads : 1, keys ? d->total_k : 1, d->v_stride));
    const int group = d->q_heads / d->kv_heads;
    PromptArgs a{out, lse, cu_q, cu_k, d->out_stride[0], d->out_stride[1], d->total_q, d->total_k, d->batch, group,
                 d->kv_heads, d->head_dim, d->causal, d->scale * kLog2e, ctx->dev_err, ctx->timeout_cycles};
    // most items that lengths summing to total_q can have: the lengths themselves are on the device
    const long long seqs = d->batch < d->total_q ? d->batch : d->total_q;
    const long long grid = ((d->total_q / kRows + seqs) * group / 2 + seqs) * d->kv_heads;
    if (grid > INT32_MAX) return fail(TB_ERR_NOT_ACCELERATED, "attention: more than 2^31 tiles");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = d->head_dim > 64;
    if (d->dtype == TB_DT_BF16)
        return wide ? launch_prompt<true, 2>(ctx, mq, mk, mv, a, grid, st) : launch_prompt<true, 1>(ctx, mq, mk, mv, a, grid, st);
    return wide ? launch_prompt<false, 2>(ctx, mq, mk, mv, a, grid, st) : launch_prompt<false, 1>(ctx, mq, mk, mv, a, grid, st);
}

}  // extern "C"
