// Attention of one new token a sequence over the paged cache.
//
// The formula is attention.cu's with one row a sequence. Every key and value is read once and used
// for the group's query heads only, so the kernel is bound by memory bandwidth: its work is cut so that
// every SM streams the same amount, and the arithmetic (mma.sync on 16 query rows, most of them
// padding) only has to keep up.
//
// Cut: a unit is one sequence, key head and at most 16 of its query heads; its keys come in tiles of 64
// tokens. The tiles of all units in a row are divided evenly over the CTAs (two on each SM), so a CTA
// takes the end of one unit, some whole units and the beginning of another. A unit that lies in one CTA
// is finished there. Of a unit that several CTAs share, each leaves its unscaled sum, maximum and sum of
// weights, and the CTA that arrives last adds them in the order of the keys: the result does not depend
// on who that is. (It does depend, in its last bits, on where the cuts fall, that is on the lengths of the
// whole batch.) Nobody waits for another CTA.
//
// A CTA: warp 4 looks the pages up and loads K and V tiles by TMA (boxes as high as the greatest common
// divisor of 64 and the page size, so that a box never crosses a page) and the query rows, three tiles
// ahead; warps 0-3 take 16 of a tile's 64 keys each for S = Q K^T, share the maximum and the weights through
// shared memory, and take a quarter of head_dim each for O += P V. Two barriers a tile.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "cache.hpp"
#include "ptx.cuh"
#include "quant.cuh"

namespace tb {

constexpr int kTokens = 64;                    // keys of a tile
constexpr int kUnitRows = 16;                  // query rows of a unit
constexpr int kConsumers = 128;
constexpr int kDecodeThreads = kConsumers + 32;
constexpr int kDecodeStages = 3;
constexpr int kQPitch = 272;                   // bytes from one query row to the next: 8 rows hit 8 bank groups
constexpr int kPPitch = 144;                   // the same for the weights
constexpr long long kDecodeDrain = 2000000000ll;  // bound on a CTA's waits for its own copies at its end

template <int DCH>
struct DecodeCfg {
    static constexpr int kTensor = DCH * kTokens * 128;  // K or V of a tile, 64-element chunks of 128-byte rows, swizzled
    static constexpr int kStage = 2 * kTensor;
    static constexpr int kSmem = 1024 + kDecodeStages * kStage + 2 * kUnitRows * kQPitch + kUnitRows * kPPitch;
};

struct DecodeArgs {
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    const int32_t *slots, *table, *lengths;
    long long q_seq, q_head, o_seq, o_head;
    int n, q_heads, kv_heads, group, chunks, head_dim, page_size, num_pages, max_seqs, max_pages;
    int box;                   // rows of a TMA box
    float scale_log2;
    float* part_o;
    float2* part_ml;
    uint32_t* arrived;
    uint32_t* err;
    long long timeout_cycles;
};

struct DecodeShared {
    uint64_t full[kDecodeStages], empty[kDecodeStages], q_full[2], q_empty[2];
    float top[4][kUnitRows], sum[4][kUnitRows];
    long long scan[kDecodeThreads / 32];
    long long start_before;    // tiles before the start's row
    int start_row;
    int abort, last;
};

// Tiles of one row's units, 0 when the row is refused. A row without tokens has one empty tile.
__device__ __forceinline__ int row_tiles(const DecodeArgs& a, int i, int& slot, int& len, uint32_t& err) {
    slot = a.slots[i];
    if (slot < 0 || slot >= a.max_seqs) {
        err |= DEV_ERR_INDEX;
        return 0;
    }
    len = a.lengths[slot];
    if (len < 0 || static_cast<long long>(len) > static_cast<long long>(a.max_pages) * a.page_size) {
        err |= DEV_ERR_INDEX;
        return 0;
    }
    return max(1, (len + kTokens - 1) / kTokens);
}

// This CTA's tiles, segment by segment: tiles [t0, t1) of one unit.
struct Walk {
    long long x, end, rem;   // next tile, end of the CTA's tiles, tiles of row i before x
    int i, nt, len, slot;
    int unit, t0, t1;
    long long unit_start;    // the unit's first tile
    __device__ void begin(const DecodeArgs& a, long long x0, long long x1, int row, long long before) {
        x = x0;
        end = x1;
        i = row;
        rem = x0 - before;
        uint32_t e = 0;
        nt = x < end ? row_tiles(a, i, slot, len, e) : 0;
    }
    __device__ bool next(const DecodeArgs& a) {
        if (x >= end) return false;
        const int units = a.kv_heads * a.chunks;
        while (rem >= static_cast<long long>(nt) * units) {
            uint32_t e = 0;
            if (++i >= a.n) return false;  // (x < end: a row with tiles follows, unless lengths change meanwhile)
            nt = row_tiles(a, i, slot, len, e);
            rem = 0;
        }
        unit = static_cast<int>(rem / nt);
        t0 = static_cast<int>(rem - static_cast<long long>(unit) * nt);
        t1 = static_cast<int>(min(static_cast<long long>(nt), t0 + (end - x)));
        unit_start = x - t0;
        x += t1 - t0;
        rem += t1 - t0;
        return true;
    }
};

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <bool BF16, int DCH>
__global__ void __launch_bounds__(kDecodeThreads, 2)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs a) {
    using Cfg = DecodeCfg<DCH>;
    extern __shared__ uint8_t raw[];
    __shared__ DecodeShared sh;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sq = ring + kDecodeStages * Cfg::kStage;
    uint8_t* sp = sq + 2 * kUnitRows * kQPitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &sh.abort;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kDecodeStages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], 4);
        }
        fence_mbar_init();
        sh.abort = 0;
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    grid_dependency_wait();

    // All tiles, this CTA's part of them, and the row where it begins. Four rows a thread and pass.
    const int units = a.kv_heads * a.chunks;
    uint32_t err = 0;
    auto pass = [&](int i0, long long (&w)[4]) {
        long long s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 4 * static_cast<int>(threadIdx.x) + j;
            int slot, len;
            w[j] = i < a.n ? static_cast<long long>(row_tiles(a, i, slot, len, err)) * units : 0;
            s += w[j];
        }
        return s;
    };
    auto block_prefix = [&](long long v, long long& total) {  // exclusive, over the block
        long long p = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) p += y;
        }
        __syncthreads();
        if (lane == 31) sh.scan[warp] = p;
        __syncthreads();
        long long pre = 0;
        total = 0;
#pragma unroll
        for (int k = 0; k < kDecodeThreads / 32; ++k) {
            if (k < warp) pre += sh.scan[k];
            total += sh.scan[k];
        }
        return pre + p - v;
    };
    constexpr int kStep = 4 * kDecodeThreads;
    long long w[4], total = 0, sum = 0, pre = 0;
    for (int i0 = 0; i0 < a.n; i0 += kStep) {
        sum = pass(i0, w);
        long long t;
        pre = block_prefix(sum, t);
        total += t;
    }
    if (err != 0 && blockIdx.x == 0) atomicOr(a.err, err);
    const long long ctas = min(static_cast<long long>(gridDim.x), total);
    if (blockIdx.x >= ctas) return;
    auto bound = [&](long long c) { return c * total / ctas; };
    const long long x0 = bound(blockIdx.x), x1 = bound(blockIdx.x + 1);
    long long before = 0;
    for (int i0 = 0; i0 < a.n; i0 += kStep) {
        if (a.n > kStep) {  // (otherwise the first pass' values are still there)
            sum = pass(i0, w);
            long long t;
            pre = block_prefix(sum, t) + before;
            before += t;
        }
        long long at = pre;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (at <= x0 && x0 < at + w[j]) {
                sh.start_row = i0 + 4 * static_cast<int>(threadIdx.x) + j;
                sh.start_before = at;
            }
            at += w[j];
        }
    }
    __syncthreads();
    Walk walk;
    walk.begin(a, x0, x1, sh.start_row, sh.start_before);
    const long long limit = a.timeout_cycles;

    if (warp == 4) {
        // ---------------------------------------------------------------- loads
        const int pieces = kTokens / a.box;  // at most 8
        const long long drain = limit > kDecodeDrain ? limit : kDecodeDrain;
        uint32_t it = 0, seg = 0;
        bool ok = true;
        while (ok && walk.next(a)) {
            const int head = walk.unit / a.chunks, chunk = walk.unit - head * a.chunks;
            const int rows = min(kUnitRows, a.group - chunk * kUnitRows);
            const int32_t* table = a.table + static_cast<long long>(walk.slot) * a.max_pages;
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sh.q_empty[seg & 1], ((seg >> 1) & 1) ^ 1, abort_flag, limit));
            if (!ok) break;
            const uint32_t row_bytes = a.head_dim * 2;
            if (lane == 0) mbar_arrive_expect_tx(&sh.q_full[seg & 1], rows * row_bytes);
            __syncwarp();
            if (lane < rows)
                bulk_load(sq + (seg & 1) * kUnitRows * kQPitch + lane * kQPitch,
                          a.q + static_cast<long long>(walk.i) * a.q_seq +
                              static_cast<long long>(head * a.group + chunk * kUnitRows + lane) * a.q_head,
                          row_bytes, &sh.q_full[seg & 1]);
            ++seg;
            // lane p < pieces loads piece p of every tile; its page is looked up one tile ahead
            auto lookup = [&](int t) {
                const long long tok = static_cast<long long>(t) * kTokens + lane * a.box;
                return lane < pieces && tok < walk.len ? table[tok / a.page_size] : -1;
            };
            int page = lookup(walk.t0);
            for (int t = walk.t0; t < walk.t1; ++t, ++it) {
                const int s = it % kDecodeStages;
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&sh.empty[s], ((it / kDecodeStages) & 1) ^ 1, abort_flag, limit));
                if (!ok) break;
                const int tok = t * kTokens + lane * a.box;
                const bool mine = lane < pieces && tok < walk.len;
                const int count = __popc(__ballot_sync(0xffffffffu, mine));
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[s], count * a.box * 256 * DCH);
                __syncwarp();
                int p = page;
                if (mine && (p < 0 || p >= a.num_pages)) {  // refused, but the copies that were announced are made
                    atomicOr(a.err, DEV_ERR_INDEX);
                    p = 0;
                }
                if (t + 1 < walk.t1) page = lookup(t + 1);
                if (mine) {
                    const int row = (p * a.kv_heads + head) * a.page_size + tok % a.page_size;
                    uint8_t* k = ring + s * Cfg::kStage + lane * a.box * 128;
#pragma unroll
                    for (int c = 0; c < DCH; ++c) {
                        tma_load_2d(k + c * kTokens * 128, &tmK, &sh.full[s], 64 * c, row);
                        tma_load_2d(k + Cfg::kTensor + c * kTokens * 128, &tmV, &sh.full[s], 64 * c, row);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) {
            atomicOr(a.err, DEV_ERR_TIMEOUT);
            *abort_flag = 1;
        }
        // every issued load lands before the CTA may exit
        for (uint32_t i = it > kDecodeStages ? it - kDecodeStages : 0; i < it; ++i)
            mbar_wait_bounded(&sh.full[i % kDecodeStages], (i / kDecodeStages) & 1, nullptr, drain);
        for (uint32_t i = seg > 2 ? seg - 2 : 0; i < seg; ++i)
            mbar_wait_bounded(&sh.q_full[i & 1], (i >> 1) & 1, nullptr, drain);
        return;
    }

    // -------------------------------------------------------------------- arithmetic
    // A wait that gives up raises the abort flag and the warp goes on without its data (later waits
    // return at once), so the four warps always meet at the same barriers.
    auto wait = [&](uint64_t* bar, uint32_t ph) {
        if (!mbar_wait_bounded(bar, ph, abort_flag, limit) && *abort_flag == 0) {
            atomicOr(a.err, DEV_ERR_TIMEOUT);
            *abort_flag = 1;
        }
        __syncwarp();
    };
    const int ksteps = a.head_dim / 16;
    const int r0 = lane >> 2, cpair = 2 * (lane & 3), mat = lane >> 3, mrow = lane & 7;
    uint32_t it = 0, seg = 0;
    while (walk.next(a)) {
        const int head = walk.unit / a.chunks, chunk = walk.unit - head * a.chunks;
        const int rows = min(kUnitRows, a.group - chunk * kUnitRows);
        // Q fragments
        uint32_t qf[4 * DCH][4];
        wait(&sh.q_full[seg & 1], (seg >> 1) & 1);
        {
            const uint32_t qa = smem_u32(sq + (seg & 1) * kUnitRows * kQPitch) + ((mat & 1) * 8 + mrow) * kQPitch + (mat >> 1) * 16;
#pragma unroll
            for (int k = 0; k < 4 * DCH; ++k) {
                if (k < ksteps) ldmatrix_x4(qa + k * 32, qf[k]);
                if (r0 >= rows) qf[k][0] = qf[k][2] = 0;
                if (r0 + 8 >= rows) qf[k][1] = qf[k][3] = 0;
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_empty[seg & 1]);
        ++seg;
        float o[DCH][2][4] = {};        // head_dim pairs of 8: pair warp + 4 c
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        for (int t = walk.t0; t < walk.t1; ++t, ++it) {
            const int s = it % kDecodeStages;
            const uint32_t kb = smem_u32(ring + s * Cfg::kStage), vb = kb + Cfg::kTensor;
            wait(&sh.full[s], (it / kDecodeStages) & 1);
            // scores of this warp's 16 keys
            float c[2][4] = {};
            {
                const int tok = 16 * warp + (mat >> 1) * 8 + mrow;
                const uint32_t ka = kb + tok * 128;
#pragma unroll
                for (int k = 0; k < 4 * DCH; ++k) {
                    if (k < ksteps) {
                        uint32_t b[4];
                        const int v = (2 * k + (mat & 1)) & 7;
                        ldmatrix_x4(ka + (k >> 2) * (kTokens * 128) + ((v ^ (tok & 7)) << 4), b);
                        mma_16816<BF16>(c[0], qf[k], b[0], b[1]);
                        mma_16816<BF16>(c[1], qf[k], b[2], b[3]);
                    }
                }
            }
            const int live = walk.len - t * kTokens;  // keys of the tile that exist
            if (live < kTokens) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * warp + 8 * j + cpair + (e & 1) >= live) c[j][e] = -INFINITY;
            }
            float t0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
            float t1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
            if ((lane & 3) == 0) {
                sh.top[warp][r0] = t0;
                sh.top[warp][r0 + 8] = t1;
            }
            consumer_sync();
            t0 = fmaxf(fmaxf(sh.top[0][r0], sh.top[1][r0]), fmaxf(sh.top[2][r0], sh.top[3][r0])) * a.scale_log2;
            t1 = fmaxf(fmaxf(sh.top[0][r0 + 8], sh.top[1][r0 + 8]), fmaxf(sh.top[2][r0 + 8], sh.top[3][r0 + 8])) * a.scale_log2;
            const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
            const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
            const float f0 = exp2_fast(m0 - b0), f1 = exp2_fast(m1 - b1);
            m0 = n0;
            m1 = n1;
            l0 *= f0;
            l1 *= f1;
            uint8_t* pw = sp + r0 * kPPitch + (16 * warp + cpair) * 2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float u0 = exp2_fast(fmaf(c[j][0], a.scale_log2, -b0)), u1 = exp2_fast(fmaf(c[j][1], a.scale_log2, -b0));
                const float w0 = exp2_fast(fmaf(c[j][2], a.scale_log2, -b1)), w1 = exp2_fast(fmaf(c[j][3], a.scale_log2, -b1));
                l0 += u0 + u1;
                l1 += w0 + w1;
                *reinterpret_cast<uint32_t*>(pw + 16 * j) = pack2<BF16>(u0, u1);
                *reinterpret_cast<uint32_t*>(pw + 8 * kPPitch + 16 * j) = pack2<BF16>(w0, w1);
            }
#pragma unroll
            for (int d = 0; d < DCH; ++d)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    o[d][j][0] *= f0;
                    o[d][j][1] *= f0;
                    o[d][j][2] *= f1;
                    o[d][j][3] *= f1;
                }
            consumer_sync();
            // O += P V over all 64 keys, this warp's part of head_dim
            const uint32_t pa = smem_u32(sp) + ((mat & 1) * 8 + mrow) * kPPitch + (mat >> 1) * 16;
#pragma unroll
            for (int k = 0; k < kTokens / 16; ++k) {
                uint32_t p[4];
                ldmatrix_x4(pa + k * 32, p);
                const int tok = 16 * k + (mat & 1) * 8 + mrow;
                // keys past the end have weight 0, but what lies in their place may be NaN
                const int left = live - 16 * k - cpair;
                const uint32_t lo = left >= 2 ? 0xFFFFFFFFu : (left == 1 ? 0x0000FFFFu : 0u);
                const uint32_t hi = left >= 10 ? 0xFFFFFFFFu : (left == 9 ? 0x0000FFFFu : 0u);
#pragma unroll
                for (int d = 0; d < DCH; ++d) {
                    const int pair = warp + 4 * d;
                    if (pair < ksteps) {
                        uint32_t b[4];
                        const int v = (2 * pair + (mat >> 1)) & 7;
                        ldmatrix_x4_trans(vb + (pair >> 2) * (kTokens * 128) + tok * 128 + ((v ^ (tok & 7)) << 4), b);
                        mma_16816<BF16>(o[d][0], p, b[0] & lo, b[1] & hi);
                        mma_16816<BF16>(o[d][1], p, b[2] & lo, b[3] & hi);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.empty[s]);
        }
        // the sum of weights over the quad and the four warps
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if ((lane & 3) == 0) {
            sh.sum[warp][r0] = l0;
            sh.sum[warp][r0 + 8] = l1;
        }
        consumer_sync();
        l0 = (sh.sum[0][r0] + sh.sum[1][r0]) + (sh.sum[2][r0] + sh.sum[3][r0]);
        l1 = (sh.sum[0][r0 + 8] + sh.sum[1][r0 + 8]) + (sh.sum[2][r0 + 8] + sh.sum[3][r0 + 8]);
        const int qh = head * a.group + chunk * kUnitRows;  // the unit's first query head
        uint16_t* out = a.out + static_cast<long long>(walk.i) * a.o_seq + static_cast<long long>(qh) * a.o_head;
        float* lse = a.lse ? a.lse + static_cast<long long>(walk.i) * a.q_heads + qh : nullptr;
        const bool any = walk.len > 0;
        if (walk.t0 == 0 && walk.t1 == walk.nt) {
            const float i0 = any ? 1.f / l0 : 0.f, i1 = any ? 1.f / l1 : 0.f;
#pragma unroll
            for (int d = 0; d < DCH; ++d) {
                const int pair = warp + 4 * d;
                if (pair >= ksteps) continue;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int col = 16 * pair + 8 * j + cpair;
                    if (r0 < rows)
                        *reinterpret_cast<uint32_t*>(out + r0 * a.o_head + col) = any ? pack2<BF16>(o[d][j][0] * i0, o[d][j][1] * i0) : 0u;
                    if (r0 + 8 < rows)
                        *reinterpret_cast<uint32_t*>(out + (r0 + 8) * a.o_head + col) = any ? pack2<BF16>(o[d][j][2] * i1, o[d][j][3] * i1) : 0u;
                }
            }
            if (lse != nullptr && warp == 0 && (lane & 3) == 0) {
                if (r0 < rows) lse[r0] = any ? ((m0 == -INFINITY ? 0.f : m0) + log2f(l0)) * kLn2 : -INFINITY;
                if (r0 + 8 < rows) lse[r0 + 8] = any ? ((m1 == -INFINITY ? 0.f : m1) + log2f(l1)) * kLn2 : -INFINITY;
            }
            continue;
        }
        // A part of a unit. Parts that begin a unit lie in a CTA's second place, others in its first.
        auto cta_of = [&](long long x) { return ((x + 1) * ctas - 1) / total; };
        const long long c0 = cta_of(walk.unit_start), c1 = cta_of(walk.unit_start + walk.nt - 1);
        const long long place = 2ll * blockIdx.x + (walk.t0 == 0 ? 1 : 0);
        float* po = a.part_o + place * kUnitRows * a.head_dim;
#pragma unroll
        for (int d = 0; d < DCH; ++d) {
            const int pair = warp + 4 * d;
            if (pair >= ksteps) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = 16 * pair + 8 * j + cpair;
                if (r0 < rows) *reinterpret_cast<float2*>(po + r0 * a.head_dim + col) = make_float2(o[d][j][0], o[d][j][1]);
                if (r0 + 8 < rows) *reinterpret_cast<float2*>(po + (r0 + 8) * a.head_dim + col) = make_float2(o[d][j][2], o[d][j][3]);
            }
        }
        if (warp == 0 && (lane & 3) == 0) {
            a.part_ml[place * kUnitRows + r0] = make_float2(m0, l0);
            a.part_ml[place * kUnitRows + r0 + 8] = make_float2(m1, l1);
        }
        __threadfence();
        consumer_sync();
        if (threadIdx.x == 0) {
            const uint32_t parts = static_cast<uint32_t>(c1 - c0 + 1);
            const bool last = atomicAdd(a.arrived + c0, 1u) == parts - 1;
            if (last) a.arrived[c0] = 0;  // nobody else of this call comes here any more
            sh.last = last;
            __threadfence();
        }
        consumer_sync();
        if (sh.last) {
            // the parts in the order of the keys: c0's second place, the others' first
            const int vecs = a.head_dim / 4;
            for (int e = threadIdx.x; e < rows * vecs; e += kConsumers) {
                const int row = e / vecs, v = e - row * vecs;
                float m = -INFINITY, l = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                for (long long c = c0; c <= c1; c += 4) {
                    float2 ml[4];
                    float4 x[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (c + j > c1) continue;
                        const long long from = 2 * (c + j) + (c + j == c0 ? 1 : 0);
                        ml[j] = __ldcg(a.part_ml + from * kUnitRows + row);
                        x[j] = __ldcg(reinterpret_cast<const float4*>(a.part_o + (from * kUnitRows + row) * a.head_dim) + v);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (c + j > c1) continue;
                        const float mm = fmaxf(m, ml[j].x), b = mm == -INFINITY ? 0.f : mm;
                        const float f = exp2_fast(m - b), g = exp2_fast(ml[j].x - b);
                        m = mm;
                        l = l * f + ml[j].y * g;
                        acc.x = acc.x * f + x[j].x * g;
                        acc.y = acc.y * f + x[j].y * g;
                        acc.z = acc.z * f + x[j].z * g;
                        acc.w = acc.w * f + x[j].w * g;
                    }
                }
                const float inv = 1.f / l;  // (a unit in parts has tokens)
                *reinterpret_cast<uint2*>(out + row * a.o_head + 4 * v) =
                    make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
                if (lse != nullptr && v == 0) lse[row] = ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2;
            }
        }
        consumer_sync();  // sh.last and sh.sum are free again
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

static int box_rows(int page_size) {  // the greatest common divisor of 64 and the page size (a multiple of 8)
    int r = 64;
    while (page_size % r) r /= 2;
    return r;
}

tb_status decode_create(tb_cache* c) {
    const tb_cache_desc& d = c->d;
    c->decode_ctas = 2 * c->ctx->num_sms;
    const size_t places = 2 * static_cast<size_t>(c->decode_ctas);
    TB_CUDA(cudaMalloc(&c->part_o, places * kUnitRows * d.head_dim * sizeof(float)));
    TB_CUDA(cudaMalloc(&c->part_ml, places * kUnitRows * sizeof(float2)));
    TB_CUDA(cudaMalloc(&c->arrived, c->decode_ctas * sizeof(uint32_t)));
    TB_CUDA(cudaMemset(c->arrived, 0, c->decode_ctas * sizeof(uint32_t)));
    const uint64_t rows = static_cast<uint64_t>(d.num_pages) * d.kv_heads * d.page_size;
    const uint64_t dims[2] = {static_cast<uint64_t>(d.head_dim), rows};
    const uint64_t stride[1] = {static_cast<uint64_t>(d.head_dim) * 2};
    const uint32_t box[2] = {64, static_cast<uint32_t>(box_rows(d.page_size))};
    const CUtensorMapDataType type = d.dtype == TB_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    c->k_map.resize(d.layers);
    c->v_map.resize(d.layers);
    for (int l = 0; l < d.layers; ++l) {
        const size_t at = static_cast<size_t>(l) * rows * d.head_dim * 2;
        TB_TRY(encode_tiled(&c->k_map[l], type, 2, static_cast<const char*>(c->b.k_pages) + at, dims, stride, box, CU_TENSOR_MAP_SWIZZLE_128B));
        TB_TRY(encode_tiled(&c->v_map[l], type, 2, static_cast<const char*>(c->b.v_pages) + at, dims, stride, box, CU_TENSOR_MAP_SWIZZLE_128B));
    }
    return TB_OK;
}

void decode_destroy(tb_cache* c) {
    if (c->part_o) cudaFree(c->part_o);
    if (c->part_ml) cudaFree(c->part_ml);
    if (c->arrived) cudaFree(c->arrived);
}

template <bool BF16, int DCH>
static tb_status launch_decode(tb_cache* c, int layer, const DecodeArgs& a, cudaStream_t st) {
    auto* kernel = decode_kernel<BF16, DCH>;
    static bool ready = false;  // the attribute is per function and process-wide
    if (!ready) {
        TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeCfg<DCH>::kSmem));
        ready = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(c->decode_ctas));
    cfg.blockDim = dim3(kDecodeThreads);
    cfg.dynamicSmemBytes = DecodeCfg<DCH>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA(cudaLaunchKernelEx(&cfg, kernel, c->k_map[layer], c->v_map[layer], a));
    c->ctx->launches++;
    return TB_OK;
}

}  // namespace tb

using namespace tb;

extern "C" {

TB_API tb_status tb_cache_attend(tb_cache* c, int32_t layer, const int32_t* slots, int32_t n, int32_t q_heads,
                                 float scale, const void* q, int64_t q_seq_stride, int64_t q_head_stride, void* out,
                                 int64_t out_seq_stride, int64_t out_head_stride, float* lse, void* stream) {
    if (!c) return fail(TB_ERR_INVALID_ARGUMENT, "cache attend: null cache");
    const tb_cache_desc& d = c->d;
    TB_TRY(attention_check("cache attend", d.dtype, q_heads, d.kv_heads, d.head_dim, scale));
    if (layer < 0 || layer >= d.layers) return fail(TB_ERR_SHAPE_MISMATCH, "cache attend: layer %d of %d", layer, d.layers);
    if (n < 0) return fail(TB_ERR_SHAPE_MISMATCH, "cache attend: negative count");
    if (n > 65535 || q_heads > 4096) return fail(TB_ERR_NOT_ACCELERATED, "cache attend: more than 65535 rows or 4096 heads");
    if (n == 0) return TB_OK;
    if (!slots || !q || !out) return fail(TB_ERR_INVALID_ARGUMENT, "cache attend: null pointer");
    if (q_seq_stride < 0 || q_head_stride < 0 || out_seq_stride < 0 || out_head_stride < 0)
        return fail(TB_ERR_SHAPE_MISMATCH, "cache attend: negative stride");
    if (!aligned16(q) || !aligned16(out) || ((q_seq_stride | q_head_stride | out_seq_stride | out_head_stride) & 7))
        return fail(TB_ERR_INVALID_ARGUMENT, "cache attend: tensors must be 16-byte aligned with strides that are multiples of 8");
    const int group = q_heads / d.kv_heads;
    DecodeArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    a.slots = slots;
    a.table = c->b.page_table;
    a.lengths = c->b.lengths;
    a.q_seq = q_seq_stride;
    a.q_head = q_head_stride;
    a.o_seq = out_seq_stride;
    a.o_head = out_head_stride;
    a.n = n;
    a.q_heads = q_heads;
    a.kv_heads = d.kv_heads;
    a.group = group;
    a.chunks = (group + kUnitRows - 1) / kUnitRows;
    a.head_dim = d.head_dim;
    a.page_size = d.page_size;
    a.num_pages = d.num_pages;
    a.max_seqs = d.max_seqs;
    a.max_pages = d.max_pages;
    a.box = box_rows(d.page_size);
    a.scale_log2 = scale * kLog2e;
    a.part_o = c->part_o;
    a.part_ml = c->part_ml;
    a.arrived = c->arrived;
    a.err = c->ctx->dev_err;
    a.timeout_cycles = c->ctx->timeout_cycles;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool wide = d.head_dim > 64;
    if (d.dtype == TB_DT_BF16)
        return wide ? launch_decode<true, 2>(c, layer, a, st) : launch_decode<true, 1>(c, layer, a, st);
    return wide ? launch_decode<false, 2>(c, layer, a, st) : launch_decode<false, 1>(c, layer, a, st);
}

}  // extern "C"
