// Attention of one new token a sequence over the paged cache.
//
// The formula is attention.cu's with one row a sequence. For groups of up to 16 query heads a key head every key and
// value is read once and used for that group only, so the kernel is bound by memory bandwidth: its work is cut so that
// every SM streams the same amount, and the arithmetic only has to keep up. Keys and dimensions take the long side of
// mma.sync's 16 x 8 x 16 and the query rows the short one: a unit's rows are padded to 8, or to 16 in groups above 8.
// (A group above 16 is several units, each of which asks for its keys again.)
//
// Cut: a unit is one sequence, key head and at most 8 (for groups above 8: 16) of its query heads; its keys
// come in tiles of 64 tokens. The tiles of all units in a row are divided evenly over the CTAs (two on each
// SM), so a CTA takes the end of one unit, some whole units and the beginning of another. A unit that lies in
// one CTA is finished there. Of a unit that several CTAs share, each leaves its unscaled sum, maximum and sum
// of weights, and the CTA that arrives last adds them in the order of the keys: the result does not depend
// on who that is. (It does depend, in its last bits, on where the cuts fall, that is on the lengths of the
// whole batch.) Nobody waits for another CTA.
//
// A CTA: warp 4 looks the pages up and loads K and V tiles by TMA (boxes as high as the greatest common
// divisor of 64 and the page size, so that a box never crosses a page) and the query rows, as many tiles
// ahead as the ring holds (96 KB). Warps 0-3 take 16 of a tile's 64 keys each for S^T = K Q^T, share the
// maximum and the weights through shared memory, and take a quarter of head_dim each for
// O^T += V^T P^T: two barriers a tile, and nothing to join among the warps when the CTA leaves a unit
// (warps with a maximum and a result of their own need no barriers, but joining them made 32 contexts
// of up to 1023 tokens of 32 heads 29.6 us instead of 24.7). Tiles of heads of at most 64 are half as large
// and share two barriers in pairs while a CTA's part of a unit has two (98 contexts of 5678 tokens, one head:
// 34.2 -> 31.5 us; 8 of 4000 to 20000, 16 heads to each of 4 key heads: 29.6 -> 26.9). Tiles of 128 keys
// instead cut short contexts too coarsely (40 of up to 300 tokens 7.3 -> 7.9 us).
//
// Measured: 64 contexts of up to 16384 tokens (8 key heads of 128, 1.66 GB) 247 us = 6.7 TB/s; two of 20 to 30
// thousand (216 MB) 43.6 us = 5.0 TB/s: of some 63,000 cycles of a CTA its first tile's arrival takes 9,500 (slot,
// length, page, tile one after the other) and its result 3,000; the 32 short ones (73 MB) 22.2 us, bound by the
// latency of the units that a CTA goes through (one of two tiles takes some 6,000 cycles).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attention.cuh"
#include "cache.hpp"
#include "ptx.cuh"
#include "quant.cuh"

namespace tb {

constexpr int kTokens = 64;                    // keys of a tile
constexpr int kUnitRows = 16;                  // query rows of a unit at most
constexpr int kConsumers = 128;
constexpr int kDecodeThreads = kConsumers + 32;
constexpr int kQPitch = 272;                   // bytes from one query row to the next: 8 rows hit 8 bank groups
constexpr long long kDecodeDrain = 2000000000ll;  // bound on a CTA's waits for its own copies at its end

template <int DCH>
struct DecodeCfg {
    static constexpr int kTensor = DCH * kTokens * 128;  // K or V of a tile, 64-element chunks of 128-byte rows, swizzled
    static constexpr int kStage = 2 * kTensor;
    static constexpr int kStages = DCH == 2 ? 3 : 6;
    static constexpr int kAtOnce = DCH == 2 ? 1 : 2;     // tiles between two barriers at most
    static constexpr int kPPitch = kAtOnce * kTokens * 2 + 16;  // bytes of one row of weights: 8 rows hit 8 bank groups
    static constexpr int kSmem = 1024 + kStages * kStage + kUnitRows * kQPitch + kUnitRows * kPPitch;
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
    uint64_t full[6], empty[6], q_full[4], q_empty[4];
    float top[4][kUnitRows], sum[4][kUnitRows];
    int abort, last;
};

// Tiles of a row's units, 0 when the row is refused. A row without tokens has one empty tile.
__device__ __forceinline__ bool row_ok(const DecodeArgs& a, int slot, int len) {
    return slot >= 0 && slot < a.max_seqs && len >= 0 && static_cast<long long>(len) <= static_cast<long long>(a.max_pages) * a.page_size;
}
__device__ __forceinline__ int row_tiles(int len) { return max(1, (len + kTokens - 1) / kTokens); }

// a / b for a >= 0, b > 0; nearly always of 32 bits, where a division is ten times as fast.
__device__ __forceinline__ long long quotient(long long a, long long b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// This CTA's tiles, segment by segment: tiles [t0, t1) of one unit.
struct Walk {
    long long x, end;        // the next tile and the end of the CTA's
    int i, nt, len, slot;    // row, tiles of each of its units, tokens
    int unit, t0, t1;
    long long unit_start;    // the unit's first tile
    // From tile x0, which is `rem` tiles into row i's units.
    __device__ void begin(long long x0, long long x1, int row, int row_slot, int row_len, long long rem) {
        x = x0;
        end = x1;
        i = row;
        slot = row_slot;
        len = row_len;
        nt = row_tiles(len);
        unit = static_cast<int>(quotient(rem, nt));
        t1 = static_cast<int>(rem - static_cast<long long>(unit) * nt);
    }
    __device__ bool next(const DecodeArgs& a) {
        if (x >= end) return false;
        if (t1 == nt) {
            t1 = 0;
            ++unit;
        }
        t0 = t1;
        if (unit == a.kv_heads * a.chunks) {
            unit = 0;
            do {
                if (++i >= a.n) return false;  // (x < end: a row with tiles follows, unless lengths change meanwhile)
                slot = a.slots[i];
                len = a.lengths[min(max(slot, 0), a.max_seqs - 1)];
            } while (!row_ok(a, slot, len));
            nt = row_tiles(len);
        }
        t1 = static_cast<int>(min(static_cast<long long>(nt), t0 + (end - x)));
        unit_start = x - t0;
        x += t1 - t0;
        return true;
    }
};

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// NT: query rows of a unit / 8.
template <bool BF16, int DCH, int NT>
__global__ void __launch_bounds__(kDecodeThreads, 2)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs a) {
    using Cfg = DecodeCfg<DCH>;
    constexpr int S = Cfg::kStages, kPPitch = Cfg::kPPitch;
    extern __shared__ uint8_t raw[];
    __shared__ DecodeShared sh;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sq = ring + S * Cfg::kStage;
    uint8_t* sp = sq + kUnitRows * kQPitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &sh.abort;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 4);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], 4);
        }
        fence_mbar_init();
        sh.abort = 0;
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();

    __syncthreads();  // the barriers are made
    // All tiles, this CTA's part of them, and the row where it begins: each warp for itself, four rows a
    // lane and pass, so that no barrier stands before the first load.
    const int units = a.kv_heads * a.chunks;
    uint32_t err = 0;
    int slot[4], len[4];
    long long w[4];
    auto pass = [&](int i0) {  // tiles of the lane's four rows, before it (exclusive) and of the warp's 128
        const int i = i0 + 4 * lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) slot[j] = i + j < a.n ? a.slots[i + j] : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) len[j] = a.lengths[min(max(slot[j], 0), a.max_seqs - 1)];
        long long sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool ok = row_ok(a, slot[j], len[j]);
            w[j] = i + j < a.n && ok ? static_cast<long long>(row_tiles(len[j])) * units : 0;
            if (i + j < a.n && !ok) err |= DEV_ERR_INDEX;
            sum += w[j];
        }
        long long p = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) p += y;
        }
        return longlong2{p - sum, __shfl_sync(0xffffffffu, p, 31)};
    };
    constexpr int kStep = 128;
    longlong2 part{0, 0};
    long long total = 0;
    for (int i0 = 0; i0 < a.n; i0 += kStep) {
        part = pass(i0);
        total += part.y;
    }
    if (err != 0 && blockIdx.x == 0) atomicOr(a.err, err);
    // one tile a CTA is enough: 2 and 3 at least made one user's 333 tokens 6.9 and 7.6 us instead of 6.4
    const long long ctas = min(static_cast<long long>(gridDim.x), total);
    if (blockIdx.x >= ctas) return;
    // the first `longer` CTAs take share + 1 tiles, the others share
    const long long share = quotient(total, ctas), longer = total - share * ctas;
    auto bound = [&](long long c) { return c * share + min(c, longer); };
    auto cta_of = [&](long long x) {
        const long long split = longer * (share + 1);
        return x < split ? quotient(x, share + 1) : longer + quotient(x - split, share);
    };
    const long long x0 = bound(blockIdx.x), x1 = bound(blockIdx.x + 1ll);
    Walk walk;
    {
        long long before = 0;
        for (int i0 = 0; i0 < a.n; i0 += kStep) {
            if (a.n > kStep) part = pass(i0);  // (otherwise the first pass' values are still there)
            if (x0 < before + part.y) {
                long long at = before + part.x;
                int j0 = 0;
                bool here = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!here) {
                        if (at <= x0 && x0 < at + w[j]) {
                            here = true;
                            j0 = j;
                        } else {
                            at += w[j];
                        }
                    }
                }
                const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
                const int row_slot = j0 == 0 ? slot[0] : (j0 == 1 ? slot[1] : (j0 == 2 ? slot[2] : slot[3]));
                const int row_len = j0 == 0 ? len[0] : (j0 == 1 ? len[1] : (j0 == 2 ? len[2] : len[3]));
                walk.begin(x0, x1, __shfl_sync(0xffffffffu, i0 + 4 * lane + j0, from), __shfl_sync(0xffffffffu, row_slot, from),
                           __shfl_sync(0xffffffffu, row_len, from), x0 - __shfl_sync(0xffffffffu, at, from));
                break;
            }
            before += part.y;
        }
    }
    const long long limit = a.timeout_cycles;
    // Query rows of the segments under way: 1, 2 or 4 of them in the 16-row buffer.
    const int q_slots = NT > 1 ? 1 : (a.group > 4 ? 2 : 4), q_step = kUnitRows / q_slots * kQPitch;

    if (warp == 4) {
        // ---------------------------------------------------------------- loads
        const int pieces = kTokens / a.box;  // at most 8
        const long long drain = limit > kDecodeDrain ? limit : kDecodeDrain;
        // A place in the ring or of the query rows is free. Warps 0-3 release places without their data when they have given
        // up; the abort flag, raised before, then tells that a copy may still be on its way there, and that its barrier
        // must not be armed once more.
        auto free_place = [&](uint64_t* bar, uint32_t ph) {
            return __all_sync(0xffffffffu, mbar_wait_bounded(bar, ph, abort_flag, limit) && *abort_flag == 0) != 0;
        };
        uint32_t it = 0, seg = 0;
        bool ok = true;
        while (ok && walk.next(a)) {
            const int head = walk.unit / a.chunks, chunk = walk.unit - head * a.chunks;
            const int rows = min(8 * NT, a.group - chunk * 8 * NT);
            const int32_t* table = a.table + static_cast<long long>(walk.slot) * a.max_pages;
            // lane p < pieces loads piece p of every tile; its page and its place there are found one tile ahead (one
            // division for both: pages of 8 tokens 40.2 -> 39.0 us, though 16 contexts in pages of 16 20.3 -> 20.7)
            int inside = 0;  // the piece's first token in its page
            auto lookup = [&](int t) {
                const int tok = t * kTokens + lane * a.box;
                const int at = tok / a.page_size;
                inside = tok - at * a.page_size;
                return lane < pieces && tok < walk.len ? table[at] : -1;
            };
            int page = lookup(walk.t0);
            const int qs = seg & (q_slots - 1);
            ok = free_place(&sh.q_empty[qs], ((seg / q_slots) & 1) ^ 1);
            if (!ok) break;
            const uint32_t row_bytes = a.head_dim * 2;
            if (lane == 0) mbar_arrive_expect_tx(&sh.q_full[qs], rows * row_bytes);
            __syncwarp();
            if (lane < rows)
                bulk_load(sq + qs * q_step + lane * kQPitch,
                          a.q + static_cast<long long>(walk.i) * a.q_seq +
                              static_cast<long long>(head * a.group + chunk * 8 * NT + lane) * a.q_head,
                          row_bytes, &sh.q_full[qs]);
            ++seg;
            for (int t = walk.t0; t < walk.t1; ++t, ++it) {
                const int s = it % S;
                ok = free_place(&sh.empty[s], ((it / S) & 1) ^ 1);
                if (!ok) break;
                const int tok = t * kTokens + lane * a.box;
                const bool mine = lane < pieces && tok < walk.len;
                const int count = __popc(__ballot_sync(0xffffffffu, mine));
                if (lane == 0) mbar_arrive_expect_tx(&sh.full[s], count * a.box * 256 * DCH);
                __syncwarp();
                int p = page;
                const int row0 = inside;
                if (mine && (p < 0 || p >= a.num_pages)) {  // refused, but the copies that were announced are made
                    atomicOr(a.err, DEV_ERR_INDEX);
                    p = 0;
                }
                if (t + 1 < walk.t1) page = lookup(t + 1);
                if (mine) {
                    const int row = (p * a.kv_heads + head) * a.page_size + row0;
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
        for (uint32_t i = it > S ? it - S : 0; i < it; ++i)
            mbar_wait_bounded(&sh.full[i % S], (i / S) & 1, nullptr, drain);
        for (uint32_t i = seg > static_cast<uint32_t>(q_slots) ? seg - q_slots : 0; i < seg; ++i)
            mbar_wait_bounded(&sh.q_full[i & (q_slots - 1)], (i / q_slots) & 1, nullptr, drain);
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
        const int rows = min(8 * NT, a.group - chunk * 8 * NT);
        // Q^T as right operands
        uint32_t qf[NT][4 * DCH][2];
        const int qs = seg & (q_slots - 1);
        wait(&sh.q_full[qs], (seg / q_slots) & 1);
#pragma unroll
        for (int h = 0; h < NT; ++h) {
            // (rows past the unit's are whatever lies there, and are set to 0)
            const uint32_t qa = smem_u32(sq) + qs * q_step + (8 * h + mrow) * kQPitch + mat * 16;
#pragma unroll
            for (int k = 0; k < 4 * DCH; k += 2) {
                uint32_t b[4] = {0, 0, 0, 0};
                if (k < ksteps) ldmatrix_x4(qa + k * 32, b);
                const bool row = 8 * h + r0 < rows;
                qf[h][k][0] = row ? b[0] : 0u;
                qf[h][k][1] = row ? b[1] : 0u;
                qf[h][k + 1][0] = row ? b[2] : 0u;
                qf[h][k + 1][1] = row ? b[3] : 0u;
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_empty[qs]);
        ++seg;
        float o[DCH][NT][4] = {};       // O^T: 16 dimensions by 8 rows each, dimensions 16 (warp + 4 d)
        float m[NT][2], l[NT][2];       // of rows 8 h + cpair and the next
#pragma unroll
        for (int h = 0; h < NT; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[h][e] = -INFINITY;
                l[h][e] = 0.f;
            }
        // `tiles` tiles of the ring from tile t on
        auto step = [&](int t, auto tiles) {
            constexpr int T = decltype(tiles)::value;
            uint32_t kb[T];
#pragma unroll
            for (int u = 0; u < T; ++u) {
                const int s = (it + u) % S;
                kb[u] = smem_u32(ring + s * Cfg::kStage);
                wait(&sh.full[s], ((it + u) / S) & 1);
            }
            const int live = walk.len - t * kTokens;  // keys from the first tile's start that exist
            float c[NT][T][4] = {}, d[NT][T][4] = {};
#pragma unroll
            for (int u = 0; u < T; ++u) {
                const int tok = 16 * warp + (mat & 1) * 8 + mrow;
                const uint32_t ka = kb[u] + tok * 128;
#pragma unroll
                for (int k = 0; k < 4 * DCH; ++k) {
                    if (k < ksteps) {
                        uint32_t x[4];
                        const int v = (2 * k + (mat >> 1)) & 7;
                        ldmatrix_x4(ka + (k >> 2) * (kTokens * 128) + ((v ^ (tok & 7)) << 4), x);
                        // (even and odd steps in sums of their own: half the chain)
#pragma unroll
                        for (int h = 0; h < NT; ++h) mma_16816<BF16>(k & 1 ? d[h][u] : c[h][u], x, qf[h][k][0], qf[h][k][1]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < NT; ++h) {
#pragma unroll
                for (int u = 0; u < T; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        c[h][u][e] += d[h][u][e];
                        if (kTokens * u + 16 * warp + r0 + (e & 2) * 4 >= live) c[h][u][e] = -INFINITY;
                    }
                float top[2] = {fmaxf(c[h][0][0], c[h][0][2]), fmaxf(c[h][0][1], c[h][0][3])};
#pragma unroll
                for (int u = 1; u < T; ++u) {
                    top[0] = fmaxf(top[0], fmaxf(c[h][u][0], c[h][u][2]));
                    top[1] = fmaxf(top[1], fmaxf(c[h][u][1], c[h][u][3]));
                }
#pragma unroll
                for (int i = 4; i < 32; i *= 2) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], i));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], i));
                }
                if (r0 == 0) *reinterpret_cast<float2*>(&sh.top[warp][8 * h + cpair]) = make_float2(top[0], top[1]);
            }
            consumer_sync();
#pragma unroll
            for (int h = 0; h < NT; ++h) {
                float2 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float2*>(&sh.top[i][8 * h + cpair]);
                const float top[2] = {fmaxf(fmaxf(w[0].x, w[1].x), fmaxf(w[2].x, w[3].x)) * a.scale_log2,
                                      fmaxf(fmaxf(w[0].y, w[1].y), fmaxf(w[2].y, w[3].y)) * a.scale_log2};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mm = fmaxf(m[h][e], top[e]), b = mm == -INFINITY ? 0.f : mm;
                    const float f = exp2_fast(m[h][e] - b);
                    m[h][e] = mm;
                    l[h][e] *= f;
#pragma unroll
                    for (int u = 0; u < T; ++u) {
                        c[h][u][e] = exp2_fast(fmaf(c[h][u][e], a.scale_log2, -b));
                        c[h][u][e + 2] = exp2_fast(fmaf(c[h][u][e + 2], a.scale_log2, -b));
                        l[h][e] = l[h][e] + c[h][u][e] + c[h][u][e + 2];
                    }
#pragma unroll
                    for (int i = 0; i < DCH; ++i) {
                        o[i][h][e] *= f;
                        o[i][h][e + 2] *= f;
                    }
                }
                // the weights by rows, 16 of this warp's keys a tile
#pragma unroll
                for (int u = 0; u < T; ++u) {
                    uint8_t* pw = sp + (8 * h + r0) * kPPitch + (kTokens * u + 16 * warp + cpair) * 2;
                    *reinterpret_cast<uint32_t*>(pw) = movmatrix_trans(pack2<BF16>(c[h][u][0], c[h][u][1]));
                    *reinterpret_cast<uint32_t*>(pw + 16) = movmatrix_trans(pack2<BF16>(c[h][u][2], c[h][u][3]));
                }
            }
            consumer_sync();
            // O^T += V^T P^T over all keys, this warp's part of head_dim
            const uint32_t pa = smem_u32(sp) + mrow * kPPitch + mat * 16;
#pragma unroll
            for (int k = 0; k < T * kTokens / 16; k += 2) {
                const uint32_t vb = kb[k / (kTokens / 16)] + Cfg::kTensor;
                uint32_t p[NT][4];
#pragma unroll
                for (int h = 0; h < NT; ++h) ldmatrix_x4(pa + 8 * h * kPPitch + k * 32, p[h]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int tok = 16 * ((k + j) % (kTokens / 16)) + (mat >> 1) * 8 + mrow;
                    // keys past the end have weight 0, but what lies in their place may be NaN
                    const int left = live - 16 * (k + j) - cpair;
                    const uint32_t lo = left >= 2 ? 0xFFFFFFFFu : (left == 1 ? 0x0000FFFFu : 0u);
                    const uint32_t hi = left >= 10 ? 0xFFFFFFFFu : (left == 9 ? 0x0000FFFFu : 0u);
#pragma unroll
                    for (int i = 0; i < DCH; ++i) {
                        const int part = warp + 4 * i;
                        if (part < ksteps) {
                            uint32_t x[4];
                            const int v = (2 * part + (mat & 1)) & 7;
                            ldmatrix_x4_trans(vb + (part >> 2) * (kTokens * 128) + tok * 128 + ((v ^ (tok & 7)) << 4), x);
                            x[0] &= lo;
                            x[1] &= lo;
                            x[2] &= hi;
                            x[3] &= hi;
#pragma unroll
                            for (int h = 0; h < NT; ++h) mma_16816<BF16>(o[i][h], x, p[h][2 * j], p[h][2 * j + 1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) {
#pragma unroll
                for (int u = 0; u < T; ++u) mbar_arrive(&sh.empty[(it + u) % S]);
            }
            it += T;
        };
        int t = walk.t0;
        if constexpr (Cfg::kAtOnce == 2)
            for (; t + 2 <= walk.t1; t += 2) step(t, std::integral_constant<int, 2>());
        for (; t < walk.t1; ++t) step(t, std::integral_constant<int, 1>());
        // ---------------------------------------------------------------- the unit's end
#pragma unroll
        for (int h = 0; h < NT; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int i = 4; i < 32; i *= 2) l[h][e] += __shfl_xor_sync(0xffffffffu, l[h][e], i);
                if (r0 == 0) sh.sum[warp][8 * h + cpair + e] = l[h][e];
            }
        consumer_sync();
        const int qh = head * a.group + chunk * 8 * NT;  // the unit's first query head
        uint16_t* out = a.out + static_cast<long long>(walk.i) * a.o_seq + static_cast<long long>(qh) * a.o_head;
        float* lse = a.lse ? a.lse + static_cast<long long>(walk.i) * a.q_heads + qh : nullptr;
        const bool whole = walk.t0 == 0 && walk.t1 == walk.nt;
        // Parts that begin a unit lie in a CTA's second place, others in its first.
        const long long place = 2ll * blockIdx.x + (walk.t0 == 0 ? 1 : 0);
        float* po = a.part_o + place * kUnitRows * a.head_dim;
#pragma unroll
        for (int h = 0; h < NT; ++h) {
            float inv[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 8 * h + cpair + e;
                const float sum = (sh.sum[0][row] + sh.sum[1][row]) + (sh.sum[2][row] + sh.sum[3][row]);
                inv[e] = walk.len > 0 ? __fdividef(1.f, sum) : 0.f;
                if (warp == 0 && r0 == 0 && row < rows) {
                    if (!whole) a.part_ml[place * kUnitRows + row] = make_float2(m[h][e], sum);
                    // (no key: -inf + log 0. The maximum passes over scores of NaN, their sum does not)
                    else if (lse != nullptr) lse[row] = (m[h][e] + __log2f(sum)) * kLn2;
                }
            }
#pragma unroll
            for (int i = 0; i < DCH; ++i) {
                const int dim = 16 * (warp + 4 * i);
                if (dim >= a.head_dim) continue;
                if (whole) {
                    // by rows: two dimensions a lane
                    const uint32_t x = movmatrix_trans(pack2<BF16>(o[i][h][0] * inv[0], o[i][h][1] * inv[1]));
                    const uint32_t y = movmatrix_trans(pack2<BF16>(o[i][h][2] * inv[0], o[i][h][3] * inv[1]));
                    if (8 * h + r0 < rows) {
                        uint16_t* dst = out + (8 * h + r0) * a.o_head + dim + cpair;
                        *reinterpret_cast<uint32_t*>(dst) = x;
                        *reinterpret_cast<uint32_t*>(dst + 8) = y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 8 * h + cpair + (e & 1);
                        if (row < rows) po[row * a.head_dim + dim + r0 + (e & 2) * 4] = o[i][h][e];
                    }
                }
            }
        }
        if (whole) continue;
        consumer_sync();  // the part has been written
        const long long c0 = cta_of(walk.unit_start), c1 = cta_of(walk.unit_start + walk.nt - 1);
        const int parts = static_cast<int>(c1 - c0) + 1;
        if (threadIdx.x == 0) {
            // releases what the barrier above has shown this thread, and acquires the other parts
            uint32_t old;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(a.arrived + c0) : "memory");
            const bool last = old == static_cast<uint32_t>(parts - 1);
            if (last) a.arrived[c0] = 0;  // nobody else of this call comes here any more
            sh.last = last;
        }
        consumer_sync();
        if (sh.last) {
            // the parts in the order of the keys: c0's second place, the others' first; eight of them loaded at a time
            constexpr int kBatch = 8;
            const int vecs = a.head_dim / 4;
            const float2* ml0 = a.part_ml + 2 * c0 * kUnitRows;
            const float* o0 = a.part_o + 2 * c0 * kUnitRows * a.head_dim;
            for (int e = threadIdx.x; e < rows * vecs; e += kConsumers) {
                const int row = e / vecs, v = e - row * vecs;
                float mm = -INFINITY, ll = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int c = 0; c < parts; c += kBatch) {
                    float2 ml[kBatch];
                    float4 x[kBatch];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        ml[j] = make_float2(-INFINITY, 0.f);
                        x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (c + j < parts) {
                            const int at = (2 * (c + j) + (c + j == 0 ? 1 : 0)) * kUnitRows + row;
                            ml[j] = __ldcg(ml0 + at);
                            x[j] = __ldcg(reinterpret_cast<const float4*>(o0 + static_cast<long long>(at) * a.head_dim) + v);
                        }
                    }
                    float top = mm;
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) top = fmaxf(top, ml[j].x);
                    const float b = top == -INFINITY ? 0.f : top, f = exp2_fast(mm - b);
                    mm = top;
                    ll *= f;
                    acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        const float g = exp2_fast(ml[j].x - b);
                        ll = fmaf(ml[j].y, g, ll);
                        acc.x = fmaf(x[j].x, g, acc.x);
                        acc.y = fmaf(x[j].y, g, acc.y);
                        acc.z = fmaf(x[j].z, g, acc.z);
                        acc.w = fmaf(x[j].w, g, acc.w);
                    }
                }
                const float inv = __fdividef(1.f, ll);  // (a unit in parts has tokens)
                *reinterpret_cast<uint2*>(out + row * a.o_head + 4 * v) =
                    make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
                if (lse != nullptr && v == 0) lse[row] = (mm + __log2f(ll)) * kLn2;
            }
        }
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

static size_t part_places(const tb_cache* c) { return 4 * static_cast<size_t>(c->ctx->num_sms); }  // two a CTA

size_t decode_bytes(const tb_cache* c) {
    return part_places(c) * kUnitRows * (c->d.head_dim * sizeof(float) + sizeof(float2)) + part_places(c) / 2 * sizeof(uint32_t) * 4;
}

tb_status decode_create(tb_cache* c) {
    const tb_cache_desc& d = c->d;
    c->decode_ctas = 2 * c->ctx->num_sms;
    c->part_o = static_cast<float*>(c->blob);
    c->part_ml = reinterpret_cast<float2*>(c->part_o + part_places(c) * kUnitRows * d.head_dim);
    c->arrived = reinterpret_cast<uint32_t*>(c->part_ml + part_places(c) * kUnitRows);
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

template <bool BF16, int DCH, int NT>
static tb_status launch_decode(tb_cache* c, int layer, const DecodeArgs& a, cudaStream_t st) {
    auto* kernel = decode_kernel<BF16, DCH, NT>;
    static OncePerDevice once;
    TB_TRY(once([&]() -> tb_status {
        TB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DecodeCfg<DCH>::kSmem));
        return TB_OK;
    }));
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

template <bool BF16>
static tb_status launch_decode(tb_cache* c, int layer, const DecodeArgs& a, cudaStream_t st) {
    // groups above 8 would read every key once more for each 8 query heads: 16 of them share a unit there
    const bool two = a.group > 8;
    if (a.head_dim > 64) return two ? launch_decode<BF16, 2, 2>(c, layer, a, st) : launch_decode<BF16, 2, 1>(c, layer, a, st);
    return two ? launch_decode<BF16, 1, 2>(c, layer, a, st) : launch_decode<BF16, 1, 1>(c, layer, a, st);
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
    TB_TRY(device_check("cache attend", c->ctx));
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
    const int unit = group > 8 ? 16 : 8;
    a.chunks = (group + unit - 1) / unit;
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
    return d.dtype == TB_DT_BF16 ? launch_decode<true>(c, layer, a, st) : launch_decode<false>(c, layer, a, st);
}

}  // extern "C"
