// Paged key-value cache: page bookkeeping on the device (reserve, fork, free,
// compact), writing new keys and values, and copying page contents.
//
// Bookkeeping is integer work on a few thousand words with an order to keep (the
// lowest free page goes to the first slot that needs one), so each call's
// bookkeeping is one block of 1024 threads: prefix sums over the slots' needs and
// over the free pages, no atomics whose order could show in the result. It checks
// everything before it changes anything, so a refused call leaves the state as it
// was. Such a block's time is its chain of dependent accesses, some 0.7 us each: values that
// only the end of a call changes are read through L1, eight lanes take a slot's pages so that 128 slots
// are looked at together, and checks share a barrier (fork of 64 children, with its copies, 31.9 -> 25.9 us; 26.2 since
// copies count their vectors in 64 bits).
// Moving page contents is a second, grid-wide kernel that reads the list the first one left; it is bound by
// memory bandwidth.
#include <cuda_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <new>

#include "attention.cuh"
#include "cache.hpp"
#include "ptx.cuh"
#include "quant.cuh"

namespace tb {

constexpr int kBook = 1024;  // threads of a bookkeeping block

struct CacheView {
    int32_t *table, *lengths, *refs;
    int32_t *marks, *offsets, *taken, *remap, *jobs, *job_src, *job_dst, *job_rows;
    int num_pages, max_seqs, max_pages, page_size;
    uint32_t* err;
};

static CacheView view_of(const tb_cache* c) {
    return CacheView{c->b.page_table, c->b.lengths, c->b.refs, c->marks, c->offsets, c->taken, c->remap, c->jobs,
                     c->job_src, c->job_dst, c->job_rows, c->d.num_pages, c->d.max_seqs, c->d.max_pages,
                     c->d.page_size, c->ctx->dev_err};
}

// Exclusive prefix sum of one value a thread over the block; `total` the sum. `s` is 33 words.
__device__ __forceinline__ int block_scan(int v, int* s, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s[warp] = x;
    __syncthreads();
    if (warp == 0) {
        const int w = lane < kBook / 32 ? s[lane] : 0;
        int a = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, a, o);
            if (lane >= o) a += y;
        }
        s[lane] = a - w;
        if (lane == 31) s[32] = a;
    }
    __syncthreads();
    const int r = s[warp] + x - v;
    total = s[32];
    __syncthreads();
    return r;
}

__device__ __forceinline__ int pages_for(int tokens, int page_size) { return (tokens + page_size - 1) / page_size; }

// The lowest `need` free pages into c.taken; false when there are fewer. Four pages a thread and
// pass; the passes stop as soon as enough are found.
__device__ bool find_free(const CacheView& c, int need, int* s) {
    int found = 0;
    for (int p0 = 0; p0 < c.num_pages && found < need; p0 += 4 * kBook) {
        const int p = p0 + 4 * static_cast<int>(threadIdx.x);
        bool f[4];
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = p + j < c.num_pages && __ldcg(c.refs + p + j) == 0;
            n += f[j];
        }
        int total;
        int at = found + block_scan(n, s, total);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (f[j]) {
                if (at < need) c.taken[at] = p + j;
                ++at;
            }
        found += total;
    }
    __syncthreads();
    return found >= need;
}

// Takes distinct slots: false (for the whole block) when one is out of range, occurs twice or has
// a length outside the cache. Leaves marks set; clear_marks undoes them.
__device__ bool mark_slots(const CacheView& c, const int32_t* slots, int n) {
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kBook) {
        const int s = slots[i];
        if (s < 0 || s >= c.max_seqs) {
            bad = true;
            continue;
        }
        if (atomicExch(c.marks + s, 1) != 0) bad = true;
        const int len = __ldcg(c.lengths + s);
        if (len < 0 || static_cast<long long>(len) > static_cast<long long>(c.max_pages) * c.page_size) bad = true;
    }
    return !__syncthreads_or(bad);
}
__device__ void clear_marks(const CacheView& c, const int32_t* slots, int n) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kBook) {
        const int s = slots[i];
        if (s >= 0 && s < c.max_seqs) c.marks[s] = 0;
    }
}

// Eight lanes a slot: calls f(page) for the first pages of the slots i0, i0 + 128, ...: all of them, or only
// those filled to the end. lengths and table change only at a call's end, so they may come from L1.
template <class F>
__device__ __forceinline__ void for_pages(const CacheView& c, const int32_t* slots, int n, bool full_only, F f) {
    for (int i = threadIdx.x >> 3; i < n; i += kBook / 8) {
        const int s = slots[i], len = c.lengths[s];
        const int np = full_only ? len / c.page_size : pages_for(len, c.page_size);
        const int32_t* row = c.table + static_cast<long long>(s) * c.max_pages;
#pragma unroll 4
        for (int j = threadIdx.x & 7; j < np; j += 8) f(row[j]);
    }
}

__global__ void __launch_bounds__(kBook) cache_reserve_kernel(CacheView c, const int32_t* slots, const int32_t* counts,
                                                              int n) {
    __shared__ int s[33];
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    bool bad = !mark_slots(c, slots, n);
    if (!bad) {
        for (int i = threadIdx.x; i < n; i += kBook) {
            const int cnt = counts ? counts[i] : 1;
            const long long len = static_cast<long long>(__ldcg(c.lengths + slots[i])) + cnt;
            if (cnt < 0 || len > static_cast<long long>(c.max_pages) * c.page_size) bad = true;
        }
    }
    bad = __syncthreads_or(bad);
    uint32_t err = bad ? DEV_ERR_INDEX : 0u;
    if (!bad) {
        long long need = 0;  // the same in every thread
        for (int i0 = 0; i0 < n; i0 += kBook) {
            const int i = i0 + threadIdx.x;
            int w = 0;  // at most max_pages, 2^20
            if (i < n) {
                const int len = __ldcg(c.lengths + slots[i]);
                w = pages_for(len + (counts ? counts[i] : 1), c.page_size) - pages_for(len, c.page_size);
            }
            int total;
            const int at = block_scan(w, s, total);
            if (need + total > c.num_pages) {
                need = static_cast<long long>(c.num_pages) + 1;  // cannot be met
                break;
            }
            if (i < n) c.offsets[i] = static_cast<int>(need) + at;
            need += total;
        }
        if (need > c.num_pages || !find_free(c, static_cast<int>(need), s)) err = DEV_ERR_PAGES;
    }
    __syncthreads();
    if (err == 0) {
        for (int i = threadIdx.x >> 5; i < n; i += kBook / 32) {
            const int slot = slots[i], cnt = counts ? counts[i] : 1;
            const int len = __ldcg(c.lengths + slot), at = __ldcg(c.offsets + i);
            const int p0 = pages_for(len, c.page_size), p1 = pages_for(len + cnt, c.page_size);
            for (int j = p0 + (threadIdx.x & 31); j < p1; j += 32) {
                const int p = __ldcg(c.taken + at + j - p0);
                c.table[static_cast<long long>(slot) * c.max_pages + j] = p;
                c.refs[p] = 1;
            }
            __syncwarp();
            if ((threadIdx.x & 31) == 0) c.lengths[slot] = len + cnt;
        }
    } else if (threadIdx.x == 0) {
        atomicOr(c.err, err);
    }
    clear_marks(c, slots, n);
}

__global__ void __launch_bounds__(kBook) cache_free_kernel(CacheView c, const int32_t* slots, int n) {
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    bool bad = !mark_slots(c, slots, n);
    if (!bad) {
        for_pages(c, slots, n, false, [&](int p) { bad |= p < 0 || p >= c.num_pages; });
        bad = __syncthreads_or(bad);
    }
    if (!bad) {
        for_pages(c, slots, n, false, [&](int p) { atomicSub(c.refs + p, 1); });
        __syncthreads();  // every row has been read
        for (int i = threadIdx.x >> 3; i < n; i += kBook / 8) {
            const int slot = slots[i], np = pages_for(c.lengths[slot], c.page_size);
            for (int j = threadIdx.x & 7; j < np; j += 8) c.table[static_cast<long long>(slot) * c.max_pages + j] = -1;
            __syncwarp(0xFFu << (threadIdx.x & 24));
            if ((threadIdx.x & 7) == 0) c.lengths[slot] = 0;
        }
    } else if (threadIdx.x == 0) {
        atomicOr(c.err, DEV_ERR_INDEX);
    }
    clear_marks(c, slots, n);
}

__global__ void __launch_bounds__(kBook) cache_fork_kernel(CacheView c, const int32_t* parents, const int32_t* children,
                                                           int n) {
    __shared__ int s[33];
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    bool bad = !mark_slots(c, children, n);
    for (int i = threadIdx.x; i < n; i += kBook) {
        const int p = parents[i];
        if (p < 0 || p >= c.max_seqs || __ldcg(c.marks + p) != 0) {
            bad = true;
        } else {
            const int len = c.lengths[p];
            if (len < 0 || static_cast<long long>(len) > static_cast<long long>(c.max_pages) * c.page_size) bad = true;
        }
    }
    bad = __syncthreads_or(bad);
    if (!bad) {
        auto look = [&](int p) { bad |= p < 0 || p >= c.num_pages; };
        for_pages(c, children, n, false, look);
        for_pages(c, parents, n, false, look);
        bad = __syncthreads_or(bad);
    }
    uint32_t err = bad ? DEV_ERR_INDEX : 0u;
    if (!bad) {
        // what the children held goes back, full pages are shared
        for_pages(c, children, n, false, [&](int p) { atomicSub(c.refs + p, 1); });
        for_pages(c, parents, n, true, [&](int p) { atomicAdd(c.refs + p, 1); });
        int need = 0;  // a page for each last page that is not full
        for (int i0 = 0; i0 < n; i0 += kBook) {
            const int i = i0 + threadIdx.x;
            const int w = i < n && c.lengths[parents[i]] % c.page_size != 0;
            int total;
            const int at = block_scan(w, s, total);
            if (i < n) c.offsets[i] = need + at;
            need += total;
        }
        __syncthreads();
        if (!find_free(c, need, s)) {
            err = DEV_ERR_PAGES;
            for_pages(c, parents, n, true, [&](int p) { atomicSub(c.refs + p, 1); });
            for_pages(c, children, n, false, [&](int p) { atomicAdd(c.refs + p, 1); });
        } else {
            for (int i = threadIdx.x >> 3; i < n; i += kBook / 8) {
                const int lane = threadIdx.x & 7, child = children[i];
                const int len = c.lengths[parents[i]];
                const int32_t* from = c.table + static_cast<long long>(parents[i]) * c.max_pages;
                int32_t* to = c.table + static_cast<long long>(child) * c.max_pages;
                const int full = len / c.page_size, rows = len % c.page_size;
                const int had = pages_for(c.lengths[child], c.page_size);
#pragma unroll 4
                for (int j = lane; j < max(full, had); j += 8) to[j] = j < full ? from[j] : -1;
                __syncwarp(0xFFu << (threadIdx.x & 24));
                if (lane == 0) {
                    if (rows != 0) {
                        const int at = __ldcg(c.offsets + i), p = __ldcg(c.taken + at);
                        to[full] = p;
                        c.refs[p] = 1;
                        c.job_src[at] = from[full];
                        c.job_dst[at] = p;
                        c.job_rows[at] = rows;
                    }
                    c.lengths[child] = len;
                }
            }
            if (threadIdx.x == 0) c.jobs[0] = need;
        }
    }
    if (err != 0 && threadIdx.x == 0) {
        c.jobs[0] = 0;
        atomicOr(c.err, err);
    }
    clear_marks(c, children, n);
}

// Which pages move where. Two passes over refs: the pages in use, then the k-th page in use at or
// above that number and the k-th free page below it.
__global__ void __launch_bounds__(kBook) cache_compact_kernel(CacheView c, int32_t* refs_out) {
    __shared__ int s[33];
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    constexpr int kStep = 4 * kBook;
    int live = 0, r[4];
    auto load = [&](int p) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = p + j < c.num_pages ? __ldcg(c.refs + p + j) : 0;
    };
    for (int p0 = 0; p0 < c.num_pages; p0 += kStep) {
        load(p0 + 4 * static_cast<int>(threadIdx.x));
        int total;
        block_scan((r[0] > 0) + (r[1] > 0) + (r[2] > 0) + (r[3] > 0), s, total);
        live += total;
    }
    int moves = 0, holes = 0;
    for (int p0 = 0; p0 < c.num_pages; p0 += kStep) {
        const int p = p0 + 4 * static_cast<int>(threadIdx.x);
        if (c.num_pages > kStep) load(p);  // (otherwise they are still there)
        int n = 0;  // pages that move in the low half, holes in the high one: at most 4096 of each a step
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            n += p + j >= live && r[j] > 0;
            n += (p + j < live && r[j] <= 0) << 16;
        }
        int total;
        const int at = block_scan(n, s, total);
        int an = moves + (at & 0xFFFF), ah = holes + (at >> 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (p + j >= live && r[j] > 0) {
                c.job_src[an] = p + j;
                c.job_rows[an] = c.page_size;
                ++an;
            }
            if (p + j < live && r[j] <= 0) c.job_dst[ah++] = p + j;
            if (p + j < c.num_pages) {
                c.remap[p + j] = p + j;
                refs_out[p + j] = r[j];
            }
        }
        moves += total & 0xFFFF;
        holes += total >> 16;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += kBook) {
        const int src = __ldcg(c.job_src + k), dst = __ldcg(c.job_dst + k);
        c.remap[src] = dst;
        refs_out[dst] = __ldcg(refs_out + src);
        refs_out[src] = 0;
    }
    if (threadIdx.x == 0) c.jobs[0] = moves;
}

// ---------------------------------------------------------------------------
// Page contents
// ---------------------------------------------------------------------------

struct CopyArgs {
    uint4 *k, *v;
    const int32_t *src, *dst, *rows;  // rows null: whole pages
    const int32_t* count;             // null: n pairs
    int n;
    int layers, heads, num_pages;
    int row_vecs, page_size;          // 16-byte vectors a token and head; tokens a page
    // compact: page table entries through remap, by the same launch
    const int32_t *table, *remap;
    int32_t* table_out;
    long long table_n;
    uint32_t* err;
};

// A warp moves one head of one page (page_size * head_dim contiguous elements, 4 KB at 16 tokens of
// 128), eight 16-byte vectors a lane in flight: bound by memory bandwidth (a compaction's 319 MB in 51.6 us,
// 6.2 TB/s).
__global__ void __launch_bounds__(256) cache_copy_kernel(CopyArgs a) {
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const long long warps = static_cast<long long>(gridDim.x) * 8;
    const long long w0 = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int n = a.count ? __ldcg(a.count) : a.n;
    const int per_page = a.layers * 2 * a.heads;
    const long long page_vecs = static_cast<long long>(a.page_size) * a.row_vecs;
    for (long long u = w0; u < static_cast<long long>(n) * per_page; u += warps) {
        const int job = static_cast<int>(u / per_page);
        int r = static_cast<int>(u - static_cast<long long>(job) * per_page);
        const int head = r % a.heads;
        r /= a.heads;
        uint4* base = r & 1 ? a.v : a.k;
        const int layer = r >> 1;
        const int src = __ldcg(a.src + job), dst = __ldcg(a.dst + job);
        if (src < 0 || src >= a.num_pages || dst < 0 || dst >= a.num_pages) {
            if (lane == 0) atomicOr(a.err, DEV_ERR_INDEX);
            continue;
        }
        const long long vecs = static_cast<long long>(a.rows ? __ldcg(a.rows + job) : a.page_size) * a.row_vecs;  // up to 2^34
        const uint4* from = base + ((static_cast<long long>(layer) * a.num_pages + src) * a.heads + head) * page_vecs;
        uint4* to = base + ((static_cast<long long>(layer) * a.num_pages + dst) * a.heads + head) * page_vecs;
        for (long long i = lane; i < vecs; i += 256) {
            uint4 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + 32 * j < vecs) x[j] = __ldcs(from + i + 32 * j);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + 32 * j < vecs) __stcs(to + i + 32 * j, x[j]);
        }
    }
    if (a.table_out != nullptr) {
        const long long step = static_cast<long long>(gridDim.x) * 256;
        for (long long e = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; e < a.table_n; e += step) {
            const int p = a.table[e];
            if (p >= a.num_pages) atomicOr(a.err, DEV_ERR_INDEX);
            a.table_out[e] = p < 0 || p >= a.num_pages ? p : __ldcg(a.remap + p);
        }
    }
}

struct WriteArgs {
    const uint4 *k, *v;
    long long k_token, k_head, v_token, v_head;  // strides in 16-byte vectors
    uint4 *k_layer, *v_layer;
    const int32_t *slots, *offsets, *table, *lengths;
    int n, heads, page_size, num_pages, max_seqs, max_pages;
    int row_vecs;
    long long total;
    uint32_t* err;
};

// A warp writes the key or the value of one token: heads * head_dim elements, eight 16-byte vectors a lane in
// flight. The token's slot is found by a 32-way search of the offsets (two steps for up to 1024 slots).
// Bound by memory bandwidth: 13,256 tokens of 32 heads of 128, 349 MB, in 59 us (5.9 TB/s; with four vectors a
// lane and the division by a head's vectors at run time 67 us). VECS: vectors of a head (head_dim / 8),
// 0: any number.
template <int VECS>
__global__ void __launch_bounds__(128) cache_write_kernel(WriteArgs a) {
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const long long t = w >> 1;
    if (t >= a.total) return;
    // the last i in [lo, hi) with offsets[i] <= t
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int i = lo + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, i < hi && a.offsets[i] <= t);
        const int k = 31 - __clz(le | 1u);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    const int first = a.offsets[lo], end = a.offsets[lo + 1];
    const int slot = a.slots[lo];
    bool bad = t < first || t >= end || slot < 0 || slot >= a.max_seqs;
    int pos = -1, page = -1;
    if (!bad) {
        const long long at = static_cast<long long>(a.lengths[slot]) - (end - t);
        bad = at < 0 || at >= static_cast<long long>(a.max_pages) * a.page_size;
        if (!bad) {
            pos = static_cast<int>(at);
            page = a.table[static_cast<long long>(slot) * a.max_pages + pos / a.page_size];
            bad = page < 0 || page >= a.num_pages;
        }
    }
    if (bad) {
        if (lane == 0) atomicOr(a.err, DEV_ERR_INDEX);
        return;
    }
    const int row_vecs = VECS ? VECS : a.row_vecs;
    const bool is_v = w & 1;
    const uint4* from = is_v ? a.v + t * a.v_token : a.k + t * a.k_token;
    const long long hs = is_v ? a.v_head : a.k_head;
    const long long page_vecs = static_cast<long long>(a.page_size) * row_vecs;  // of one head, up to 2^34
    uint4* to = (is_v ? a.v_layer : a.k_layer) + page * a.heads * page_vecs + static_cast<long long>(pos % a.page_size) * row_vecs;
    const int vecs = a.heads * row_vecs;  // at most 2^30
    for (int i0 = lane; i0 < vecs; i0 += 256) {
        uint4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + 32 * j, h = i / row_vecs;
            if (i < vecs) x[j] = __ldcs(from + h * hs + (i - h * row_vecs));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + 32 * j, h = i / row_vecs;
            if (i < vecs) to[h * page_vecs + (i - h * row_vecs)] = x[j];
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

static tb_status cache_check(const tb_cache* c, const char* op, int n, bool distinct, std::initializer_list<const void*> ptrs) {
    if (!c) return fail(TB_ERR_INVALID_ARGUMENT, "%s: null cache", op);
    if (n < 0) return fail(TB_ERR_SHAPE_MISMATCH, "%s: negative count", op);
    if (distinct && n > c->d.max_seqs)
        return fail(TB_ERR_SHAPE_MISMATCH, "%s: %d distinct slots of a cache of %d", op, n, c->d.max_seqs);
    if (n == 0) return TB_OK;
    for (const void* p : ptrs)
        if (!p) return fail(TB_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
    return TB_OK;
}

// Launches as a programmatic dependent of the kernel before it (its start-up overlaps that
// kernel's end; every kernel here waits for it before it reads anything).
template <class... P, class... A>
static tb_status launch(tb_context* ctx, void (*kernel)(P...), int grid, int block, cudaStream_t st, A... args) {
    TB_TRY(device_check("cache", ctx));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    TB_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    ctx->launches++;
    return TB_OK;
}

// Workspaces come from a pool of the context that keeps up to 64 MB of what was freed: mapping 5 MB anew for
// each cache and unmapping it took 0.5 to 1.5 ms.
static cudaError_t workspace_alloc(tb_context* ctx, size_t bytes, void** out) {
    if (!ctx->pool) {
        cudaMemPoolProps props = {};
        props.allocType = cudaMemAllocationTypePinned;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = ctx->device;
        cudaError_t e = cudaMemPoolCreate(&ctx->pool, &props);
        if (e != cudaSuccess) {
            ctx->pool = nullptr;
            return e;
        }
        uint64_t keep = 64u << 20;
        cudaMemPoolSetAttribute(ctx->pool, cudaMemPoolAttrReleaseThreshold, &keep);
    }
    return cudaMallocFromPoolAsync(out, bytes, ctx->pool, nullptr);
}

static CopyArgs copy_args(const tb_cache* c) {
    CopyArgs a{};
    a.k = static_cast<uint4*>(c->b.k_pages);
    a.v = static_cast<uint4*>(c->b.v_pages);
    a.layers = c->d.layers;
    a.heads = c->d.kv_heads;
    a.num_pages = c->d.num_pages;
    a.row_vecs = c->d.head_dim / 8;
    a.page_size = c->d.page_size;
    a.err = c->ctx->dev_err;
    return a;
}

static tb_status launch_copy(tb_cache* c, const CopyArgs& a, long long most, cudaStream_t st) {
    const long long units = most * c->d.layers * 2 * c->d.kv_heads;
    const long long blocks = std::max<long long>((units + 7) / 8, a.table_out ? (a.table_n + 255) / 256 : 1);
    const int grid = static_cast<int>(std::min<long long>(blocks, static_cast<long long>(c->ctx->num_sms) * 8));
    return launch(c->ctx, cache_copy_kernel, std::max(grid, 1), 256, st, a);
}

}  // namespace tb

using namespace tb;

extern "C" {

TB_API tb_status tb_cache_create(tb_context* ctx, const tb_cache_desc* d, const tb_cache_buffers* b, tb_cache** out) {
    if (!out) return fail(TB_ERR_INVALID_ARGUMENT, "cache: null argument");
    *out = nullptr;
    if (!ctx || !d || !b) return fail(TB_ERR_INVALID_ARGUMENT, "cache: null argument");
    if (!b->k_pages || !b->v_pages || !b->page_table || !b->lengths || !b->refs)
        return fail(TB_ERR_INVALID_ARGUMENT, "cache: null buffer");
    if (!aligned16(b->k_pages) || !aligned16(b->v_pages))
        return fail(TB_ERR_INVALID_ARGUMENT, "cache: pages must be 16-byte aligned");
    if (d->dtype != TB_DT_BF16 && d->dtype != TB_DT_FP16)
        return fail(TB_ERR_DTYPE_MISMATCH, "cache: unsupported type %d (FP16 or BF16)", d->dtype);
    if (d->layers < 1 || d->kv_heads < 1 || d->num_pages < 1 || d->max_seqs < 1 || d->max_pages < 1)
        return fail(TB_ERR_SHAPE_MISMATCH, "cache: every dimension must be positive");
    if (d->head_dim < 16 || d->head_dim > 128 || d->head_dim % 16)
        return fail(TB_ERR_NOT_ACCELERATED, "cache: head_dim %d is not a multiple of 16 up to 128", d->head_dim);
    if (d->page_size < 8 || d->page_size % 8)
        return fail(TB_ERR_NOT_ACCELERATED, "cache: page_size %d is not a multiple of 8", d->page_size);
    // token positions and page rows are int32, and so are the prefix sums over 1024 slots' page needs
    if (d->num_pages > (1 << 20) || d->max_pages > (1 << 20))
        return fail(TB_ERR_NOT_ACCELERATED, "cache: more than 2^20 pages");
    const long long rows = static_cast<long long>(d->num_pages) * d->kv_heads;
    if (static_cast<long long>(d->page_size) > (1ll << 30) / rows || rows > (1ll << 30) ||
        static_cast<long long>(d->max_pages) * d->page_size > (1ll << 30) ||
        d->layers > (1 << 16) || static_cast<long long>(d->layers) * d->kv_heads > (1ll << 29))
        return fail(TB_ERR_NOT_ACCELERATED, "cache: more than 2^30 rows or 2^16 layers");
    // a token's key is written with 32-bit indexes of 16-byte vectors
    if (static_cast<long long>(d->kv_heads) * (d->head_dim / 8) > (1ll << 30))
        return fail(TB_ERR_NOT_ACCELERATED, "cache: more than 2^33 elements in a token's key");
    TB_TRY(device_check("cache", ctx));
    tb_cache* c = new (std::nothrow) tb_cache;
    if (!c) return fail(TB_ERR_INVALID_ARGUMENT, "cache: out of host memory");
    c->ctx = ctx;
    c->device = ctx->device;
    c->d = *d;
    c->b = *b;
    // one allocation: the attention's workspace (16-byte pieces first), then the words that begin as zero
    const size_t words = 2 * static_cast<size_t>(d->max_seqs) + 5 * static_cast<size_t>(d->num_pages) + 4;
    const size_t parts = decode_bytes(c);
    cudaError_t e = workspace_alloc(ctx, parts + words * sizeof(int32_t), &c->blob);
    if (e == cudaSuccess) e = cudaMemsetAsync(c->blob, 0, parts + words * sizeof(int32_t), nullptr);
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);  // other streams may be the first to use it
    if (e != cudaSuccess) {
        tb_cache_destroy(c);
        return fail(TB_ERR_CUDA, "cache workspace: %s", cudaGetErrorString(e));
    }
    int32_t* w = reinterpret_cast<int32_t*>(static_cast<char*>(c->blob) + parts);
    c->jobs = w;
    c->marks = w + 4;
    c->offsets = c->marks + d->max_seqs;
    c->taken = c->offsets + d->max_seqs;
    c->remap = c->taken + d->num_pages;
    c->job_src = c->remap + d->num_pages;
    c->job_dst = c->job_src + d->num_pages;
    c->job_rows = c->job_dst + d->num_pages;
    tb_status st;
    try {
        st = decode_create(c);
    } catch (const std::bad_alloc&) {
        st = fail(TB_ERR_INVALID_ARGUMENT, "cache: out of host memory");
    }
    if (st != TB_OK) {
        tb_cache_destroy(c);
        return st;
    }
    *out = c;
    return TB_OK;
}

TB_API void tb_cache_destroy(tb_cache* c) {
    if (!c) return;
    if (c->blob) {
        int current = c->device;
        cudaGetDevice(&current);
        if (current != c->device) cudaSetDevice(c->device);
        // The workspace may go to another cache at once: calls on any stream are through. (A device that could not be
        // waited for, as while a stream of it is captured, keeps it.)
        if (cudaDeviceSynchronize() == cudaSuccess) cudaFreeAsync(c->blob, nullptr);
        if (current != c->device) cudaSetDevice(current);
    }
    delete c;
}

TB_API tb_status tb_cache_reserve(tb_cache* c, const int32_t* slots, const int32_t* counts, int32_t n, void* stream) {
    TB_TRY(cache_check(c, "cache reserve", n, true, {slots}));
    if (n == 0) return TB_OK;
    return launch(c->ctx, cache_reserve_kernel, 1, kBook, static_cast<cudaStream_t>(stream), view_of(c), slots, counts, n);
}

TB_API tb_status tb_cache_free(tb_cache* c, const int32_t* slots, int32_t n, void* stream) {
    TB_TRY(cache_check(c, "cache free", n, true, {slots}));
    if (n == 0) return TB_OK;
    return launch(c->ctx, cache_free_kernel, 1, kBook, static_cast<cudaStream_t>(stream), view_of(c), slots, n);
}

TB_API tb_status tb_cache_fork(tb_cache* c, const int32_t* parents, const int32_t* children, int32_t n, void* stream) {
    TB_TRY(cache_check(c, "cache fork", n, true, {parents, children}));
    if (n == 0) return TB_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    TB_TRY(launch(c->ctx, cache_fork_kernel, 1, kBook, st, view_of(c), parents, children, n));
    CopyArgs a = copy_args(c);
    a.src = c->job_src;
    a.dst = c->job_dst;
    a.rows = c->job_rows;
    a.count = c->jobs;
    return launch_copy(c, a, n, st);
}

TB_API tb_status tb_cache_copy_pages(tb_cache* c, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    TB_TRY(cache_check(c, "cache copy_pages", n, false, {src, dst}));
    if (n == 0) return TB_OK;
    CopyArgs a = copy_args(c);
    a.src = src;
    a.dst = dst;
    a.n = n;
    return launch_copy(c, a, n, static_cast<cudaStream_t>(stream));
}

TB_API tb_status tb_cache_compact(tb_cache* c, int32_t* page_table_out, int32_t* refs_out, void* stream) {
    TB_TRY(cache_check(c, "cache compact", 0, false, {}));
    if (!page_table_out != !refs_out)
        return fail(TB_ERR_INVALID_ARGUMENT, "cache compact: page_table_out and refs_out go together");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    TB_TRY(launch(c->ctx, cache_compact_kernel, 1, kBook, st, view_of(c), refs_out ? refs_out : c->b.refs));
    CopyArgs a = copy_args(c);
    a.src = c->job_src;
    a.dst = c->job_dst;
    a.rows = c->job_rows;
    a.count = c->jobs;
    a.table = c->b.page_table;
    a.remap = c->remap;
    a.table_out = page_table_out ? page_table_out : c->b.page_table;
    a.table_n = static_cast<long long>(c->d.max_seqs) * c->d.max_pages;
    return launch_copy(c, a, c->d.num_pages, st);
}

TB_API tb_status tb_cache_write(tb_cache* c, int32_t layer, const int32_t* slots, const int32_t* offsets, int32_t n,
                                int64_t total, const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                const void* v, int64_t v_token_stride, int64_t v_head_stride, void* stream) {
    TB_TRY(cache_check(c, "cache write", n, false, {slots, offsets}));
    if (layer < 0 || layer >= c->d.layers)
        return fail(TB_ERR_SHAPE_MISMATCH, "cache write: layer %d of %d", layer, c->d.layers);
    if (total < 0 || total > (1ll << 30)) return fail(TB_ERR_SHAPE_MISMATCH, "cache write: %lld rows", (long long)total);
    if (n > (1 << 30)) return fail(TB_ERR_NOT_ACCELERATED, "cache write: more than 2^30 slots");  // (32-bit search)
    if (total > 0 && n == 0) return fail(TB_ERR_SHAPE_MISMATCH, "cache write: rows without a slot");
    if (total == 0) return TB_OK;
    if (!k || !v) return fail(TB_ERR_INVALID_ARGUMENT, "cache write: null pointer");
    if (!aligned16(k) || !aligned16(v) || (k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7)
        return fail(TB_ERR_INVALID_ARGUMENT, "cache write: k and v must be 16-byte aligned with strides that are multiples of 8");
    WriteArgs a{};
    a.k = static_cast<const uint4*>(k);
    a.v = static_cast<const uint4*>(v);
    a.k_token = k_token_stride / 8;
    a.k_head = k_head_stride / 8;
    a.v_token = v_token_stride / 8;
    a.v_head = v_head_stride / 8;
    a.row_vecs = c->d.head_dim / 8;
    const long long layer_vecs = static_cast<long long>(c->d.num_pages) * c->d.kv_heads * c->d.page_size * a.row_vecs;
    a.k_layer = static_cast<uint4*>(c->b.k_pages) + layer * layer_vecs;
    a.v_layer = static_cast<uint4*>(c->b.v_pages) + layer * layer_vecs;
    a.slots = slots;
    a.offsets = offsets;
    a.table = c->b.page_table;
    a.lengths = c->b.lengths;
    a.n = n;
    a.heads = c->d.kv_heads;
    a.page_size = c->d.page_size;
    a.num_pages = c->d.num_pages;
    a.max_seqs = c->d.max_seqs;
    a.max_pages = c->d.max_pages;
    a.total = total;
    a.err = c->ctx->dev_err;
    // head_dim 128 and 64: the division by a head's vectors is a shift
    auto* kernel = a.row_vecs == 16 ? cache_write_kernel<16> : (a.row_vecs == 8 ? cache_write_kernel<8> : cache_write_kernel<0>);
    return launch(c->ctx, kernel, static_cast<int>((2 * total + 3) / 4), 128, static_cast<cudaStream_t>(stream), a);
}

}  // extern "C"
