// The paged key-value cache's handle, shared by its translation units.
#pragma once

#include <vector>

#include "internal.hpp"

namespace tb {
// The attention kernel's workspace, at the blob's start, and its maps (decode.cu).
size_t decode_bytes(const tb_cache* c);
tb_status decode_create(tb_cache* c);
}  // namespace tb

struct tb_cache {
    tb_context* ctx = nullptr;
    int device = 0;  // the context's, which may be gone when the cache is destroyed
    tb_cache_desc d{};
    tb_cache_buffers b{};
    // Bookkeeping workspace (device), part of the blob:
    int32_t* marks = nullptr;    // [max_seqs] zero between calls: slots seen by the running call
    int32_t* offsets = nullptr;  // [max_seqs] first entry of each slot's new pages in `taken`
    int32_t* taken = nullptr;    // [num_pages] free pages found, lowest first
    int32_t* remap = nullptr;    // [num_pages] compact: new place of each page at or above `live`
    int32_t* jobs = nullptr;     // {number of copies, live pages}, then
    int32_t* job_src = nullptr;  // [num_pages] copy from this page ...
    int32_t* job_dst = nullptr;  // ... to this page ...
    int32_t* job_rows = nullptr; // ... this many tokens
    void* blob = nullptr;
    // Attention of one new token: what a CTA leaves of a unit that others share (decode.cu)
    float* part_o = nullptr;     // [2 * CTAs][16][head_dim]
    float2* part_ml = nullptr;   // [2 * CTAs][16]
    uint32_t* arrived = nullptr; // [CTAs] zero between calls
    int decode_ctas = 0;
    std::vector<CUtensorMap> k_map, v_map;  // of each layer
};
