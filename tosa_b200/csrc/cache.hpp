// The paged key-value cache's handle, shared by its translation units.
#pragma once

#include "internal.hpp"

struct tb_cache {
    tb_context* ctx = nullptr;
    tb_cache_desc d{};
    tb_cache_buffers b{};
    // Bookkeeping workspace (device), one allocation:
    int32_t* marks = nullptr;    // [max_seqs] zero between calls: slots seen by the running call
    int32_t* offsets = nullptr;  // [max_seqs] first entry of each slot's new pages in `taken`
    int32_t* taken = nullptr;    // [num_pages] free pages found, lowest first
    int32_t* remap = nullptr;    // [num_pages] compact: new place of each page at or above `live`
    int32_t* jobs = nullptr;     // {number of copies, live pages}, then
    int32_t* job_src = nullptr;  // [num_pages] copy from this page ...
    int32_t* job_dst = nullptr;  // ... to this page ...
    int32_t* job_rows = nullptr; // ... this many tokens
    void* blob = nullptr;
};
