// nmi_paged.hpp -- a paged KV cache as the kernels see it, and the bounds on what a device-side page
// table, length or offset may make them touch.
//
// The functions marked NMI_HD are plain arithmetic, also compiled for the host by the tests: every
// address the kernels form from a value in device memory (a page id, a length, a sequence's offset)
// goes through one of them.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define NMI_HD __host__ __device__ __forceinline__
#else
#define NMI_HD inline
#endif

namespace nmi {

constexpr int kPagedHead = 128;        // head dim
constexpr int kPagedTile = 16;         // positions of a tile; a page holds a whole number of them
constexpr int kPagedMinPage = kPagedTile, kPagedMaxPage = 1 << 20;

// Strides in bytes.  A head's vector of position p of sequence b is at page_table[b][p >> page_shift]
// * page_stride + head * head_stride + (p & (page_size - 1)) * token_stride.
struct PagedKv {
    uint8_t* k_pages;
    uint8_t* v_pages;
    int64_t page_stride, head_stride, token_stride;
    const int32_t* page_table;          // [batch, >= max_pages], row stride table_stride entries
    int64_t table_stride;
    const float* k_scale;               // [n_kv] or nullptr (1)
    const float* v_scale;
    int n_pages, max_pages, page_shift, n_kv;
    uint32_t* error;                    // host word to set where the device data is out of range, or nullptr
};

// A page id from the table: itself, or page 0 with *bad set where the pool has no such page.
NMI_HD int checked_page(int id, int n_pages, bool* bad) {
    if (id >= 0 && id < n_pages) return id;
    *bad = true;
    return 0;
}

// A sequence's length: at most what its row of the table holds (*bad where it says more), at least 0.
NMI_HD int checked_len(int len, int max_pages, int page_shift, bool* bad) {
    const int64_t cap = (int64_t)max_pages << page_shift;
    if (len > cap) {
        *bad = true;
        return (int)cap;
    }
    return len < 0 ? 0 : len;
}

// Packed sequence b's rows [*first, *first + result) within [0, tokens): cu[b], cu[b + 1] as they are
// where they ascend within it, else cut to it (*bad).
NMI_HD int checked_span(int c0, int c1, int tokens, int* first, bool* bad) {
    int f = c0 < 0 ? 0 : (c0 > tokens ? tokens : c0);
    int e = c1 < f ? f : (c1 > tokens ? tokens : c1);
    if (f != c0 || e != c1) *bad = true;
    *first = f;
    return e - f;
}

// Decode attention: tiles per split when `total` tiles of all sequences are to make at most `budget`
// splits beyond the one that every sequence has; a multiple of `unit`, so that the waves of a
// workgroup get equal shares.  With n_b = max(1, ceil(tiles_b / result)) the splits of all sequences
// number at most batch + budget: sum ceil(t_b / c) <= batch + total / c.  Never more than a whole
// sequence of the most positions.
constexpr int kPagedMaxPositions = 1 << 30;
NMI_HD int split_tiles(uint32_t total, int budget, int unit) {
    const uint32_t c = (total + (uint32_t)budget - 1) / (uint32_t)budget;
    const uint32_t m = (c + (uint32_t)unit - 1) / (uint32_t)unit;
    constexpr uint32_t most = kPagedMaxPositions / kPagedTile;
    return (int)(m < 1 ? (uint32_t)unit : m > most / (uint32_t)unit ? most : m * (uint32_t)unit);
}

}  // namespace nmi
