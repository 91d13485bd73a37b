// nmi_paged.hpp -- a paged KV cache as the kernels see it, and the bounds on what a device-side page
// table, length or offset may make them touch.
//
// The functions marked NMI_HD are plain arithmetic, also compiled for the host by the tests: every
// address the kernels form from a value in device memory (a page id, a length, a sequence's offset)
// goes through one of them.  So is the rotation's sine.
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
constexpr int kPagedBlock = 16;        // positions under one scale (block scales)
static_assert(kPagedBlock == kPagedTile, "a tile has one scale");

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

// Scales of blocks, [n_pages, n_kv, page_size / kPagedBlock] each.
struct BlockScales {
    float* k;
    float* v;
};

// What a cache holds: bf16, e4m3 codes under a scale per KV head, or under one per head and block.
enum class KvForm { Bf16, E4m3, Block };

// The scale of the block of a head that holds position `pos` of a page.
NMI_HD int64_t block_index(int64_t page, int n_kv, int head, int page_shift, int pos) {
    return ((page * n_kv + head) << (page_shift - 4)) + ((pos & ((1 << page_shift) - 1)) >> 4);
}

// The biased exponent of the smallest power of two s, normal, with amax <= 448 s, of the bits of a finite amax >= 0:
// 448 is 1.75 2^8.  From 1 to 247.
NMI_HD int block_exponent(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < 1 ? 1 : e;
}
// That of the smallest power of two that is no less than a scale found in memory: itself, if an append wrote it.  1 for
// what is no scale (negative, NaN, infinite); at most what 2^-e can be had of.
NMI_HD int block_exponent_of_scale(uint32_t bits) {
    if (bits >= 0x7F800000u) return 1;
    const int e = (int)(bits >> 23) + ((bits & 0x7FFFFFu) ? 1 : 0);
    return e < 1 ? 1 : (e > 253 ? 253 : e);
}

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

// Whether packed row t, of the rows given, is one of those of the sequence with offsets c0, c1 so cut, and its
// place there.
NMI_HD bool span_holds(int c0, int c1, int t) { return c0 <= t && t < c1; }
NMI_HD int span_place(int c0, int t) { return t - (c0 < 0 ? 0 : c0); }

// The rows of packed sequence b that are stored or counted, where `before` is the end of the earlier sequences' rows
// (0 at first): [*first, *first + result), none of them an earlier sequence's.  *place: the first one's place in the
// sequence.
NMI_HD int later_span(int c0, int c1, int tokens, int before, int* first, int* place, bool* bad) {
    int f = 0;
    int n = checked_span(c0, c1, tokens, &f, bad);
    *place = 0;
    if (f < before) {
        if (n > 0) *bad = true;
        const int cut = before - f < n ? before - f : n;
        *place = cut;
        n -= cut;
        f += cut;
    }
    *first = f;
    return n;
}

// Of `total` pages that come back to a stack of n_pages, `count` of them there, those that it has room for (*bad where
// there are more, which are not looked at): whatever the lengths claim, less than 2^31.
NMI_HD uint32_t pages_back(uint32_t total, int count, int n_pages, bool* bad) {
    const uint32_t room = (uint32_t)(n_pages - count);
    if (total > room) *bad = true;
    return total < room ? total : room;
}

// Blocks of kPagedBlock positions that n positions from `pos` on lie in.
NMI_HD int blocks_of(int64_t pos, int n) { return n > 0 ? (int)(((pos & (kPagedBlock - 1)) + n + kPagedBlock - 1) / kPagedBlock) : 0; }
// At most so many of `tokens` rows in `batch` sequences: each has 30 positions at most that are not its own in its blocks.
NMI_HD int64_t most_blocks(int64_t tokens, int64_t batch) {
    const int64_t n = batch < tokens ? batch : tokens, by = (tokens + 30 * n) / kPagedBlock;
    return by < tokens ? by : tokens;
}
// Pages that n positions from `pos` on complete, and at most so many of `tokens` rows in `batch` sequences.
NMI_HD int pages_completed(int64_t pos, int n, int page_shift) {
    return n > 0 ? (int)(((pos + n) >> page_shift) - (pos >> page_shift)) : 0;
}
NMI_HD int64_t most_pages_completed(int64_t tokens, int64_t batch, int page_shift) {
    const int64_t n = batch < tokens ? batch : tokens;
    return (tokens >> page_shift) + n;
}

// cos and sin of 2 pi f, |f| <= 1/2: f = q / 4 + y with |y| <= 1/8, the Taylor polynomials of y's angle
// t, |t| <= pi / 4, turned by q quarters.  In 64 bits, each rounded once at the end: what the polynomials leave
// out (t^17 / 17! < 5e-17, t^16 / 16! < 2e-15) is less than 2^-48 of the value, so a result is the nearest
// float but for values as close as that to the middle of two.
NMI_HD void cos_sin(double f, float* cos_f, float* sin_f) {
    const double q = __builtin_rint(4.0 * f), t = 6.283185307179586 * __builtin_fma(q, -0.25, f), z = t * t;
    double s = __builtin_fma(z, -1.0 / 1307674368000.0, 1.0 / 6227020800.0);
    double c = __builtin_fma(z, -1.0 / 87178291200.0, 1.0 / 479001600.0);
    s = __builtin_fma(z, s, -1.0 / 39916800.0);
    c = __builtin_fma(z, c, -1.0 / 3628800.0);
    s = __builtin_fma(z, s, 1.0 / 362880.0);
    c = __builtin_fma(z, c, 1.0 / 40320.0);
    s = __builtin_fma(z, s, -1.0 / 5040.0);
    c = __builtin_fma(z, c, -1.0 / 720.0);
    s = __builtin_fma(z, s, 1.0 / 120.0);
    c = __builtin_fma(z, c, 1.0 / 24.0);
    s = __builtin_fma(z, s, -1.0 / 6.0);
    c = __builtin_fma(z, c, -0.5);
    const float sf = (float)__builtin_fma(t * z, s, t), cf = (float)__builtin_fma(z, c, 1.0);
    const int k = (int)q;                                       // -2 .. 2
    const float cs = (k & 1) ? sf : cf, sn = (k & 1) ? cf : sf;
    *cos_f = ((k + 1) & 2) ? -cs : cs;
    *sin_f = (k & 2) ? -sn : sn;
}

// Decode attention: tiles per wave when all sequences' tiles, `total` of them in a row, are dealt to at
// most `waves` waves, at least `unit` to each.
constexpr int kPagedMaxPositions = 1 << 30;
constexpr int kPagedWaves = 4;          // per workgroup
NMI_HD int range_tiles(uint32_t total, int waves, int unit) {
    const uint32_t c = (total + (uint32_t)waves - 1) / (uint32_t)waves;
    return c > (uint32_t)unit ? (int)c : unit;
}

// Wave x's tiles [range_first(x), range_first(x + 1)) of that row; none where the row is shorter.
NMI_HD uint32_t range_first(uint32_t x, int c, uint32_t total) {
    const uint64_t f = (uint64_t)x * (uint32_t)c;
    return f < total ? (uint32_t)f : total;
}

// Whether tile `at` of that row is to be looked for among the 64 sequences after those from b0 on, up to
// whose last the row has `upto` tiles.  Never past the batch, whatever the lengths: they are read again on
// the way, and may by then be less than those that `at` was dealt by.
NMI_HD bool look_on(uint32_t at, uint32_t upto, int b0, int batch) { return at >= upto && b0 + 64 < batch; }

// The pieces of a sequence with tiles [first, first + tiles) of the row, one at least.  A workgroup all
// of whose tiles are the sequence's takes them together, as one piece; of another, each wave takes a
// piece.  So there are `head` waves' pieces of the first workgroup (from `wave` on), `joint` workgroups',
// `tail` waves' of the last.  A piece that wave x, or the workgroup whose first wave is x, has of
// sequence b is left in slot x + b: going along the row, x or b or both grow from one piece to the
// next, so no two share a slot, and waves + batch slots are enough.
struct Pieces {
    int wave, head, joint, tail;
    NMI_HD int count() const { return head + joint + tail; }
    NMI_HD int owner(int i) const {     // x of piece i
        if (i < head) return wave + i;
        const int group = wave / kPagedWaves + (head > 0 ? 1 : 0);
        if (i < head + joint) return (group + i - head) * kPagedWaves;
        return (group + joint) * kPagedWaves + i - head - joint;
    }
};
// Whether workgroup x has no tiles but the sequence's.
NMI_HD bool is_joint(uint32_t x, uint32_t first, uint32_t tiles, int c, uint32_t total) {
    return first <= range_first(x * kPagedWaves, c, total) && first + tiles >= range_first((x + 1) * kPagedWaves, c, total);
}
NMI_HD Pieces pieces_of(uint32_t first, uint32_t tiles, int c, uint32_t total) {
    const uint32_t w0 = first / (uint32_t)c, w1 = (first + tiles - 1) / (uint32_t)c;
    const uint32_t g0 = w0 / kPagedWaves, g1 = w1 / kPagedWaves;
    const bool joint0 = is_joint(g0, first, tiles, c, total), joint1 = is_joint(g1, first, tiles, c, total);
    Pieces p;
    p.wave = (int)w0;
    if (g0 == g1) {
        p.head = joint0 ? 0 : (int)(w1 - w0 + 1);
        p.joint = joint0 ? 1 : 0;
        p.tail = 0;
    } else {
        p.head = joint0 ? 0 : (int)(kPagedWaves * (g0 + 1) - w0);
        p.tail = joint1 ? 0 : (int)(w1 - kPagedWaves * g1 + 1);
        p.joint = (int)(g1 - g0 + 1) - (p.head ? 1 : 0) - (p.tail ? 1 : 0);
    }
    return p;
}

}  // namespace nmi
