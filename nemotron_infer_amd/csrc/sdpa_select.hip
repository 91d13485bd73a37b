// sdpa_select.hip -- the pages that a new token attends, chosen by a score of each page, for gfx950.
//
// A sequence of P pages, P > n_select, attends its newest and those n_select - 1 of the others with the largest
//
//   score = max over the query heads h of the KV head of  sum_d max(q_hd, 0) hi_d + min(q_hd, 0) lo_d,
//
// lo, hi the page's bounds (kv_bounds.hip): no key of the page has a larger product with any of these heads, but for what
// the bounds' rounding to bf16 takes (nothing of bf16 keys and of codes under powers of two).  Ties go to the earlier
// page, NaN comes first (a page that holds one is attended, as the attention over all would).  The chosen ones, in their
// order, are a page table of their own for each KV head, which the attention of
// sdpa_decode_paged.hip then goes through; the newest one is last, so that a length says where they end.
//
// Which pages are chosen must not hang on the order of a sum: scores are summed in 64 bits (the products are exact
// there) and rounded to float32 once.  Each dim adds both its products, of which one is 0: what the query does not use
// takes no bits of the sum, however large it is (and 0 times an infinity is NaN).  (Float32 sums instead, in an earlier
// form, took 1 us of 20 less for one sequence of 100001 positions, 2 of 43 for 20 documents.)
//
// Scores.  Bound: the 64-bit arithmetic of many pages, latency of few (length and page id, then bounds and queries).  16
// lanes take a page, 8 dims each, the queries' positive and negative parts in their registers; a wave takes 4 pages at a
// time, all of the chunk's query heads at once so that their sums hide one another's latency, and asks for the next pages'
// bounds as those at hand are used: their upper ones first, so that both need not be held at once (4 heads: 166
// registers, 3 waves to a SIMD, where 178 leave 2: 8 sequences of 60000 33.0 us for the whole call, so 31.2).  (One head after
// another, in an earlier form, 40 sequences of 4000: 39.0 where that took 36.7; 16 pages a wave, 4 lanes each, the queries
// in LDS: 36.8, but one sequence of 60000 18.6 where that took 17.0.)
// A sequence's KV head is dealt to as many workgroups as all of them leave it of 2 per CU, which are at work at once; to 8,
// as far as 6 per CU allow, where that is fewer, since the longest of many sequences would then take long by itself.
// 2 / 3 / 4 / 6 / 8 / 12 per CU, the whole call, 40 / 8 heads: one sequence of 100001 positions 18.5 / 19.4 / 19.6 / 19.5 / 19.7 /
// 19.7 us, 8 of 40000 26.5 / 27.6 / 27.9 / 29.5 / 31.6 / 31.1, 40 of 4000 39.1 / 38.2 / 38.6 / 38.8 / 41.2 / 42.1, 20 documents of 900
// to 30000 46.7 / 40.0 / 39.2 / 39.8 / 39.9 / 41.4; so 18.5, 26.6, 39.0 and 39.6.  (The pages of all sequences in equal shares, an
// earlier form: 20 documents 43.4 where that took 43.1, and one sequence 21.0 where that took 20.6.)
// Choice: one workgroup for a sequence's KV head: the range of the scores cut into 1024 bins, counted in LDS, the bin
// with the last one wanted cut again while it has many, its few ranked one against another; then one pass in order.
// Bound: latency, a handful of barriers: 5.6 to 6.0 us (traced) of 1562 pages; four passes of 8 bits and a scan for each 256 pages,
// an earlier form, took 12.4.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"
#include "nmi_packed.hpp"

#include <algorithm>

namespace nmi {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kHeads = 5;               // query heads at a time at most: 32 registers each
constexpr int kPerCu = 2, kPerCuMost = 6, kPerHead = 8;     // scores' workgroups
constexpr int kBinBits = 10, kSelectThreads = 1 << kBinBits, kSelectWaves = kSelectThreads / 64;
constexpr int kKeys = 6144;             // keys and page ids of a sequence kept in LDS
constexpr int kFew = 64;                // keys ranked by a wave

struct Sequence {
    int len, pages;
    bool bad;
};
__device__ __forceinline__ Sequence sequence(const SelectArgs& a, int b) {
    Sequence s;
    s.bad = false;
    s.len = checked_len(load_const(a.lens + b), a.kv.max_pages, a.kv.page_shift, &s.bad);
    s.pages = (int)(((int64_t)s.len + (1 << a.kv.page_shift) - 1) >> a.kv.page_shift);
    return s;
}

// The sums over 16 lanes, in all of them.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int CTRL, int N>
__device__ __forceinline__ void add_dpp_f64(double (&v)[N]) {
    double w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = dpp_f64<CTRL>(v[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += w[i];
}
template <int N>
__device__ __forceinline__ void row_sums16_f64(double (&v)[N]) {
    add_dpp_f64<0xB1>(v);
    add_dpp_f64<0x4E>(v);
    add_dpp_f64<0x141>(v);
    add_dpp_f64<0x140>(v);
}

// A workgroup takes every parts-th 16 pages of a sequence's KV head.  HEADS: query heads at a time (the last ones again where
// there are fewer: their scores are the same).
template <int HEADS>
__global__ __launch_bounds__(kThreads) void page_score_kernel(const SelectArgs a, int parts) {
    if (a.select == 1) return;                          // (the newest page, whatever the scores)
    const int part = blockIdx.x % parts, g = (int)(blockIdx.x / parts % a.kv.n_kv), b = (int)(blockIdx.x / parts / a.kv.n_kv);
    const int lane = threadIdx.x & 63, sub = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t* row = a.kv.page_table + b * a.kv.table_stride;
    const int first = (part * kWaves + wave) * 4 + (lane >> 4), stride = parts * kWaves * 4;
    // (entries of the table's row, whatever they hold, asked for beside the length)
    auto page_id = [&](int p) { return row[min(p, a.kv.max_pages - 1)]; };
    int32_t id = page_id(first), id_after = page_id(first + stride);
    const Sequence s = sequence(a, b);
    const int n = s.pages - 1;
    if (s.pages <= a.select || (part * kWaves + wave) * 4 >= n) return;
    auto at = [&](int32_t id, bool* bad) {
        *bad = false;
        const int page = checked_page(id, a.kv.n_pages, bad);
        return a.bounds + (((int64_t)page * a.kv.n_kv + g) * 2) * kPagedHead + 8 * sub;
    };
    // 8 dims' products with one bound
    auto add = [](uint4 v, const double (&q)[HEADS][8], double (&sum)[HEADS]) {
        float x[8];
        unpack8(v, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double y = x[i];
#pragma unroll
            for (int h = 0; h < HEADS; ++h) sum[h] = __builtin_fma(q[h][i], y, sum[h]);
        }
    };
    float* scores = a.scores + ((int64_t)b * a.kv.n_kv + g) * a.kv.max_pages;
    for (int h0 = 0; h0 < a.group; h0 += HEADS) {
        // a page's bounds are on their way while those before are used, and the id of the next one's
        bool bad;
        const uint16_t* bounds = at(id, &bad);
        uint4 lo = load16(bounds), hi = load16(bounds + kPagedHead);
        id = id_after;
        double above[HEADS][8], below[HEADS][8];        // max(q, 0) and min(q, 0); NaN in both
#pragma unroll
        for (int h = 0; h < HEADS; ++h) {
            float x[8];
            unpack8(load16(a.q + (int64_t)b * a.ldq + (int64_t)(g * a.group + min(h0 + h, a.group - 1)) * kPagedHead + 8 * sub), x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                above[h][i] = __builtin_elementwise_maximum(x[i], 0.f);
                below[h][i] = __builtin_elementwise_minimum(x[i], 0.f);
            }
        }
        for (int p = first; __builtin_amdgcn_ballot_w64(p < n); p += stride) {      // (all lanes, for the sums over them)
            const bool was_bad = bad;
            bounds = at(id, &bad);
            id = page_id(p + 2 * stride);
            double sum[HEADS];
#pragma unroll
            for (int h = 0; h < HEADS; ++h) sum[h] = 0.0;
            add(hi, above, sum);
            hi = load16(bounds + kPagedHead);
            add(lo, below, sum);
            lo = load16(bounds);
            row_sums16_f64(sum);
            float best = -INFINITY;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) best = __builtin_elementwise_maximum(best, (float)sum[h]);      // (NaN stays)
            if (sub == 0 && p < n) {
                if (h0) best = __builtin_elementwise_maximum(best, scores[p]);
                scores[p] = was_bad ? NAN : best;       // (a bad page is the attention's to report)
            }
        }
        if (h0 + HEADS < a.group) id = page_id(first), id_after = page_id(first + stride);
    }
}

// Unsigned keys in the order of the scores: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Inclusive sums over the workgroup, the sum of all to *total.  Every thread takes part; `sums` is free afterwards only
// behind a barrier.
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t (&sums)[kSelectWaves], uint32_t* total) {
    v = wave_scan_u32(v);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    const uint32_t s = wave_scan_u32(lane < kSelectWaves ? sums[lane] : 0u);
    *total = lane_u32(s, 63);
    return v + (wave ? lane_u32(s, wave - 1) : 0u);
}

__global__ __launch_bounds__(kSelectThreads) void page_select_kernel(const SelectArgs a) {
    __shared__ uint32_t keys[kKeys];
    __shared__ int32_t ids[kKeys];
    __shared__ uint32_t bins[kSelectThreads];
    __shared__ uint32_t sums[3][kSelectWaves];
    __shared__ uint32_t found[3];                       // a bin, the keys in it, and those in larger ones
    __shared__ uint32_t few[kFew];
    const int tid = threadIdx.x, lane = tid & 63, g = (int)(blockIdx.x % a.kv.n_kv), b = (int)(blockIdx.x / a.kv.n_kv);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Sequence s = sequence(a, b);
    const int32_t* row = a.kv.page_table + b * a.kv.table_stride;
    const int64_t mine = ((int64_t)b * a.kv.n_kv + g) * a.select;
    auto put = [&](int64_t i, int place, int32_t id) {  // (a length that the table does not hold: no page, which the attention reports)
        if (a.rows) a.rows[mine + i] = s.bad ? -1 : id;
        if (a.selected) a.selected[mine + i] = place;
    };
    const int kept = min(s.pages, a.select);
    if (a.selected)
        for (int64_t i = kept + tid; i < a.select; i += kSelectThreads) a.selected[mine + i] = -1;     // (up to 2^31 - 1)
    if (g == 0 && tid == 0 && a.out_lens)
        a.out_lens[b] = s.pages <= a.select ? s.len : s.len - ((s.pages - a.select) << a.kv.page_shift);
    if (s.pages <= a.select) {
        for (int i = tid; i < s.pages; i += kSelectThreads) put(i, i, row[i]);
        return;
    }
    const int n = s.pages - 1;                          // those to choose from
    if (tid == 0) put(a.select - 1, n, row[n]);
    uint32_t want = (uint32_t)a.select - 1;
    if (!want) return;
    const float* scores = a.scores + ((int64_t)b * a.kv.n_kv + g) * a.kv.max_pages;
    const bool here = n <= kKeys;
    uint32_t lo = 0xFFFFFFFFu, hi = 0;                  // the range of the keys
    for (int i = tid; i < n; i += kSelectThreads) {
        const int32_t id = here ? row[i] : 0;
        const uint32_t k = key_of(scores[i]);
        if (here) keys[i] = k, ids[i] = id;
        lo = min(lo, k);
        hi = max(hi, k);
    }
    auto key = [&](int i) { return here ? keys[i] : key_of(scores[i]); };
    lo = ~wave_max_u32(~lo);
    hi = wave_max_u32(hi);
    if (lane == 0) sums[0][wave] = ~lo, sums[1][wave] = hi;
    bins[tid] = 0;
    __syncthreads();
    lo = ~wave_max_u32(lane < kSelectWaves ? sums[0][lane] : 0u);
    hi = wave_max_u32(lane < kSelectWaves ? sums[1][lane] : 0u);

    // The want-th largest key is in [lo, hi], counted from the largest of that range.  The range is cut into as many equal bins as
    // there are threads, and the bin that has it becomes the range, until few keys are in it or all are equal.
    for (;;) {
        const uint32_t span = hi - lo;
        const int shift = max(0, 32 - (span ? __builtin_clz(span) : 32) - kBinBits);
        for (int i = tid; i < n; i += kSelectThreads) {
            const uint32_t k = key(i);
            if (k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> shift], 1u);
        }
        __syncthreads();
        const uint32_t bin = kSelectThreads - 1 - tid, c = bins[bin];   // thread t: the t-th bin from above
        uint32_t all;
        const uint32_t upto = group_scan(c, sums[2], &all);
        if (upto >= want && upto - c < want) found[0] = bin, found[1] = c, found[2] = upto - c;
        bins[bin] = 0;
        __syncthreads();
        const uint32_t in_bin = found[1];
        want -= found[2];
        lo += found[0] << shift;
        hi = lo + min(hi - lo, (1u << shift) - 1);
        if (in_bin <= kFew || shift == 0) break;
        __syncthreads();                                // (found is read by all)
    }
    // Few: each ranked among them.  `lo` becomes the key itself, `want` the keys equal to it that are taken.
    if (hi != lo) {
        for (int i = tid; i < n; i += kSelectThreads) {
            const uint32_t k = key(i);
            if (k >= lo && k <= hi) few[atomicAdd(&bins[0], 1u)] = k;
        }
        __syncthreads();
        const int m = (int)bins[0];
        const uint32_t k = lane < m ? few[lane] : 0u;
        uint32_t above = 0, equal = 0;
        for (int i = 0; i < m; ++i) {
            const uint32_t other = lane_u32(k, i);
            above += other > k;
            equal += other == k;
        }
        const uint64_t hit = __builtin_amdgcn_ballot_w64(lane < m && above < want && above + equal >= want);
        const int who = __builtin_ctzll(hit);
        lo = lane_u32(k, who);
        want -= lane_u32(above, who);
    }
    // all that are larger, and the first `want` that are equal
    uint32_t larger = 0, equal = 0;                     // of those before the ones at hand
    for (int i0 = 0, turn = 0; i0 < n; i0 += kSelectThreads, turn ^= 1) {
        const int i = i0 + tid;
        const uint32_t k = i < n ? key(i) : 0u;
        const uint32_t is_larger = i < n && k > lo, is_equal = i < n && k == lo;
        uint32_t all;
        const uint32_t upto = group_scan(is_larger << 16 | is_equal, sums[turn], &all);
        const uint32_t larger_upto = larger + (upto >> 16), equal_upto = equal + (upto & 0xFFFFu);
        if (is_larger || (is_equal && equal_upto <= want))
            put((int64_t)larger_upto + min(equal_upto, want) - 1, i, here ? ids[i] : row[i]);
        larger += all >> 16;
        equal += all & 0xFFFFu;
    }
}

}  // namespace

hipError_t launch_page_select(const SelectArgs& a, hipStream_t stream) {
    const int64_t groups = (int64_t)a.batch * a.kv.n_kv;
    if (a.select < a.kv.max_pages) {
        // (no more than one for each 16 pages that a sequence may have)
        auto per_head = [&](int per_cu) { return std::max<int64_t>(1, per_cu * device_info().num_cu / groups); };
        const int64_t most = ((int64_t)a.kv.max_pages + 15) / 16;
        const int p = (int)std::min(most, std::max(per_head(kPerCu), std::min<int64_t>(per_head(kPerCuMost), kPerHead)));
        const int chunks = (a.group + kHeads - 1) / kHeads;
        const dim3 grid((uint32_t)(groups * p)), block(kThreads);
        switch ((a.group + chunks - 1) / chunks) {
            case 1: hipLaunchKernelGGL(page_score_kernel<1>, grid, block, 0, stream, a, p); break;
            case 2: hipLaunchKernelGGL(page_score_kernel<2>, grid, block, 0, stream, a, p); break;
            case 3: hipLaunchKernelGGL(page_score_kernel<3>, grid, block, 0, stream, a, p); break;
            case 4: hipLaunchKernelGGL(page_score_kernel<4>, grid, block, 0, stream, a, p); break;
            default: hipLaunchKernelGGL(page_score_kernel<kHeads>, grid, block, 0, stream, a, p);
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(page_select_kernel, dim3((uint32_t)groups), dim3(kSelectThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace nmi
