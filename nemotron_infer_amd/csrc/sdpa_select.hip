// sdpa_select.hip -- the pages that a new token attends, chosen by a score of each page, for gfx950.
//
// A sequence of P pages, P > n_select, attends its newest and those n_select - 1 of the others with the largest
//
//   score = max over the query heads h of the KV head of  sum_d max(q_hd, 0) hi_d + min(q_hd, 0) lo_d,
//
// lo, hi the page's bounds (kv_bounds.hip): no key of the page has a larger product with any of these heads.  Ties
// go to the earlier page, NaN comes first (a page that holds one is attended, as the attention over all would).
// The chosen ones, in their order, are a page table of their own for each KV head, which the attention of
// sdpa_decode_paged.hip then goes through; the newest one is last, so that a length says where they end.
//
// Which pages are chosen must not hang on the order of a sum: scores are summed in 64 bits (the products are exact
// there) and rounded to float32 once.  With mid = (lo + hi) / 2 and half = (hi - lo) / 2, exact in 64 bits for what
// bf16 holds, a term is q mid + |q| half: two multiply-adds, the magnitude for nothing.
//
// Scores.  Bound: reading the bounds, 512 bytes a page and head.  16 lanes take a page, 8 dims each, the queries in
// their registers; a wave takes 4 pages at a time.
// Choice: one workgroup for a sequence's KV head: the n-th largest by four counts of 8 bits each, in LDS, then one
// pass in order.  Bound: latency.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"
#include "nmi_packed.hpp"

#include <algorithm>

namespace nmi {

namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kHeads = 5;               // query heads at a time: 16 registers each
constexpr int kKeys = 8192;             // scores of a sequence kept in LDS

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

// The sum over 16 lanes, in all of them.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double row_sum16_f64(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    v += dpp_f64<0x140>(v);
    return v;
}

// A workgroup takes every parts-th 16 pages of a sequence's KV head.
__global__ __launch_bounds__(kThreads) void page_score_kernel(const SelectArgs a, int parts) {
    const int part = blockIdx.x % parts, g = (int)(blockIdx.x / parts % a.kv.n_kv), b = (int)(blockIdx.x / parts / a.kv.n_kv);
    const Sequence s = sequence(a, b);
    if (s.pages <= a.select) return;
    const int lane = threadIdx.x & 63, sub = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t* row = a.kv.page_table + b * a.kv.table_stride;
    float* scores = a.scores + ((int64_t)b * a.kv.n_kv + g) * a.kv.max_pages;
    const int chunks = (a.group + kHeads - 1) / kHeads, per = (a.group + chunks - 1) / chunks;
    for (int h0 = 0; h0 < a.group; h0 += per) {
        const int heads = min(per, a.group - h0);
        double q[kHeads][8];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            float x[8];
            unpack8(load16(a.q + (int64_t)b * a.ldq + (int64_t)(g * a.group + h0 + min(h, heads - 1)) * kPagedHead + 8 * sub), x);
#pragma unroll
            for (int i = 0; i < 8; ++i) q[h][i] = x[i];
        }
        for (int p0 = (part * kWaves + wave) * 4; p0 < s.pages - 1; p0 += parts * kWaves * 4) {
            const int p = p0 + (lane >> 4);
            bool none = p >= s.pages - 1, bad = false;
            const int page = none ? 0 : checked_page(row[p], a.kv.n_pages, &bad);
            const uint16_t* bounds = a.bounds + (((int64_t)page * a.kv.n_kv + g) * 2) * kPagedHead + 8 * sub;
            float lo[8], hi[8];
            unpack8(load16(bounds), lo);
            unpack8(load16(bounds + kPagedHead), hi);
            double mid[8], half[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mid[i] = 0.5 * ((double)lo[i] + (double)hi[i]);
                half[i] = 0.5 * ((double)hi[i] - (double)lo[i]);
            }
            float best = -INFINITY;
#pragma unroll
            for (int h = 0; h < kHeads; ++h) {
                if (h >= heads) break;
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum = __builtin_fma(q[h][i], mid[i], sum);
                    sum = __builtin_fma(__builtin_fabs(q[h][i]), half[i], sum);
                }
                best = __builtin_elementwise_maximum(best, (float)row_sum16_f64(sum));      // (NaN stays)
            }
            if (sub == 0 && !none) {
                if (h0) best = __builtin_elementwise_maximum(best, scores[p]);
                scores[p] = bad ? NAN : best;           // (a bad page is the attention's to report)
            }
        }
    }
}

// Unsigned keys in the order of the scores: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Inclusive sums over the workgroup, the sum of all to *total.
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t (&sums)[kWaves], uint32_t* total) {
    v = wave_scan_u32(v);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? sums[w] : 0u;
        all += sums[w];
    }
    *total = all;
    return before + v;
}

__global__ __launch_bounds__(kThreads) void page_select_kernel(const SelectArgs a) {
    __shared__ uint32_t keys[kKeys];
    __shared__ uint32_t bins[256];
    __shared__ uint32_t sums[kWaves];
    __shared__ uint32_t found[2];       // a digit, and how many of the larger keys are wanted beside it
    const int tid = threadIdx.x, g = (int)(blockIdx.x % a.kv.n_kv), b = (int)(blockIdx.x / a.kv.n_kv);
    const Sequence s = sequence(a, b);
    const int32_t* row = a.kv.page_table + b * a.kv.table_stride;
    const int64_t mine = ((int64_t)b * a.kv.n_kv + g) * a.select;
    auto put = [&](int64_t i, int place) {      // (a length that the table does not hold: no page, which the attention reports)
        if (a.rows) a.rows[mine + i] = s.bad ? -1 : row[place];
        if (a.selected) a.selected[mine + i] = place;
    };
    const int kept = min(s.pages, a.select);
    if (a.selected)
        for (int i = kept + tid; i < a.select; i += kThreads) a.selected[mine + i] = -1;
    if (g == 0 && tid == 0 && a.out_lens)
        a.out_lens[b] = s.pages <= a.select ? s.len : s.len - ((s.pages - a.select) << a.kv.page_shift);
    if (s.pages <= a.select) {
        for (int i = tid; i < s.pages; i += kThreads) put(i, i);
        return;
    }
    const int n = s.pages - 1;                  // those to choose from
    if (tid == 0) put(a.select - 1, n);
    uint32_t want = (uint32_t)a.select - 1;
    if (!want) return;
    const float* scores = a.scores + ((int64_t)b * a.kv.n_kv + g) * a.kv.max_pages;
    const bool here = n <= kKeys;
    if (here)
        for (int i = tid; i < n; i += kThreads) keys[i] = key_of(scores[i]);
    auto key = [&](int i) { return here ? keys[i] : key_of(scores[i]); };
    // the want-th largest key, 8 bits at a time: `top` its bits so far
    uint32_t top = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        bins[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t k = key(i);
            if ((k & mask) == top) atomicAdd(&bins[k >> shift & 255], 1u);
        }
        __syncthreads();
        const uint32_t c = bins[255 - tid];     // thread t: digit 255 - t, and the sum of those from there up
        uint32_t all;
        const uint32_t upto = group_scan(c, sums, &all);
        if (upto >= want && upto - c < want) {
            found[0] = 255 - tid;
            found[1] = want - (upto - c);
        }
        __syncthreads();
        top |= found[0] << shift;
        want = found[1];
        __syncthreads();
    }
    // all that are larger, and the first `want` that are equal
    uint32_t out = 0, equal = 0;
    for (int i0 = 0; i0 < n; i0 += kThreads) {
        const int i = i0 + tid;
        const uint32_t k = i < n ? key(i) : 0u;
        const uint32_t is_equal = i < n && k == top;
        uint32_t all_equal, all;
        const uint32_t rank = equal + group_scan(is_equal, sums, &all_equal);
        const uint32_t take = i < n && (k > top || (is_equal && rank <= want));
        const uint32_t place = out + group_scan(take, sums, &all);
        if (take) put(place - 1, i);
        equal += all_equal;
        out += all;
    }
}

}  // namespace

hipError_t launch_page_select(const SelectArgs& a, hipStream_t stream) {
    const int64_t groups = (int64_t)a.batch * a.kv.n_kv;
    if (a.select < a.kv.max_pages) {
        // as many workgroups as are resident, or one for each 16 pages that a sequence may have
        const int64_t most = ((int64_t)a.kv.max_pages + 15) / 16, parts = std::max<int64_t>(1, 8 * device_info().num_cu / groups);
        const int p = (int)std::min(most, parts);
        hipLaunchKernelGGL(page_score_kernel, dim3((uint32_t)(groups * p)), dim3(kThreads), 0, stream, a, p);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(page_select_kernel, dim3((uint32_t)groups), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace nmi
