// kv_assign.hip -- the pages of a pool handed to the sequences that grow, and taken back from those that end, with
// what the kernels of the step need of it (first positions, lengths, packed offsets, the tokens' slots), for gfx950.
//
// The free pages are a stack in device memory.  Sequences that end push theirs, in the sequences' order and each in
// its positions'; then those that grow pop theirs in the same order: with need_b pages for sequence b, page j of b is
// the stack's entry count - 1 - (sum of need_i, i < b) - j.  A sequence is granted all of its new tokens or none: none
// where its row of the table is too short, or where it needs pages and the needs up to its own are more than the
// stack holds.  So everything follows from prefix sums, and equal inputs give equal tables.
//
// Bound: latency; a step of a batch moves some kilobytes.  One workgroup, since the stack is one: 1024 sequences at
// a time in its threads, sums over them by DPP and LDS; what varies in length (pages pushed and popped, slots) is
// dealt to the threads one by one, each finding its sequence by a binary search over the sums in LDS.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"
#include "nmi_packed.hpp"

namespace nmi {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add_sat(uint32_t v) {
    return __builtin_elementwise_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
// Inclusive sums over the workgroup's threads, saturating at 2^32 - 1 (more than there can be of anything here), the sum of
// all to *total.  Every thread takes part; `sums` is free afterwards only behind a barrier.
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t (&sums)[kWaves], uint32_t* total) {
    v = dpp_add_sat<0x111, 0xF>(v);
    v = dpp_add_sat<0x112, 0xF>(v);
    v = dpp_add_sat<0x114, 0xF>(v);
    v = dpp_add_sat<0x118, 0xF>(v);
    v = dpp_add_sat<0x142, 0xA>(v);
    v = dpp_add_sat<0x143, 0xC>(v);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t s = sums[w];
        if (w < wave) before = __builtin_elementwise_add_sat(before, s);
        all = __builtin_elementwise_add_sat(all, s);
    }
    *total = all;
    return __builtin_elementwise_add_sat(before, v);
}

// The first of the kThreads ascending sums that is more than e (e is less than the last).
__device__ __forceinline__ int search(const uint32_t* upto, uint32_t e) {
    int at = 0;
#pragma unroll
    for (int step = kThreads / 2; step; step >>= 1)
        if (upto[at + step - 1] <= e) at += step;
    return at;
}

__global__ __launch_bounds__(kThreads) void kv_assign_kernel(const AssignArgs a) {
    __shared__ uint32_t upto[kThreads];         // sums over the sequences at hand
    __shared__ uint32_t sums[3][kWaves];
    __shared__ int32_t base[kThreads];          // of each: pages it had; then its first new position
    const int tid = threadIdx.x;
    const int size = 1 << a.page_shift;
    const int64_t cap = (int64_t)a.max_pages << a.page_shift;
    bool bad = false;
    int count = *a.free_count;
    if (count < 0 || count > a.n_pages) bad = true, count = count < 0 ? 0 : a.n_pages;

    // pages that come back
    for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
        const int b = b0 + tid;
        uint32_t back = 0;
        if (b < a.batch && a.add && a.add[b] < 0) {
            const int len = checked_len(a.lens[b], a.max_pages, a.page_shift, &bad);
            back = ((uint32_t)len + size - 1) >> a.page_shift;
        }
        uint32_t total;
        upto[tid] = group_scan(back, sums[0], &total);
        base[tid] = (int32_t)back;
        __syncthreads();
        for (uint32_t e = tid; e < total; e += kThreads) {
            const int i = search(upto, e);
            const uint32_t j = e - (upto[i] - (uint32_t)base[i]);
            const int id = a.table[(int64_t)(b0 + i) * a.table_stride + j];
            if (id < 0 || id >= a.n_pages || (int64_t)count + e >= a.n_pages) bad = true;
            if ((int64_t)count + e < a.n_pages) a.free_pages[count + e] = id;
        }
        count = (int)min((int64_t)count + total, (int64_t)a.n_pages);
        __syncthreads();
    }

    // pages handed out, and what follows from them
    uint32_t needed = 0, rows_before = 0, taken = 0;    // of the sequences before those at hand; pages granted
    for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
        const int b = b0 + tid;
        const int len = b < a.batch ? a.lens[b] : -1, add = b < a.batch ? (a.add ? a.add[b] : 1) : 0;
        const int used = (int)(((uint32_t)max(len, 0) + size - 1) >> a.page_shift);
        const bool wants = len >= 0 && add > 0;
        bool fits = wants && (int64_t)len + add <= cap;
        if (len > cap) bad = true;
        const uint32_t rows = add > 0 ? (uint32_t)add : 0u;
        uint32_t all_rows = 0, rows_upto = 0;
        if (a.cu) {
            rows_upto = __builtin_elementwise_add_sat(group_scan(rows, sums[0], &all_rows), rows_before);
            all_rows = __builtin_elementwise_add_sat(all_rows, rows_before);
            if (rows && rows_upto > (uint32_t)a.tokens) bad = true, fits = false;       // rows that are not there
        } else if (add > 1) {
            bad = true, fits = false;
        }
        const uint32_t need = fits ? (uint32_t)(((int64_t)len + add + size - 1) >> a.page_shift) - used : 0u;
        uint32_t all_need;
        const uint32_t need_upto = __builtin_elementwise_add_sat(group_scan(need, sums[1], &all_need), needed);
        const bool granted = fits && (need == 0 || need_upto <= (uint32_t)count);
        uint32_t granted_need;
        upto[tid] = group_scan(granted ? need : 0u, sums[2], &granted_need);
        base[tid] = used;
        if (b < a.batch) {
            a.start[b] = granted ? len : -1;
            a.kv_lens[b] = granted ? len + add : 0;
            a.lens_out[b] = granted ? len + add : (len >= 0 && add < 0 ? -1 : len);
            if (a.cu) {
                if (b == 0) a.cu[0] = 0;
                a.cu[b + 1] = (int32_t)min(rows_upto, (uint32_t)a.tokens);
            }
        }
        __syncthreads();
        // (those granted pages are the first that need any: their sums have no gaps)
        for (uint32_t e = tid; e < granted_need; e += kThreads) {
            const int i = search(upto, e);
            const uint32_t first = i ? upto[i - 1] : 0u;
            const int id = a.free_pages[count - 1 - (int64_t)(taken + e)];
            if (id < 0 || id >= a.n_pages) bad = true;
            a.table[(int64_t)(b0 + i) * a.table_stride + base[i] + (e - first)] = id;
        }
        __syncthreads();
        auto slot = [&](int s, int64_t pos) {
            const int id = a.table[(int64_t)s * a.table_stride + (pos >> a.page_shift)];
            if (id < 0 || id >= a.n_pages) {
                bad = true;
                return (int64_t)-1;
            }
            return (int64_t)id * size + (pos & (size - 1));
        };
        if (!a.cu) {
            if (b < a.batch) a.slots[b] = granted ? slot(b, len) : -1;
        } else {
            upto[tid] = min(rows_upto, (uint32_t)a.tokens);
            base[tid] = granted ? len : -1;
            __syncthreads();
            const uint32_t stop = min(all_rows, (uint32_t)a.tokens);
            for (uint32_t t = min(rows_before, (uint32_t)a.tokens) + tid; t < stop; t += kThreads) {
                const int i = search(upto, t);
                const uint32_t first = i ? upto[i - 1] : min(rows_before, (uint32_t)a.tokens);
                a.slots[t] = base[i] >= 0 ? slot(b0 + i, (int64_t)base[i] + (t - first)) : -1;
            }
            rows_before = all_rows;
        }
        needed = __builtin_elementwise_add_sat(needed, all_need);
        taken += granted_need;
        __syncthreads();
    }
    if (a.cu)
        for (uint32_t t = min(rows_before, (uint32_t)a.tokens) + tid; t < (uint32_t)a.tokens; t += kThreads) a.slots[t] = -1;
    if (tid == 0) *a.free_count_out = count - (int)taken;
    if (bad) report(a.error);
}

}  // namespace

hipError_t launch_kv_assign(const AssignArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(kv_assign_kernel, dim3(1), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace nmi
