// kv_assign.hip -- the pages of a pool handed to the sequences that grow, and taken back from those that end, with
// what the kernels of the step need of it (first positions, lengths, packed offsets, the tokens' slots), for gfx950.
//
// The free pages are a stack in device memory.  Sequences that end push theirs, in the sequences' order and each in
// its positions'; then those that grow pop theirs in the same order: with need_b pages for sequence b, page j of b is
// the stack's entry count - 1 - (sum of need_i, i < b) - j.  A sequence is granted all of its new tokens or none: none
// where its row of the table is too short, or where it needs pages and the needs up to its own are more than the
// stack holds.  So everything follows from prefix sums, and equal inputs give equal tables.  No page has two owners: there
// are no counts of them, so what several sequences share must not come back here before its last owner ends.
//
// Bound: latency; a step of a batch moves some kilobytes.  One workgroup, since the stack is one: up to 1024 sequences
// at a time in its threads (256 of them for a decode step of as many: 4.0 us where 1024 threads took 4.9), sums over them
// by DPP and LDS; what varies in length (pages pushed and popped, slots) is dealt to the threads one by one, each finding
// its sequence by a binary search over the sums in LDS.  Measured (graph replays): a step of 1 / 32 / 256 / 1024 sequences
// 2.8 / 3.3 / 4.0 / 6.9 us, of 4000 23.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"
#include "nmi_packed.hpp"

namespace nmi {

namespace {

// Packed rows up to which the workgroup finds their slots too; more get a launch of their own.  One launch / two, graph
// replays: a prompt of 8000 6.6 / 7.3 us, 60 prompts of 9.5 thousand rows 10.4 / 8.0, of 33 thousand 23 / 8.7.
constexpr int kOneLaunch = 6144;
constexpr int kTurn = 4;                // elements of a thread at once, where there are many

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add_sat(uint32_t v) {
    return __builtin_elementwise_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
// Inclusive sums over a wave's lanes, saturating at 2^32 - 1 (more than there can be of anything here).
__device__ __forceinline__ uint32_t wave_scan_sat(uint32_t v) {
    v = dpp_add_sat<0x111, 0xF>(v);
    v = dpp_add_sat<0x112, 0xF>(v);
    v = dpp_add_sat<0x114, 0xF>(v);
    v = dpp_add_sat<0x118, 0xF>(v);
    v = dpp_add_sat<0x142, 0xA>(v);
    v = dpp_add_sat<0x143, 0xC>(v);
    return v;
}

// THREADS sequences at a time.
template <int THREADS>
struct Group {
    static constexpr int kWaves = THREADS / 64;
    // Inclusive sums of N values over the workgroup's threads (in place), the sums of all to `total`.  Every thread takes
    // part; `sums` is free afterwards only behind a barrier.
    template <int N>
    static __device__ __forceinline__ void scan(uint32_t (&v)[N], uint32_t (&sums)[N][kWaves], uint32_t (&total)[N]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = wave_scan_sat(v[i]);
            if (lane == 63) sums[i][wave] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t s = wave_scan_sat(lane < kWaves ? sums[i][lane] : 0u);
            total[i] = lane_u32(s, 63);
            if (wave) v[i] = __builtin_elementwise_add_sat(v[i], lane_u32(s, wave - 1));
        }
    }
    // The first of `n` ascending sums, a power of two up to THREADS, that is more than e (e is less than the last).
    static __device__ __forceinline__ int search(const uint32_t* upto, int n, uint32_t e) {
        int at = 0;
        for (int step = n >> 1; step; step >>= 1)
            if (upto[at + step - 1] <= e) at += step;
        return at;
    }
    // The same for kTurn elements at once, whose look-ups do not wait for one another.
    static __device__ __forceinline__ void search(const uint32_t* upto, int n, const uint32_t (&e)[kTurn], int (&at)[kTurn]) {
#pragma unroll
        for (int k = 0; k < kTurn; ++k) at[k] = 0;
        for (int step = n >> 1; step; step >>= 1) {
            uint32_t u[kTurn];
#pragma unroll
            for (int k = 0; k < kTurn; ++k) u[k] = upto[at[k] + step - 1];
#pragma unroll
            for (int k = 0; k < kTurn; ++k) at[k] += u[k] <= e[k] ? step : 0;
        }
    }
};

template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_assign_kernel(const AssignArgs a) {
    typedef Group<THREADS> G;
    __shared__ uint32_t upto[THREADS];          // sums over the sequences at hand
    __shared__ int32_t base[THREADS];           // of each: pages it had; then its first new position
    __shared__ uint32_t sums[3][G::kWaves];
    __shared__ uint32_t granted_pages;          // of the sequences at hand
    const int tid = threadIdx.x, lane = tid & 63;
    const int size = 1 << a.page_shift;
    const int64_t cap = (int64_t)a.max_pages << a.page_shift;
    bool bad = false;
    // (what the first sequences are, and the stack's height, asked for at once)
    const bool one = tid < a.batch;
    const int len_0 = one ? a.lens[tid] : -1, add_0 = one ? (a.add ? a.add[tid] : 1) : 0;
    int count = *a.free_count;
    if (count < 0 || count > a.n_pages) bad = true, count = count < 0 ? 0 : a.n_pages;
    // entries of `upto` that are looked through
    const int n = min(1 << (32 - __builtin_clz(a.batch)), THREADS);

    // pages that come back
    if (a.add)
        for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
            const int b = b0 + tid;
            const int add = b0 ? (b < a.batch ? a.add[b] : 0) : add_0;
            const int len = b0 ? (b < a.batch ? a.lens[b] : -1) : len_0;
            uint32_t back[1] = {0}, total[1];
            if (add < 0) back[0] = ((uint32_t)checked_len(len, a.max_pages, a.page_shift, &bad) + size - 1) >> a.page_shift;
            const uint32_t mine = back[0];
            G::scan(back, reinterpret_cast<uint32_t(&)[1][G::kWaves]>(sums[0]), total);
            if (total[0]) {
                upto[tid] = back[0];
                base[tid] = (int32_t)mine;
                __syncthreads();
                const uint32_t stop = pages_back(total[0], count, a.n_pages, &bad);
                for (uint32_t e = tid; e < stop; e += THREADS) {
                    const int i = G::search(upto, n, e);
                    const uint32_t j = e - (upto[i] - (uint32_t)base[i]);
                    const int id = a.table[(int64_t)(b0 + i) * a.table_stride + j];
                    if (id < 0 || id >= a.n_pages) bad = true;
                    a.free_pages[count + e] = id;
                }
                count += (int)stop;
            }
            __syncthreads();
        }

    // pages handed out, and what follows from them
    uint32_t needed = 0, rows_before = 0, taken = 0;    // of the sequences before those at hand; pages granted
    const uint32_t tokens = (uint32_t)a.tokens;
    for (int b0 = 0; b0 < a.batch; b0 += THREADS) {
        const int b = b0 + tid;
        const int add = b0 ? (b < a.batch ? (a.add ? a.add[b] : 1) : 0) : add_0;
        const int len = b0 ? (b < a.batch ? a.lens[b] : -1) : len_0;
        const int used = (int)(((uint32_t)max(len, 0) + size - 1) >> a.page_shift);
        bool fits = len >= 0 && add > 0 && (int64_t)len + add <= cap;
        if (len > cap) bad = true;
        // (rows first: those past the tokens given are not granted, and ask for no pages)
        uint32_t rows_upto = 0, all_rows = 0;
        if (a.cu) {
            uint32_t v[1] = {add > 0 ? (uint32_t)add : 0u}, total[1];
            G::scan(v, reinterpret_cast<uint32_t(&)[1][G::kWaves]>(sums[0]), total);
            rows_upto = __builtin_elementwise_add_sat(v[0], rows_before);
            all_rows = __builtin_elementwise_add_sat(total[0], rows_before);
            if (add > 0 && rows_upto > tokens) bad = true, fits = false;
        } else if (add > 1) {
            bad = true, fits = false;
        }
        const uint32_t need = fits ? (uint32_t)(((int64_t)len + add + size - 1) >> a.page_shift) - used : 0u;
        if (tid == 0) granted_pages = 0;
        uint32_t v[1] = {need}, all_need[1];
        G::scan(v, reinterpret_cast<uint32_t(&)[1][G::kWaves]>(sums[1]), all_need);
        const uint32_t need_upto = __builtin_elementwise_add_sat(v[0], needed);
        const bool granted = fits && (need == 0 || need_upto <= (uint32_t)count);
        // (those granted pages are the first that need any)
        const uint32_t most = wave_max_u32(granted && need ? v[0] : 0u);
        if (lane == 0 && most) atomicMax(&granted_pages, most);
        upto[tid] = v[0];
        base[tid] = used;
        if (b < a.batch) {
            a.start[b] = granted ? len : -1;
            a.kv_lens[b] = granted ? len + add : 0;
            a.lens_out[b] = granted ? len + add : (len >= 0 && add < 0 ? -1 : len);
            if (a.cu) {
                if (b == 0) a.cu[0] = 0;
                a.cu[b + 1] = (int32_t)min(rows_upto, tokens);
            }
        }
        __syncthreads();
        const uint32_t pages = granted_pages;
        for (uint32_t e = tid; e < pages; e += THREADS) {
            const int i = G::search(upto, n, e);
            const uint32_t first = i ? upto[i - 1] : 0u;
            const int id = a.free_pages[count - 1 - (int64_t)(taken + e)];
            if (id < 0 || id >= a.n_pages) bad = true;
            a.table[(int64_t)(b0 + i) * a.table_stride + base[i] + (e - first)] = id;
        }
        __syncthreads();
        auto slot = [&](int id, int64_t pos) {
            if (id < 0 || id >= a.n_pages) {
                bad = true;
                return (int64_t)-1;
            }
            return (int64_t)id * size + (pos & (size - 1));
        };
        if (!a.cu) {
            if (b < a.batch)
                a.slots[b] = granted ? slot(a.table[(int64_t)b * a.table_stride + (len >> a.page_shift)], len) : -1;
        } else if (a.slots) {
            upto[tid] = min(rows_upto, tokens);
            base[tid] = granted ? len : -1;
            __syncthreads();
            const uint32_t begin = min(rows_before, tokens), stop = min(all_rows, tokens);
            for (uint32_t t0 = begin + tid; t0 < stop; t0 += kTurn * THREADS) {
                uint32_t t[kTurn];
                int i[kTurn], id[kTurn];
                int64_t pos[kTurn];
#pragma unroll
                for (int k = 0; k < kTurn; ++k) t[k] = min(t0 + k * THREADS, stop - 1);
                G::search(upto, n, t, i);
#pragma unroll
                for (int k = 0; k < kTurn; ++k) {
                    const int start = base[i[k]];
                    pos[k] = start < 0 ? -1 : (int64_t)start + (t[k] - (i[k] ? upto[i[k] - 1] : begin));
                    if (start >= 0) id[k] = a.table[(int64_t)(b0 + i[k]) * a.table_stride + (pos[k] >> a.page_shift)];
                }
#pragma unroll
                for (int k = 0; k < kTurn; ++k)
                    if (t0 + k * THREADS < stop) a.slots[t[k]] = pos[k] >= 0 ? slot(id[k], pos[k]) : -1;
            }
        }
        rows_before = all_rows;
        needed = __builtin_elementwise_add_sat(needed, all_need[0]);
        taken += pages;
        __syncthreads();
    }
    if (a.cu && a.slots)
        for (uint32_t t = min(rows_before, tokens) + tid; t < tokens; t += THREADS) a.slots[t] = -1;
    if (tid == 0) *a.free_count_out = count - (int)taken;
    if (bad) report(a.error);
}

// The slots of packed rows, of the offsets, first positions and table that the kernel above leaves.  A workgroup takes
// kSlotRows rows, and the sequences that have them as many at a time.
constexpr int kSlotThreads = 256, kSlotRows = kTurn * kSlotThreads, kWindow = 1024;
__global__ __launch_bounds__(kSlotThreads) void kv_slots_kernel(const AssignArgs a) {
    typedef Group<kWindow> G;
    __shared__ uint32_t upto[kWindow];          // the ends of the sequences at hand, from the b0-th on
    __shared__ int32_t base[kWindow];           // their first new positions
    __shared__ uint32_t before[kSlotThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t t_first = blockIdx.x * kSlotRows, t_end = min(t_first + kSlotRows, (uint32_t)a.tokens);
    const int64_t size = (int64_t)1 << a.page_shift;
    // the sequences whose rows end at or before the first row
    uint32_t ended = 0;
    for (int b = tid; b < a.batch; b += kSlotThreads) ended += (uint32_t)a.cu[b + 1] <= t_first;
    ended = lane_u32(wave_scan_u32(ended), 63);
    if (lane == 0) before[tid >> 6] = ended;
    __syncthreads();
    int b0 = 0;
#pragma unroll
    for (int w = 0; w < kSlotThreads / 64; ++w) b0 += (int)before[w];
    bool bad = false;
    uint32_t begin = t_first;
    for (; begin < t_end && b0 < a.batch; b0 += kWindow) {
        for (int i = tid; i < kWindow; i += kSlotThreads) {
            upto[i] = (uint32_t)a.cu[min(b0 + i + 1, a.batch)];
            base[i] = a.start[min(b0 + i, a.batch - 1)];
        }
        const uint32_t first_row = (uint32_t)a.cu[b0];          // of sequence b0
        __syncthreads();
        const uint32_t stop = min(t_end, upto[kWindow - 1]);
        const uint32_t t0 = begin + tid;
        if (t0 < stop) {
            uint32_t t[kTurn];
            int i[kTurn], id[kTurn];
            int64_t pos[kTurn];
#pragma unroll
            for (int k = 0; k < kTurn; ++k) t[k] = min(t0 + k * kSlotThreads, stop - 1);
            G::search(upto, kWindow, t, i);
#pragma unroll
            for (int k = 0; k < kTurn; ++k) {
                const int start = base[i[k]];
                pos[k] = start < 0 ? -1 : (int64_t)start + (t[k] - (i[k] ? upto[i[k] - 1] : first_row));
                if (start >= 0) id[k] = a.table[(int64_t)(b0 + i[k]) * a.table_stride + (pos[k] >> a.page_shift)];
            }
#pragma unroll
            for (int k = 0; k < kTurn; ++k) {
                if (t0 + k * kSlotThreads >= stop) break;
                const bool none = pos[k] < 0, out = !none && (id[k] < 0 || id[k] >= a.n_pages);
                bad |= out;
                a.slots[t[k]] = none || out ? -1 : id[k] * size + (pos[k] & (size - 1));
            }
        }
        begin = max(begin, stop);
        __syncthreads();
    }
    for (uint32_t t = begin + tid; t < t_end; t += kSlotThreads) a.slots[t] = -1;      // behind the last sequence
    if (bad) report(a.error);
}

}  // namespace

hipError_t launch_kv_assign(const AssignArgs& a, hipStream_t stream) {
    if (a.batch <= 256 && a.tokens <= 1024) hipLaunchKernelGGL(kv_assign_kernel<256>, dim3(1), dim3(256), 0, stream, a);
    else if (!a.cu || a.tokens <= kOneLaunch) hipLaunchKernelGGL(kv_assign_kernel<1024>, dim3(1), dim3(1024), 0, stream, a);
    else {
        AssignArgs first = a;
        first.slots = nullptr;
        hipLaunchKernelGGL(kv_assign_kernel<1024>, dim3(1), dim3(1024), 0, stream, first);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        hipLaunchKernelGGL(kv_slots_kernel, dim3((a.tokens + kSlotRows - 1) / kSlotRows), dim3(kSlotThreads), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace nmi
