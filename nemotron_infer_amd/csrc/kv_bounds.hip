// kv_bounds.hip -- the smallest and largest key of pages of a paged KV cache, dim by dim, for gfx950.
//
//   bounds[page, head, 0, d] = min over the page's positions of k[d],  bounds[page, head, 1, d] = max,
//
// of the keys that the page stands for (codes times their scales in float32), rounded to the nearest bf16, for every page
// that the call's new positions complete; a dim with a NaN has NaN for both.  bf16 keys, and codes (4 significant bits)
// under powers of two, lose nothing by it; under other scales a bound may lie 2^-8 of its value inside the keys.  The
// newest page of a sequence needs none: it is attended whatever its score.
//
// Bound: latency (offsets, page id, keys one after another), then reading the pages, once.  A wave's load is one row of
// bf16, or two of e4m3 codes (4 bytes a lane), so that a lane keeps its dims and, where the waves of a workgroup share a
// page, only their results meet in LDS.  Measured: 12.6 MB of 3 prompts 5.3 us.
#include "nmi_device.hpp"
#include "nmi_launch.hpp"
#include "nmi_packed.hpp"

namespace nmi {

namespace {

// log2 of the largest page that a wave takes by itself.  Alone / together (8000 tokens of 8 heads, graph replays, bf16 and
// block scales): pages of 16 5.8, 5.4 / 8.1, 8.4 us, of 32 6.3, 5.4 / 5.7, 5.9, of 64 8.0, 6.7 / 5.7, 5.4.
constexpr int kAloneShift = 4;
// Loads of a wave on their way at once.  4 / 8 / 16 (the same): pages of 256 10.6, 7.9 / 8.1, 6.9 / 7.5, 6.9 us, of 64
// 5.8, 5.3 / 5.5, 5.2 / 5.7, 5.2.
constexpr int kWaves = 4, kAhead = 8;

// TOGETHER: the waves of a workgroup share a head's page; otherwise each has a head of its own.
template <KvForm FORM, bool TOGETHER>
__global__ __launch_bounds__(64 * kWaves) void kv_bounds_kernel(const BoundsArgs a) {
    constexpr bool CODES = FORM != KvForm::Bf16;
    constexpr int kDims = CODES ? 4 : 2, kRows = CODES ? 2 : 1;         // per lane; per load of a wave
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = TOGETHER ? (int)blockIdx.y : (int)blockIdx.y * kWaves + wave;
    if (h >= a.kv.n_kv) return;
    const bool teller = h == 0 && lane == 0 && (!TOGETHER || wave == 0);
    const int shift = a.kv.page_shift, size = 1 << shift;
    int b;
    int64_t page_place;
    if (a.cu) {
        if (blockIdx.x + 1 == gridDim.x) {
            if (h == 0 && (!TOGETHER || wave == 0)) check_offsets(a.cu, a.batch, a.tokens, a.kv.error, lane);
            return;
        }
        Packed s;
        if (!find_packed(a.cu, a.start, a.batch, a.tokens, blockIdx.x, lane,
                         [=](int64_t pos, int rows) { return pages_completed(pos, rows, shift); }, &s))
            return;
        b = s.b;
        page_place = (s.pos >> shift) + s.k;
    } else {
        b = blockIdx.x;
        const int start = load_const(a.start + b);
        if (start < 0 || !pages_completed(start, 1, shift)) return;
        page_place = start >> shift;
    }
    bool bad = page_place >= a.kv.max_pages;
    int page = 0;
    if (!bad) page = checked_page(load_const(a.kv.page_table + b * a.kv.table_stride + page_place), a.kv.n_pages, &bad);
    if (bad) {
        if (teller) report(a.kv.error);
        return;
    }
    const uint8_t* base = a.kv.k_pages + page * a.kv.page_stride + h * a.kv.head_stride + 4 * (CODES ? lane & 31 : lane);
    const int r0 = CODES ? lane >> 5 : 0;
    const float head_scale = FORM == KvForm::E4m3 && a.kv.k_scale ? load_const(a.kv.k_scale + h) : 1.f;
    const float* block_scale = FORM == KvForm::Block ? a.blocks.k + block_index(page, a.kv.n_kv, h, shift, 0) : nullptr;
    float lo[kDims], hi[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    // (a page has 16 rows at least, and a power of two of them: the waves' loads divide it)
    constexpr int kStep = (TOGETHER ? kWaves : 1) * kRows;
    for (int r = TOGETHER ? wave * kRows : 0; r < size; r += kStep * kAhead) {
        uint32_t w[kAhead];
        float s[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int row = r + j * kStep;
            if (row < size) {
                w[j] = *reinterpret_cast<const uint32_t*>(base + (row + r0) * a.kv.token_stride);
                s[j] = FORM == KvForm::Block ? load_const(block_scale + row / kPagedBlock) : head_scale;
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (r + j * kStep >= size) break;
            float x[kDims];
            if constexpr (CODES) {
                const uint2 v = e4m3x4_to_bf16(w[j]);
                x[0] = bf16lo_to_f32(v.x) * s[j], x[1] = bf16hi_to_f32(v.x) * s[j];
                x[2] = bf16lo_to_f32(v.y) * s[j], x[3] = bf16hi_to_f32(v.y) * s[j];
            } else {
                x[0] = bf16lo_to_f32(w[j]), x[1] = bf16hi_to_f32(w[j]);
            }
#pragma unroll
            for (int i = 0; i < kDims; ++i) {       // (NaN stays)
                lo[i] = __builtin_elementwise_minimum(lo[i], x[i]);
                hi[i] = __builtin_elementwise_maximum(hi[i], x[i]);
            }
        }
    }
    if constexpr (CODES) {
#pragma unroll
        for (int i = 0; i < kDims; ++i) {
            lo[i] = __builtin_elementwise_minimum(lo[i], __shfl_xor(lo[i], 32));
            hi[i] = __builtin_elementwise_maximum(hi[i], __shfl_xor(hi[i], 32));
        }
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(a.bounds) + ((int64_t)page * a.kv.n_kv + h) * kPagedHead;   // two dims each
    if constexpr (!TOGETHER) {
        if (CODES && lane >= 32) return;
#pragma unroll
        for (int i = 0; i < kDims; i += 2) {
            out[(kDims * lane + i) / 2] = pack_bf16(lo[i], lo[i + 1]);
            out[(kPagedHead + kDims * lane + i) / 2] = pack_bf16(hi[i], hi[i + 1]);
        }
    } else {
        __shared__ float sm[2][kWaves][kPagedHead];
        if (!CODES || lane < 32)
#pragma unroll
            for (int i = 0; i < kDims; ++i) {
                sm[0][wave][kDims * lane + i] = lo[i];
                sm[1][wave][kDims * lane + i] = hi[i];
            }
        __syncthreads();
        if (tid >= kPagedHead) return;
        const int side = tid >> 6, d = 2 * (tid & 63);
        float x = sm[side][0][d], y = sm[side][0][d + 1];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            const float u = sm[side][w][d], v = sm[side][w][d + 1];
            x = side ? __builtin_elementwise_maximum(x, u) : __builtin_elementwise_minimum(x, u);
            y = side ? __builtin_elementwise_maximum(y, v) : __builtin_elementwise_minimum(y, v);
        }
        out[tid] = pack_bf16(x, y);
    }
}

template <KvForm FORM>
hipError_t launch(const BoundsArgs& a, hipStream_t stream) {
    const int64_t jobs = a.cu ? most_pages_completed(a.tokens, a.batch, a.kv.page_shift) + 1 : a.batch;
    if (a.kv.page_shift <= kAloneShift)
        hipLaunchKernelGGL((kv_bounds_kernel<FORM, false>), dim3((uint32_t)jobs, (a.kv.n_kv + kWaves - 1) / kWaves),
                           dim3(64 * kWaves), 0, stream, a);
    else
        hipLaunchKernelGGL((kv_bounds_kernel<FORM, true>), dim3((uint32_t)jobs, a.kv.n_kv), dim3(64 * kWaves), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_bounds(const BoundsArgs& a, KvForm form, hipStream_t stream) {
    switch (form) {
        case KvForm::Bf16: return launch<KvForm::Bf16>(a, stream);
        case KvForm::E4m3: return launch<KvForm::E4m3>(a, stream);
        default: return launch<KvForm::Block>(a, stream);
    }
}

}  // namespace nmi
